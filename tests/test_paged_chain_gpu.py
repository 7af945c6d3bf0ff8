"""The whole chain of the paged cache (prefill, continuation, free, fork, compaction, decode steps with
and without a shared prefix) against the one-sequence path, every sequence of every pass.

A router whose k-th and next scores nearly tie turns one rounding into another expert and with it the
rest of a forward. So a token's experts and weights are decided once, by the path that meets the
token (with all tokens before it) first, and every later pass over it takes the same. What is left
between the two paths is rounding.

Tolerance: the one of tests/test_paged_gpu.py for logits. Each path may differ from the oracle by a max
relative error e = 2e-2 and a cosine c = 0.999, so the two from each other by 2 e and 2 c^2 - 1. The K
and V rows of the full-attention layers, which the paged path reads back from the table's pages, are
held to that cosine, row by row: a linear map of the normalised hidden states (and a rotation) that
the logits are a linear map of, too. A row of another token has a cosine near 0 (256 dims: 0.06), a
key rotated one position too far one of about 0.93 (the mean of cos(1e4^-u) over u in [0, 1])."""
import pytest
import torch

from tests._util import COS_TOL
from tests.test_paged_gpu import _ok
from tests.test_streams_gpu import _model, _prompts

pytestmark = pytest.mark.gpu


class Experts:
    """Every MoE layer's experts and weights, decided once a token: ``keys`` names the rows of the
    forward to come by all their tokens so far."""

    def __init__(self, model):
        self.memo, self.keys, self.used = {}, [], 0
        for i, layer in enumerate(model.layers):
            if hasattr(layer.mlp, "route"):
                layer.mlp.route = self._wrap(i, layer.mlp.route)

    def _wrap(self, i, route):
        def wrapped(x):
            inds, w = route(x)
            k = inds.shape[-1]
            a, b = inds.reshape(-1, k).clone(), w.reshape(-1, k).clone()
            assert a.shape[0] == len(self.keys)
            for r, key in enumerate(self.keys):
                if (i, key) in self.memo:
                    a[r], b[r] = self.memo[i, key]
                    self.used += 1
                else:
                    self.memo[i, key] = a[r].clone(), b[r].clone()
            return a.reshape(inds.shape), b.reshape(w.shape)
        return wrapped


class Chain:
    def __init__(self, kind, rows):
        from lagunalab_b200 import paged
        _, self.model, _, _ = _model(kind)
        self.experts = Experts(self.model)
        self.cache = paged.PagedCache(self.model, 7, 64, rows)
        self.tokens, self.want, self.passes = {}, {}, 0

    def _plain(self, tokens):
        """(logits of all positions, per full layer its K and V rows [n, Hkv, D]) of the one-sequence
        path over the tokens."""
        key = tuple(tokens)
        if key not in self.want:
            self.experts.keys = [key[:i + 1] for i in range(len(key))]
            cache = self.model.make_cache(capacity=len(key))
            ids = torch.tensor(tokens, dtype=torch.int32, device="cuda").view(1, -1)
            logits = self.model(ids, cache)[0]
            rows = {i: [t[0, :, :len(key)].transpose(0, 1).float() for t in (c.keys, c.values)]
                    for i, c in enumerate(cache) if self.model.layers[i].self_attn.window is None}
            self.want[key] = logits, rows
        return self.want[key]

    def run(self, streams, parts, forward):
        """One pass with parts[i] new tokens of stream streams[i]; forward() gives its logits."""
        full = [self.tokens.get(s, []) + p for s, p in zip(streams, parts)]
        plain = [self._plain(f) for f in full]
        self.experts.keys = [tuple(f[:i + 1]) for f, p in zip(full, parts)
                             for i in range(len(f) - len(p), len(f))]
        before = self.experts.used
        logits = forward()
        moe = sum(hasattr(layer.mlp, "route") for layer in self.model.layers)
        assert self.experts.used - before == moe * sum(map(len, parts))
        for s, f, row, (want, rows) in zip(streams, full, logits, plain):
            self.tokens[s] = f
            _ok(row, want[-1])
            self._rows(s, rows)
        self.passes += 1

    def _rows(self, s, rows):
        c, n = self.cache, len(self.tokens[s])
        assert c.lens[s].item() == n
        pages = c.table[s, :-(-n // c.page_rows)].long()
        for layer, both in rows.items():
            for j in range(2):
                got = c.pool[layer, j, pages].transpose(1, 2).flatten(0, 1)[:n].float()
                near = torch.nn.functional.cosine_similarity(got.flatten(1), both[j].flatten(1))
                assert float(near.min()) >= 2 * COS_TOL ** 2 - 1, (layer, j, int(near.argmin()))

    def prefill(self, streams, parts):
        from lagunalab_b200 import paged
        self.run(streams, parts, lambda: paged.prefill(self.model, self.cache, streams, parts))

    def fork(self, src, dst):
        self.cache.fork(src, dst)
        self.tokens.update({d: list(self.tokens[s]) for s, d in zip(src, dst)})

    def free(self, ids):
        self.cache.free(ids)
        for s in ids:
            self.tokens.pop(s)

    def decode(self, streams, steps, prefix=0, seed=0):
        from lagunalab_b200 import paged
        self.cache.reserve(streams, [len(self.tokens[s]) + steps for s in streams])
        dec = paged.Decoder(self.model, self.cache, streams, prefix=prefix)
        for i in range(steps):
            tok = torch.randint(0, 512, (len(streams),), dtype=torch.int32,
                                generator=torch.Generator().manual_seed(100 * seed + i))
            self.run(streams, [[int(t)] for t in tok], lambda: dec.step(tok.cuda()))


@pytest.mark.parametrize("kind,rows", [("full", 16), ("full", 64), ("sliding", 32), ("sliding", 128)])
def test_every_pass_of_a_chain(kind, rows):
    c = Chain(kind, rows)
    p = lambda lens, seed: [t.tolist() for t in _prompts(lens, seed)]
    c.prefill([4, 0, 2], p([37, 5, 130], 3))
    c.prefill([2, 4, 1], p([20, 33, 9], 4))  # continuations, and a fresh one beside them
    c.free([0])
    c.fork([2, 2, 4], [0, 3, 5])
    c.cache.compact()
    c.decode([0, 2, 3, 5, 1], 3, seed=1)
    c.prefill([3, 6, 0], p([18, 70, 1], 5))  # children go on as prompts do
    c.free([4, 2, 1])
    assert c.cache.compact() > 0 or rows == 128
    shared = 150  # streams 0 and 3 are children of one
    c.decode([3, 0], 2, prefix=shared, seed=2)
    c.fork([3, 5], [1, 2])
    c.decode([1, 3, 0], 2, prefix=shared, seed=3)
    c.decode([2, 6], 2, seed=4)
    assert c.passes == 12
    # the bar tells sequences from one another
    a, b = (c._plain(c.tokens[s])[0][-1] for s in (3, 6))
    with pytest.raises(AssertionError):
        _ok(a, b)
