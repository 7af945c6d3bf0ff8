"""Serving several sequences from a paged cache (``paged``; no counterpart in the reference) against
the one-sequence path: logits of packed prefills, continuations, forks and decode steps, for the
decoder with full attention and the one with sliding windows, YaRN and layers of different head
counts.

Tolerance: the other tests hold the one-sequence path to the oracle within a max relative error e =
2e-2 and a cosine of c = 0.999 (tests/_util.py), and the paged path is held to the same bar. With a,
b the two paths' logits and r the oracle's, max|a - b| <= max|a - r| + max|b - r| <= 2 e max|r|, and
the angle between a and b is at most the sum of theirs to r, whose cosine is 2 c^2 - 1. So the two
paths may differ by 2 e and by that cosine without either being further from the oracle than it
may.

A router whose k-th and next scores nearly tie turns one rounding into another expert and with it
the rest of the forward, in either path. So the layers are also compared one by one, each on the
one-sequence path's own activations, and whole forwards where both took the same experts."""
import pytest
import torch

from tests._util import COS_TOL, REL_TOL, cos, rel_err
from tests.test_streams_gpu import _model, _prompts

pytestmark = pytest.mark.gpu


def _ok(got, want):
    assert rel_err(got, want) <= 2 * REL_TOL and cos(got, want) >= 2 * COS_TOL ** 2 - 1, \
        (rel_err(got, want), cos(got, want))


class Picks:
    """Every MoE layer's experts of the rows of the last forward, through the patchable ``route``."""

    def __init__(self, model):
        self.last = {}
        for i, layer in enumerate(model.layers):
            if hasattr(layer.mlp, "route"):
                layer.mlp.route = self._wrap(i, layer.mlp.route)

    def _wrap(self, i, route):
        def wrapped(x):
            inds, w = route(x)
            self.last[i] = inds.reshape(-1, inds.shape[-1]).sort(-1)[0]
            return inds, w
        return wrapped

    def rows(self, first, last):
        """Per token its experts in all layers."""
        layers = [v[first:last].tolist() for v in self.last.values()]
        return [tuple(map(tuple, t)) for t in zip(*layers)]


def _compare(model, picks, logits, taken, sequences):
    """Each sequence's last logits against the one-sequence path. taken: the experts of all its
    tokens, as the passes so far chose them; a sequence is held to the bar where the other path
    chose the same for every token (another expert of an earlier token is in the keys and values).
    Returns (sequences held to the bar, sequences)."""
    same = 0
    for row, mine, tokens in zip(logits, taken, sequences):
        ids = torch.tensor(tokens, dtype=torch.int32, device="cuda").view(1, -1)
        want = model.last_logits(ids, model.make_cache(capacity=len(tokens))).view(-1)
        if picks.rows(0, len(tokens)) == mine:
            _ok(row, want)
            same += 1
    return same, len(sequences)


def _activations(model, tokens):
    """Per layer (normalised input, residual stream, stream after attention) [n, H] of the
    one-sequence path over the tokens."""
    from lagunalab_b200 import ops
    m, out = model.model, []
    x = m.embed_tokens(torch.tensor(tokens, dtype=torch.int32, device="cuda").view(1, -1))
    xn = m.layers[0].input_layernorm(x)
    for i, (layer, c) in enumerate(zip(m.layers, model.make_cache(capacity=len(tokens)))):
        h = layer.self_attn(xn, None, c, residual=x)
        out.append((xn[0], x[0], h[0]))
        y = layer.mlp(layer.post_attention_layernorm(h))
        nxt = m.layers[i + 1].input_layernorm if i + 1 < len(m.layers) else m.norm
        x, xn = ops.rmsnorm(y, nxt.weight, nxt.eps, residual=h)
    return out


@pytest.mark.parametrize("kind,rows", [("full", 128), ("sliding", 16), ("sliding", 32)])
def test_layers_on_the_same_activations(kind, rows):
    """Prompts, continuations, and decode steps of forks that share their first rows, layer by
    layer: o_proj(attention) + residual of every token."""
    from lagunalab_b200 import ops, paged
    _, model, _, _ = _model(kind)
    length = {0: 60, 1: 9, 2: 165}
    acts = {s: _activations(model, _prompts([n], 10 + s)[0].tolist()) for s, n in length.items()}
    cache = paged.PagedCache(model, 5, 64, rows)
    cache.reserve([0, 1, 2], list(length.values()))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")

    def run(rows_of, plan):  # rows_of: (stream of the cache, sequence, first, last) per row of table
        table = cache.table[[r[0] for r in rows_of]]
        seq = i32([b for b, r in enumerate(rows_of) for _ in range(r[2], r[3])])
        pos = i32([p for r in rows_of for p in range(r[2], r[3])])
        batch = paged._Batch(model, cache, table, seq, pos, plan)
        for i, layer in enumerate(model.layers):
            xn, x, h = (torch.cat([acts[r[1]][i][j][r[2]:r[3]] for r in rows_of]) for j in range(3))
            got = batch.attend(i, layer.self_attn, xn, x)
            _ok(got.float() - x.float(), h.float() - x.float())

    def prompts(parts):
        n = [b - a for _, _, a, b in parts]
        cu, kv = i32([sum(n[:i]) for i in range(len(n) + 1)]), i32([p[3] for p in parts])
        run(parts, lambda Hq, Hkv, R, W: ops.prompt_plan(cu, kv, sum(n), Hq, Hkv, R, window=W))

    prompts([(0, 0, 0, 33), (1, 1, 0, 8), (2, 2, 0, 150)])
    prompts([(0, 0, 33, 59), (2, 2, 150, 164)])
    cache.lens[:3] = i32([59, 8, 164])
    cache.fork([2, 2], [3, 4])
    cache.reserve([2, 3, 4], [165] * 3)
    parts = [(s, q, length[q] - 1, length[q]) for s, q in [(2, 2), (3, 2), (4, 2)]]
    kv = i32([165] * 3)
    run(parts, lambda Hq, Hkv, R, W: ops.stream_plan(kv, Hq, Hkv, R, prefix=164, window=W))
    parts = [(s, q, length[q] - 1, length[q]) for s, q in [(0, 0), (1, 1), (2, 2)]]
    kv3 = i32([60, 9, 165])
    run(parts, lambda Hq, Hkv, R, W: ops.stream_plan(kv3, Hq, Hkv, R, window=W))


@pytest.mark.parametrize("kind,rows", [("full", 16), ("full", 64), ("sliding", 32)])
def test_packed_prefill_continuation_fork_and_decode(kind, rows):
    from lagunalab_b200 import paged
    _, model, _, _ = _model(kind)
    picks, done, full, taken = Picks(model), [], {}, {}

    def check(logits, streams, parts):
        """The last pass: parts[i] new tokens of stream streams[i], packed."""
        at = 0
        for s, p in zip(streams, parts):
            full[s] = full.get(s, []) + p
            taken[s] = taken.get(s, []) + picks.rows(at, at + len(p))
            at += len(p)
        done.append(_compare(model, picks, logits, [taken[s] for s in streams],
                             [full[s] for s in streams]))

    prompts = [p.tolist() for p in _prompts([37, 5, 130], 3)]
    cache = paged.PagedCache(model, 7, 64, rows)
    check(paged.prefill(model, cache, [4, 0, 2], prompts), [4, 0, 2], prompts)
    # a continuation of two of them, packed with a fresh one
    more = [p.tolist() for p in _prompts([20, 33, 9], 4)]
    check(paged.prefill(model, cache, [2, 4, 1], more), [2, 4, 1], more)
    # children of one stream, each with its own next tokens, beside the others
    cache.free([0])
    cache.fork([2, 2, 4], [0, 3, 5])
    for d in (full, taken):
        d.update({0: d[2], 3: d[2], 5: d[4]})
    cache.compact()
    streams = [0, 2, 3, 5, 1]
    cache.reserve(streams, [len(full[s]) + 4 for s in streams])
    dec = paged.Decoder(model, cache, streams)
    for step in range(4):
        tok = torch.randint(0, 512, (5,), generator=torch.Generator().manual_seed(step))
        check(dec.step(tok.to(torch.int32).cuda()), streams, [[int(t)] for t in tok])
    assert cache.lens.tolist() == [len(full.get(s, [])) for s in range(7)]
    assert sum(d[0] for d in done) > 0, done  # some sequence has been compared


def _children(model, prompt, n):
    from lagunalab_b200 import paged
    cache = paged.PagedCache(model, n + 1, 40, 32)
    paged.prefill(model, cache, [0], [prompt])
    streams = list(range(1, n + 1))
    cache.fork([0] * n, streams)
    cache.reserve(streams, [170] * n)
    return cache, paged.Decoder(model, cache, streams, prefix=len(prompt))


@pytest.mark.parametrize("kind", ["full", "sliding"])
def test_shared_prefix_decode_graph(kind):
    """Children of one prompt decode with the prompt read once; replayed from a CUDA graph they
    give the bits of eager steps."""
    _, model, _, _ = _model(kind)
    prompt = _prompts([150], 5)[0].tolist()
    toks = [torch.tensor([(7 * s + 31 * t) % 512 for s in range(5)], dtype=torch.int32,
                         device="cuda") for t in range(6)]
    cache_e, eager = _children(model, prompt, 5)
    cache_g, dec = _children(model, prompt, 5)
    want = [eager.step(t).clone() for t in toks]
    tok = toks[0].clone()
    assert torch.equal(dec.step(tok), want[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = dec.step(tok)
    for t in range(1, 6):
        tok.copy_(toks[t])
        graph.replay()
        assert torch.equal(logits, want[t])
    assert torch.equal(cache_g.lens, cache_e.lens) and torch.equal(cache_g.pool, cache_e.pool)


def test_generate_is_prefill_fork_and_decode():
    from lagunalab_b200 import ops, paged
    _, model, _, _ = _model("full")
    base = _prompts([90], 6)[0].tolist()
    prompts = [base + p.tolist() for p in _prompts([3, 17, 1], 7)]
    shared = 90
    while all(len(p) - 1 > shared and p[shared] == prompts[0][shared] for p in prompts):
        shared += 1
    got = paged.generate(model, prompts, 8, page_rows=16)
    cache = paged.PagedCache(model, 4, 64, 16)
    paged.prefill(model, cache, [3], [base[:shared]])
    cache.fork([3] * 3, [0, 1, 2])
    tok = ops.argmax(paged.prefill(model, cache, [0, 1, 2], [p[shared:] for p in prompts]))
    cache.reserve([0, 1, 2], [len(p) + 8 for p in prompts])
    dec, want = paged.Decoder(model, cache, [0, 1, 2], prefix=shared), []
    for _ in range(8):
        want.append(tok)
        tok = ops.argmax(dec.step(tok))
    assert got == torch.stack(want, 1).tolist()
    assert paged.generate(model, [base], 3) and len(paged.generate(model, [base], 1)[0]) == 1


def test_refusals():
    from lagunalab_b200 import paged
    _, model, _, _ = _model("full")
    cache = paged.PagedCache(model, 3, 4, 16)
    with pytest.raises(ValueError, match="twice"):
        paged.prefill(model, cache, [0, 0], [[1], [2]])
    with pytest.raises(ValueError, match="outside"):
        paged.prefill(model, cache, [3], [[1]])
    with pytest.raises(ValueError, match="one or more"):
        paged.prefill(model, cache, [0], [[]])
    with pytest.raises(ValueError, match="free pages"):
        paged.prefill(model, cache, [0, 1], [[1] * 40, [2] * 40])
    assert cache.free_pages() == 4
    paged.prefill(model, cache, [0], [[1, 2, 3]])
    with pytest.raises(ValueError, match="fork"):
        cache.fork([0], [0])
    with pytest.raises(ValueError, match="shared"):
        paged.Decoder(model, cache, [0], prefix=4)
    with pytest.raises(ValueError, match="twice"):
        paged.Decoder(model, cache, [0, 0])
    with pytest.raises(ValueError, match="page"):
        paged.PagedCache(model, 1, 1, 24)
