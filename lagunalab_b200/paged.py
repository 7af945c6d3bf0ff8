"""Serving several sequences from one paged K/V cache (no counterpart in the reference, whose caches
hold one sequence each, laguna_mlx/cache.py:66-157).

``PagedCache`` holds every layer's K and V in pages that streams share: a fork costs at most one
page of copies, a prompt that many streams begin with is stored once, and a stream that ends gives
its pages back. ``prefill`` runs the packed new tokens of several streams through the model,
``step`` one token of each; rows below a shared prefix are read once for all streams of a step.
``generate`` puts them together. Streams are rows of the cache's table.
"""
import torch

from . import ops


class PagedCache:
    """K/V of ``streams`` streams over ``pages`` pages of ``page_rows`` rows (16, 32, 64 or 128) for
    every layer of ``model``: ``pool`` bf16 [layers, 2, pages, Hkv, page_rows, head_dim]. ``table``
    int32 [streams, pages per stream], ``lens`` int32 [streams] and ``refs`` int32 [pages] live on
    the device; ``max_rows`` bounds a stream (default: the whole pool). Sliding-window layers keep
    their older rows, too: the pages are common to all layers."""

    def __init__(self, model, streams, pages, page_rows=64, max_rows=None, device="cuda"):
        a = model.args
        if page_rows not in (16, 32, 64, 128):
            raise ValueError(f"pages of {page_rows} rows (16, 32, 64 or 128)")
        if a.head_dim != 128:
            raise ValueError(f"head_dim {a.head_dim}: the paged attention takes 128")
        per = pages if max_rows is None else min(pages, -(-max_rows // page_rows))
        i = dict(dtype=torch.int32, device=device)
        self.page_rows, self.streams, self.pages = page_rows, streams, pages
        self.pool = torch.zeros(len(model.layers), 2, pages, a.num_key_value_heads, page_rows,
                                a.head_dim, dtype=torch.bfloat16, device=device)
        self.table = torch.full((streams, per), -1, **i)
        self.lens, self.refs = torch.zeros(streams, **i), torch.zeros(pages, **i)

    def _ids(self, ids):
        return torch.as_tensor(ids, dtype=torch.int32, device=self.table.device).reshape(-1)

    @staticmethod
    def _done(status, what):
        code, count = status.tolist()
        if code:
            raise ValueError(f"{what}: {ops.PAGES_ERRORS[code]}")
        return count

    def reserve(self, ids, rows):
        """Pages for ``rows[i]`` rows in all of each stream ``ids[i]``; returns the pages taken."""
        return self._done(ops.pages_reserve(self.table, self.refs, self._ids(ids), self._ids(rows),
                                            self.page_rows), "reserve")

    def fork(self, src, dst):
        """The empty streams ``dst`` become copies of the streams ``src``, sharing whole pages."""
        return self._done(ops.pages_fork(self.pool, self.table, self.lens, self.refs,
                                         self._ids(src), self._ids(dst)), "fork")

    def free(self, ids):
        """The streams ``ids`` give their pages back."""
        return self._done(ops.pages_free(self.table, self.lens, self.refs, self._ids(ids)), "free")

    def compact(self):
        """Live pages move to the lowest ids; returns how many moved."""
        return self._done(ops.pages_compact(self.pool, self.table, self.refs), "compact")

    def free_pages(self):
        return int((self.refs == 0).sum())

    @property
    def nbytes(self):
        return self.pool.numel() * self.pool.element_size()


class _Batch:
    """One pass's streams: token t belongs to row seq[t] of ``table`` at position pos[t]; a plan a
    window (layers of one kind share it)."""

    def __init__(self, model, cache, table, seq, pos, plan):
        self.cache, self.table, self.seq, self.pos = cache, table, seq, pos
        self._plan, self._plans = plan, {}
        for layer in model.layers:
            self.plan(layer.self_attn)

    def plan(self, at):
        key = (at.n_heads, at.window or 0)
        if key not in self._plans:
            self._plans[key] = self._plan(at.n_heads, at.n_kv_heads, self.cache.page_rows, key[1])
        return self._plans[key]

    def attend(self, layer, at, xn, residual):
        """o_proj(attention) [+ residual] of the packed normalised rows xn [T, H]."""
        k, v = self.cache.pool[layer]
        Hq, Hkv, D = at.n_heads, at.n_kv_heads, at.head_dim
        q, gate = ops.attn_prep_pages(at._qkvg(xn), Hq, Hkv, D, at.q_norm.weight, at.k_norm.weight,
                                      at.eps, at.rope_theta, self.seq, self.pos, self.table, k, v,
                                      gate_per_head=at.per_head_gate, rope=at.rope)
        plan, per_head = self.plan(at), at.per_head_gate
        run = ops.prompt_attention if plan.kind == "prompt" else ops.stream_attention
        o = run(q, k, v, self.table, plan, at.scale, gate=gate if per_head else None)
        o = o.view(-1, Hq * D)
        return at.o_proj(o if per_head else o * gate, residual=residual)


def _forward(model, ids, batch):
    """Final normalised hidden states [T, H] of the batch's packed tokens."""
    m = model.model
    x = m.embed_tokens(ids.reshape(1, -1)).reshape(ids.shape[0], -1)
    xn = m.layers[0].input_layernorm(x)
    for i, layer in enumerate(m.layers):
        h = batch.attend(i, layer.self_attn, xn, x)
        y = layer.mlp(layer.post_attention_layernorm(h))
        nxt = m.layers[i + 1].input_layernorm if i + 1 < len(m.layers) else m.norm
        x, xn = ops.rmsnorm(y, nxt.weight, nxt.eps, residual=h)
    return xn


def prefill(model, cache, streams, prompts):
    """The new tokens ``prompts[i]`` (int sequences, at least one token each) of each stream
    ``streams[i]`` (distinct) behind the rows it holds, packed into one pass: their rows are
    reserved and written, lengths advanced. Returns the logits [n, V] of each prompt's last
    token."""
    dev, n = cache.table.device, len(streams)
    new = [len(p) for p in prompts]
    if n != len(prompts) or n == 0 or min(new) < 1:
        raise ValueError("prefill takes one or more tokens for each of its streams")
    if len(set(int(s) for s in streams)) != n:
        raise ValueError("prefill: a stream is listed twice")
    ids_s = cache._ids(streams)
    if int(ids_s.min()) < 0 or int(ids_s.max()) >= cache.streams:
        raise ValueError(f"prefill: a stream outside [0, {cache.streams})")
    held = cache.lens[ids_s.long()]
    counts = torch.tensor(new, dtype=torch.int32, device=dev)
    kv = held + counts
    cache.reserve(ids_s, kv)
    cu = torch.zeros(n + 1, dtype=torch.int32, device=dev)
    cu[1:] = counts.cumsum(0)
    T = sum(new)
    seq = torch.repeat_interleave(torch.arange(n, dtype=torch.int32, device=dev), counts.long(),
                                  output_size=T)
    pos = torch.arange(T, dtype=torch.int32, device=dev) + (held - cu[:-1])[seq.long()]
    ids = torch.cat([torch.as_tensor(p, dtype=torch.int32).reshape(-1).to(dev) for p in prompts])
    batch = _Batch(model, cache, cache.table[ids_s.long()], seq, pos,
                   lambda Hq, Hkv, R, W: ops.prompt_plan(cu, kv, T, Hq, Hkv, R, window=W))
    h = _forward(model, ids, batch)
    cache.lens[ids_s.long()] = kv
    return model.lm_head(h[cu[1:].long() - 1])


class Decoder:
    """Decode steps of ``streams`` (distinct rows of the cache), one token of each a step. Rows
    [0, prefix) must be the same for all of them (a fork's, or the same tokens' rows); they are read
    once a step. ``reserve`` the rows to come before: a step writes row ``cache.lens`` of each
    stream and takes no page. A stream without a page for that row (freed, or past its reserved
    rows) sits the step out: its length stays, its logits are NaN, ``wrote`` (device bool [n], of
    the last step) says so; after a ``reserve`` it goes on where it was. ``step`` changes only device
    memory that the object and the cache hold, so it can be captured in a CUDA graph after a first
    call."""

    def __init__(self, model, cache, streams, prefix=0):
        if len(set(int(s) for s in streams)) != len(streams):
            raise ValueError("a stream is listed twice")
        self.model, self.cache = model, cache
        self.ids = cache._ids(streams).long()
        if int(self.ids.min()) < 0 or int(self.ids.max()) >= cache.streams:
            raise ValueError(f"a stream outside [0, {cache.streams})")
        n, dev = len(streams), cache.table.device
        self.table = cache.table[self.ids]
        self.pos = cache.lens[self.ids]
        if prefix and int(self.pos.min()) < prefix:
            raise ValueError(f"a stream holds {int(self.pos.min())} rows of the {prefix} shared")
        self.kv = self.pos + 1
        self.wrote = torch.zeros(n, dtype=torch.bool, device=dev)
        self.batch = _Batch(model, cache, self.table,
                            torch.arange(n, dtype=torch.int32, device=dev), self.pos,
                            lambda Hq, Hkv, R, W: ops.stream_plan(self.kv, Hq, Hkv, R,
                                                                  prefix=prefix, window=W))

    def step(self, tokens):
        """Logits [n, V] after one token of each stream (device int32 [n])."""
        R, M = self.cache.page_rows, self.table.shape[1]
        self.pos.copy_(self.cache.lens[self.ids])
        self.table.copy_(self.cache.table[self.ids])
        # A row that no page takes is not written, so the length must not count it: a later reserve
        # would put a page there with another stream's rows. Such a stream sees no key (kv 0).
        col = (self.pos // R).long()
        page = self.table.gather(1, col.clamp(max=M - 1)[:, None])[:, 0]
        torch.logical_and(page >= 0, col < M, out=self.wrote)
        torch.mul(self.pos + 1, self.wrote, out=self.kv)
        for plan in self.batch._plans.values():
            plan.update()
        h = _forward(self.model, tokens, self.batch)
        self.cache.lens[self.ids] = self.pos + self.wrote
        return self.model.lm_head(h).masked_fill(~self.wrote[:, None], float("nan"))


def generate(model, prompts, max_tokens, page_rows=64):
    """Greedy continuations of several prompts (int sequences), decoded together: their common
    beginning is prefilled and stored once. Returns a list of ``max_tokens`` ids a prompt."""
    prompts = [[int(t) for t in p] for p in prompts]
    n = len(prompts)
    if n == 0 or min(len(p) for p in prompts) < 1 or max_tokens < 1:
        raise ValueError("generate takes prompts of one or more tokens and max_tokens >= 1")
    shared = 0
    if n > 1:  # at least one token of every prompt stays for its own prefill
        most = min(len(p) for p in prompts) - 1
        while shared < most and all(p[shared] == prompts[0][shared] for p in prompts):
            shared += 1
    rows = [len(p) + max_tokens for p in prompts]
    first = -(-shared // page_rows)
    pages = first + sum(-(-r // page_rows) - shared // page_rows for r in rows)
    cache = PagedCache(model, n + 1, pages, page_rows, max(rows), model.lm_head.weight.device)
    streams = list(range(n))
    if shared:
        prefill(model, cache, [n], [prompts[0][:shared]])
        cache.fork([n] * n, streams)
        cache.free([n])
    logits = prefill(model, cache, streams, [p[shared:] for p in prompts])
    cache.reserve(streams, rows)
    dec = Decoder(model, cache, streams, prefix=shared)
    tok, out = ops.argmax(logits), []
    for _ in range(max_tokens - 1):
        out.append(tok)
        tok = ops.argmax(dec.step(tok))
    out.append(tok)
    return torch.stack(out, 1).tolist()
