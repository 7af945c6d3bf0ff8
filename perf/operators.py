"""The operators of the paged K/V cache, as cases to measure: causal attention of packed prompts,
attention of decode streams that share a prefix, and the cache's page operations (fork, free,
compact). Each case runs in a plain form of elementary torch operations or, where ``own`` is true,
through ``lagunalab_b200.ops``.

Layouts: K/V pages bf16 [P, Hkv, R, D], a table int32 [B, M] naming each sequence's pages; row j of
sequence b is row j % R of page table[b, j // R].
"""
import math
import random

import torch

own = False

D = 128


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # a chat server's step between turns: a few new tokens of three conversations
        dict(name="prompt_turns", op="prompt", seqs=3, new_min=1, new_max=40, hist_max=700, hq=32,
             hkv=4, rows=64, window=0, gate=True, pick=3),
        # a batch of fresh prompts of a server, of any length
        dict(name="prompt_ragged", op="prompt", seqs=16, new_min=1, new_max=1500, hist_max=0, hq=32,
             hkv=4, rows=64, window=0, gate=True, pick=5),
        # the decoder benchmark's prompt
        dict(name="prompt_8k", op="prompt", seqs=1, new_min=8192, new_max=8192, hist_max=0, hq=32,
             hkv=4, rows=64, window=0, gate=True, pick=1),
        # sliding-window layers, another head layout, small pages
        dict(name="prompt_window", op="prompt", seqs=3, new_min=2100, new_max=2600, hist_max=200,
             hq=32, hkv=8, rows=16, window=512, gate=False, pick=7),
        # chunked prefill: a chunk of new tokens late in two long documents
        dict(name="prompt_chunk", op="prompt", seqs=2, new_min=500, new_max=512, hist_max=33000,
             hq=32, hkv=4, rows=128, window=0, gate=True, pick=11),
        # one stream early in its answer: latency
        dict(name="streams_one", op="streams", streams=1, prefix=0, own_min=300, own_max=300, hq=32,
             hkv=4, rows=64, window=0, gate=True, pick=1),
        # 64 streams at the batched-decode benchmark's context, of which 8,192 rows are one prompt
        dict(name="streams_shared_8k", op="streams", streams=64, prefix=8192, own_min=1, own_max=512,
             hq=32, hkv=4, rows=64, window=0, gate=True, pick=2),
        # odd sizes: a prefix that ends inside a page, small pages, plain heads of an odd group
        dict(name="streams_odd", op="streams", streams=37, prefix=2055, own_min=1, own_max=1999,
             hq=10, hkv=2, rows=16, window=0, gate=False, pick=3),
        # samples of one long document
        dict(name="streams_shared_16k", op="streams", streams=128, prefix=16384, own_min=64,
             own_max=1024, hq=32, hkv=4, rows=128, window=0, gate=True, pick=4),
        # one reply sampled three more times, in a shallow model: latency
        dict(name="fork_reply", op="fork", sources=1, children=3, len_min=700, len_max=1000, pages=64,
             planes=8, hkv=4, rows=64, pick=6),
        # a batch of sampled continuations over the 40-layer model
        dict(name="fork_batch", op="fork", sources=8, children=64, len_min=1, len_max=1500, pages=320,
             planes=80, hkv=4, rows=64, pick=2),
        # a pool after many streams have come and gone, under half of its pages live
        dict(name="compact_pool", op="compact", streams=24, len_min=200, len_max=800, pages=512,
             planes=80, hkv=4, rows=64, pick=3),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "streams", "streams", "fork", "compact"])
    rows = rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([g for g in (1, 2, 4, 5, 7, 8, 16) if hkv * g <= 32])
    pick = rng.randrange(1 << 20)
    if op == "prompt":
        seqs = _log_int(rng, 1, 32)
        most = max(1, min(6000, int(math.sqrt(1.5e9 / (seqs * hq)))))  # the plain form's scores fit
        new_max = _log_int(rng, 1, most)
        hist = rng.choice([0, _log_int(rng, 1, max(1, min(20000, int(1.5e9 / (seqs * hq * new_max)))))])
        return dict(op=op, seqs=seqs, new_min=rng.randint(1, new_max), new_max=new_max,
                    hist_max=hist, hq=hq, hkv=hkv, rows=rows,
                    window=rng.choice([0, 0, _log_int(rng, 1, 2048)]), gate=rng.random() < 0.5,
                    pick=pick)
    if op == "streams":
        streams = _log_int(rng, 1, 128)
        prefix = rng.choice([0, _log_int(rng, 1, 16384)])
        own_max = _log_int(rng, 1, 4000 if streams < 64 else 1000)
        return dict(op=op, streams=streams, prefix=prefix, own_min=rng.randint(1, own_max),
                    own_max=own_max, hq=hq, hkv=hkv, rows=rows,
                    window=rng.choice([0, 0, _log_int(rng, 16, 8192)]), gate=rng.random() < 0.5,
                    pick=pick)
    planes = 2 * _log_int(rng, 1, 40)
    hkv = rng.choice([1, 2, 4])
    if op == "fork":
        sources = _log_int(rng, 1, 8)
        len_max = _log_int(rng, 1, 1500)
        children = _log_int(rng, 1, 64)
        pages = sources * -(-len_max // rows) + children + rng.randint(0, 40)
        return dict(op=op, sources=sources, children=children, len_min=rng.randint(1, len_max),
                    len_max=len_max, pages=pages, planes=planes, hkv=hkv, rows=rows, pick=pick)
    streams = _log_int(rng, 1, 24)
    len_max = _log_int(rng, 1, 800)
    pages = max(2, int(streams * -(-len_max // rows) * rng.uniform(1.0, 2.2)))
    pages = min(pages, 512 * 64 // rows)
    len_max = min(len_max, pages // streams * rows)
    return dict(op=op, streams=streams, len_min=rng.randint(1, max(1, len_max)),
                len_max=max(1, len_max), pages=max(pages, streams), planes=planes, hkv=hkv, rows=rows,
                pick=pick)


def _lengths(case):
    """The case's lengths (of the case alone, so that work() has them too): for prompts (new tokens,
    rows held) per sequence, for streams rows held, for the page operations rows held."""
    r = random.Random(case["pick"])
    if case["op"] == "prompt":
        new = [r.randint(case["new_min"], case["new_max"]) for _ in range(case["seqs"])]
        hist = [r.randint(case["hist_max"] // 2, case["hist_max"]) for _ in range(case["seqs"])]
        return new, [n + h for n, h in zip(new, hist)]
    if case["op"] == "streams":
        return [case["prefix"] + r.randint(case["own_min"], case["own_max"])
                for _ in range(case["streams"])]
    n = case["sources"] if case["op"] == "fork" else case["streams"]
    return [r.randint(case["len_min"], case["len_max"]) for _ in range(n)]


def work(case):
    hkv = case["hkv"]
    if case["op"] == "prompt":
        W = case["window"]
        new, kv = _lengths(case)
        pairs = rows = 0
        for n, m in zip(new, kv):
            first = m - n
            if W:
                full = max(0, min(n, first + n - W))  # tokens that see a whole window
                part = n - full
                pairs += full * W + part * (first + 1) + part * (part - 1) // 2
                rows += min(m, n + W - 1)
            else:
                pairs += n * first + n * (n + 1) // 2
                rows += m
        T = sum(new)
        return {"bytes": 2 * T * case["hq"] * D * 2 + rows * hkv * D * 2 * 2
                + (T * case["hq"] * 2 if case["gate"] else 0),
                "flops": 4 * D * case["hq"] * pairs}
    if case["op"] == "streams":
        kv, P, W = _lengths(case), case["prefix"], case["window"]
        low = [max(0, n - W) if W else 0 for n in kv]
        rows = max(0, P - min(low)) + sum(n - max(P, l) for n, l in zip(kv, low))
        return {"bytes": 2 * len(kv) * case["hq"] * D * 2 + rows * hkv * D * 2 * 2
                + (len(kv) * case["hq"] * 2 if case["gate"] else 0),
                "flops": 4 * D * case["hq"] * sum(n - l for n, l in zip(kv, low))}
    per_row = case["planes"] * hkv * D * 2
    R = case["rows"]
    if case["op"] == "fork":
        lens = _lengths(case)
        child = [lens[s] % R for s in _sources(case)]
        used = set(_sources(case))
        ints = 4 * (case["sources"] + case["children"]) * (1 + -(-case["len_max"] // R))
        return {"bytes": per_row * (sum(lens[s] % R for s in used) + sum(child)) + ints, "flops": 0}
    _, live = _scatter(case)
    n = len(live)
    moved = sum(1 for p in live if p >= n)
    return {"bytes": 2 * per_row * R * moved + 8 * case["pages"], "flops": 0}


def _sources(case):
    r = random.Random(case["pick"] + 1)
    return [r.randrange(case["sources"]) for _ in range(case["children"])]


def _scatter(case):
    """A pool's owners after use: each sequence's page ids, anywhere in the pool, and all of them."""
    R, r = case["rows"], random.Random(case["pick"] + 2)
    need = [-(-n // R) for n in _lengths(case)]
    ids = r.sample(range(case["pages"]), sum(need))
    at = [sum(need[:i]) for i in range(len(need) + 1)]
    return [ids[a:b] for a, b in zip(at, at[1:])], ids


# ---- inputs -----------------------------------------------------------------------------------

def _normal(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(torch.bfloat16)


def _table(owned, M):
    return torch.tensor([p + [-1] * (M - len(p)) for p in owned], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, hkv = case["rows"], case["hkv"]
    if case["op"] in ("prompt", "streams"):
        hq = case["hq"]
        if case["op"] == "prompt":
            new, kv = _lengths(case)
            shared = 0
        else:
            kv = _lengths(case)
            new = [1] * len(kv)
            shared = case["prefix"] // R  # whole pages; a page it ends in is copied per stream
        need = [-(-n // R) - shared for n in kv]
        total = shared + sum(need)
        ids = torch.randperm(total, generator=g, device="cuda").tolist()
        at = [shared + sum(need[:i]) for i in range(len(need) + 1)]
        table = _table([ids[:shared] + ids[a:b] for a, b in zip(at, at[1:])], max(need) + shared)
        k = _normal((total, hkv, R, D), g)
        v = _normal((total, hkv, R, D), g)
        part = case["prefix"] % R if case["op"] == "streams" else 0
        if part:  # the prefix's rows in the page that each stream has of its own are the same
            first = table[:, shared].long()
            k[first, :, :part] = k[first[:1], :, :part]
            v[first, :, :part] = v[first[:1], :, :part]
        T = sum(new)
        s = dict(case=case, k=k, v=v, table=table, q=_normal((T, hq, D), g),
                 kv_len=torch.tensor(kv, dtype=torch.int32, device="cuda"), scale=D ** -0.5,
                 gate=torch.nn.functional.softplus(_normal((T, hq), g)) if case["gate"] else None,
                 most_new=max(new), most_kv=max(kv),
                 cu=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32,
                                 device="cuda"))
        if own:  # the division of the work: made once per step, used by every layer of it
            from lagunalab_b200 import ops
            s["plan"] = (ops.prompt_plan(s["cu"], s["kv_len"], T, hq, hkv, R, window=case["window"])
                         if case["op"] == "prompt" else
                         ops.stream_plan(s["kv_len"], hq, hkv, R, prefix=case["prefix"],
                                         window=case["window"]))
        return s
    lens = _lengths(case)
    if case["op"] == "fork":
        M = -(-max(lens) // R)
        n = len(lens)
        need = [-(-m // R) for m in lens]
        ids = torch.randperm(case["pages"], generator=g, device="cuda")[:sum(need)].tolist()
        at = [sum(need[:i]) for i in range(n + 1)]
        owned = [ids[a:b] for a, b in zip(at, at[1:])] + [[]] * case["children"]
        lens = lens + [0] * case["children"]
    else:
        owned, ids = _scatter(case)
        M = max(len(p) for p in owned)
    refs = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    refs[torch.tensor(ids, device="cuda")] = 1
    s = dict(case=case, pool=_normal((case["planes"], case["pages"], hkv, R, D), g),
             table=_table(owned, M), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             refs=refs)
    s["table0"], s["refs0"] = s["table"].clone(), refs.clone()
    if case["op"] == "fork":
        s["src"] = torch.tensor(_sources(case), dtype=torch.int32, device="cuda")
        s["dst"] = torch.arange(case["sources"], case["sources"] + case["children"],
                                dtype=torch.int32, device="cuda")
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if op == "prompt":
        if own:
            from lagunalab_b200 import ops
            return ops.prompt_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], s["scale"],
                                        gate=s["gate"])
        return _attend(s, s["most_new"], 0)
    if op == "streams":
        if own:
            from lagunalab_b200 import ops
            return ops.stream_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], s["scale"],
                                        gate=s["gate"])
        return _attend(s, 1, s["case"]["prefix"])
    if op == "fork":  # the children of the last round go, new ones come
        if own:
            from lagunalab_b200 import ops
            ops.pages_free(s["table"], s["lens"], s["refs"], s["dst"])
            ops.pages_fork(s["pool"], s["table"], s["lens"], s["refs"], s["src"], s["dst"])
        else:
            _free(s["table"], s["lens"], s["refs"], s["dst"])
            _fork(s["pool"], s["table"], s["lens"], s["refs"], s["src"], s["dst"])
    else:  # the same scattered pool each time: only table and counts are put back
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        if own:
            from lagunalab_b200 import ops
            ops.pages_compact(s["pool"], s["table"], s["refs"])
        else:
            _compact(s["pool"], s["table"], s["refs"])
    return dict(pool=s["pool"], table=s["table"], lens=s["lens"], refs=s["refs"])


def _rows(pages, table, n):
    """Rows [0, n) of every sequence, in 32 bits: [B, Hkv, n, D]."""
    x = pages[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)  # [B, Hkv, M, R, D]
    return x.flatten(2, 3)[:, :, :n].float()


def _attend(s, most, prefix):
    q, cu, kv = s["q"], s["cu"].long(), s["kv_len"].long()
    W, n = s["case"]["window"], s["most_kv"]
    B, (T, hq, _), hkv = kv.numel(), q.shape, s["k"].shape[1]
    k, v = _rows(s["k"], s["table"], n), _rows(s["v"], s["table"], n)
    new = cu[1:] - cu[:-1]
    i = torch.arange(most, device=q.device)
    at = (cu[:-1, None] + i).clamp(max=T - 1)  # [B, most]
    qs = q[at].float().view(B, most, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4)
    sc = torch.matmul(qs.reshape(B, hkv, -1, D), k.transpose(2, 3)) * s["scale"]
    sc = sc.view(B, hkv, hq // hkv, most, n)
    p = (kv - new)[:, None] + i  # positions [B, most]
    j = torch.arange(n, device=q.device)
    seen = (j <= p[..., None]) & (i < new[:, None])[..., None]
    if W:
        seen &= j > p[..., None] - W
    seen = seen[:, None, None]
    sc = sc.masked_fill(~seen, -math.inf)
    e = (sc - sc.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    den = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, hkv, -1, n), v).view(B, hkv, hq // hkv, most, D)
    o = o / den.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, hq, D)[i < new[:, None]]  # [T, Hq, D]
    o = o.to(torch.bfloat16)
    return o if s["gate"] is None else (o.float() * s["gate"].float()[..., None]).to(torch.bfloat16)


def _free(table, lens, refs, ids):
    rows = table[ids.long()]
    refs.sub_(torch.bincount(rows[rows >= 0].long(), minlength=refs.numel()).to(torch.int32))
    table[ids.long()] = -1
    lens[ids.long()] = 0


def _fork(pool, table, lens, refs, src, dst):
    R, M = pool.shape[3], table.shape[1]
    src, dst = src.long(), dst.long()
    whole, part = lens[src].long() // R, lens[src].long() % R
    m = torch.arange(M, device=table.device)
    rows = torch.where(m < whole[:, None], table[src], -1)
    free = (refs == 0).nonzero().view(-1)
    refs.add_(torch.bincount(rows[rows >= 0].long(), minlength=refs.numel()).to(torch.int32))
    need = part > 0
    new = free[:int(need.sum())]
    old = table[src[need], whole[need]].long()
    rows[need.nonzero().view(-1), whole[need]] = new.to(torch.int32)
    refs[new] = 1
    table[dst] = rows
    lens[dst] = lens[src]
    r = torch.arange(R, device=table.device)
    c, r = (r < part[need][:, None]).nonzero(as_tuple=True)  # (child, row) pairs
    pool[:, new[c], :, r] = pool[:, old[c], :, r]


def _compact(pool, table, refs):
    live = refs > 0
    n = int(live.sum())
    i = torch.arange(refs.numel(), device=refs.device)
    to, at = i[~live & (i < n)], i[live & (i >= n)]
    name = i.clone()
    name[at] = to
    pool[:, to] = pool[:, at]
    table.copy_(torch.where(table >= 0, name[table.clamp(min=0).long()].to(torch.int32), -1))
    refs[to] = refs[at]
    refs[at] = 0


# ---- the operators' definition in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("fork", "compact"):
        # rows are only moved: what the plain form says of whole numbers is exact; the pool's rows
        # as the definition moves them, page by page
        return dict(pool=_moved(s), table=None, lens=None, refs=None)
    if work(case)["flops"] > 4e12:
        return None
    q, W, hkv, R = s["q"].double(), case["window"], case["hkv"], case["rows"]
    G = case["hq"] // hkv
    out = torch.zeros_like(q)
    cu, kv = s["cu"].tolist(), s["kv_len"].tolist()
    for b in range(len(kv)):
        ids = s["table"][b, :-(-kv[b] // R)].long()
        k = s["k"][ids].transpose(0, 1).reshape(hkv, -1, D)[:, :kv[b]].double()
        v = s["v"][ids].transpose(0, 1).reshape(hkv, -1, D)[:, :kv[b]].double()
        n = cu[b + 1] - cu[b]
        for a in range(0, n, 1024):
            z = min(n, a + 1024)
            pos = torch.arange(kv[b] - n + a, kv[b] - n + z, device=q.device)
            far = pos[:, None] - torch.arange(kv[b], device=q.device)  # how far back a key lies
            hide = (far < 0) | (far >= W) if W else far < 0
            for h in range(hkv):
                for g in range(G):
                    x = q[cu[b] + a:cu[b] + z, h * G + g] @ k[h].T * s["scale"]
                    x[hide] = -math.inf
                    lse = torch.logsumexp(x, -1, keepdim=True)
                    out[cu[b] + a:cu[b] + z, h * G + g] = (x - lse).exp() @ v[h]
    return out if s["gate"] is None else out * s["gate"].double()[..., None]


def _moved(s):
    case, pool, R = s["case"], s["pool"].clone(), s["case"]["rows"]
    refs, table, lens = s["refs"].tolist(), s["table"].tolist(), s["lens"].tolist()
    if case["op"] == "fork":
        free = [p for p, r in enumerate(refs) if r == 0]
        for a in s["src"].tolist():
            part = lens[a] % R
            if part:
                pool[:, free.pop(0), :, :part] = s["pool"][:, table[a][lens[a] // R], :, :part]
        return pool
    n = sum(r > 0 for r in refs)
    holes = [p for p in range(n) if refs[p] == 0]
    for to, at in zip(holes, [p for p in range(n, len(refs)) if refs[p] > 0]):
        pool[:, to] = s["pool"][:, at]
    return pool
