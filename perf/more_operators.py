"""The operators that fit a model again after pruning or quantisation, as cases to measure: the head's
cross entropy without its logits (one target a token, or the ids and weights of a reference's largest
probabilities) and its gradient, the router's balance loss with its counts, and the router's gradient.
Each case runs in a plain form of elementary torch operations or, where ``own`` is true, through
``lagunalab_b200.ops``.

Layouts: hidden rows x bf16 [T, H]; a head bf16 [V, H], or 4-bit words int32 [V, H / 8] (code i of a word
in bits 4 i) with bf16 scales and biases [V, H / 64] that stand for the weights
bf16(scale * code + bias); target ids int32 [T] or [T, K], negative ones left out; router logits fp32
[T, E], picks int32 [T, k].
"""
import math
import random

import torch

own = False


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the test decoder's head: latency
        dict(name="loss_tiny", op="loss", T=64, V=512, H=256, bits=16, K=1, skip=0.0),
        # the tokens of one short reply scored by the pruned model's 4-bit head
        dict(name="loss_reply", op="loss", T=37, V=100352, H=2048, bits=4, K=1, skip=0.1),
        # a prefill chunk of a session against the reference's 64 stored probabilities
        dict(name="loss_chunk", op="loss", T=2048, V=100352, H=2048, bits=4, K=64, skip=0.0),
        # a batch of sequences with a bf16 head, the users' turns left out
        dict(name="loss_8k", op="loss", T=8192, V=100352, H=2048, bits=16, K=1, skip=0.4),
        # odd sizes: a vocabulary and a token count that end inside a tile
        dict(name="grad_odd", op="grad", T=301, V=32003, H=1024, bits=16, K=5, skip=0.2),
        # hidden rows' gradient through the frozen 4-bit head, against stored probabilities
        dict(name="grad_frozen", op="grad", T=1000, V=100352, H=2048, bits=4, K=64, skip=0.0),
        # a training step's head: both gradients
        dict(name="grad_8k", op="grad", T=8192, V=100352, H=2048, bits=16, K=1, skip=0.4),
        # one step of the batched decode's 64 streams: latency
        dict(name="balance_64", op="balance", T=64, E=128, k=8, score="sigmoid", skip=0.0),
        # the expert-parallel benchmark's prefill
        dict(name="balance_32k", op="balance", T=32768, E=128, k=8, score="sigmoid", skip=0.1),
        # the prefill block's router
        dict(name="router_4k", op="router", T=4096, E=128, k=8, score="softmax", skip=0.0, norm=True,
             balance=True),
        # the pruned model's router over a long batch with padding
        dict(name="router_32k", op="router", T=32768, E=64, k=8, score="sigmoid", skip=0.1, norm=True,
             balance=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["loss", "loss", "grad", "grad", "balance", "router"])
    if op in ("loss", "grad"):
        bits = rng.choice([4, 16])
        H = 64 * _log_int(rng, 1, 40) if bits == 4 else 8 * _log_int(rng, 8, 320)
        V = _log_int(rng, 100, 100352)
        T = _log_int(rng, 1, min(8192, max(1, int(1.6e12 / (V * H)))))
        K = rng.choice([1, 1, _log_int(rng, 1, 64)])
        return dict(op=op, T=T, V=V, H=H, bits=bits, K=K, skip=rng.choice([0.0, 0.3, 0.9]))
    E = _log_int(rng, 4, 256)
    d = dict(op=op, T=_log_int(rng, 1, 32768), E=E, k=rng.randint(1, min(E, 12)),
             score=rng.choice(["sigmoid", "softmax"]), skip=rng.choice([0.0, 0.0, 0.4]))
    if op == "router":
        d.update(norm=rng.random() < 0.7, balance=rng.random() < 0.7)
    return d


def work(case):
    T = case["T"]
    if case["op"] in ("balance", "router"):
        E, k = case["E"], case["k"]
        mask = T if case["skip"] else 0
        if case["op"] == "balance":
            return {"bytes": 4 * T * (E + k) + mask + 8 * E, "flops": 6 * T * E}
        return {"bytes": 4 * T * (2 * E + 2 * k) + mask + 4 * E, "flops": 10 * T * E}
    V, H, K = case["V"], case["H"], case["K"]
    head = V * H * 2 if case["bits"] == 16 else V * H // 2 + V * (H // 64) * 4
    inputs = 2 * T * H + head + T * K * (4 if K == 1 else 8)
    if case["op"] == "loss":
        return {"bytes": inputs + 8 * T, "flops": 2 * T * V * H}
    dw = case["bits"] == 16
    return {"bytes": inputs + 8 * T + 2 * T * H + (2 * V * H if dw else 0),
            "flops": (6 if dw else 4) * T * V * H}


# ---- inputs -----------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    T = case["T"]
    if case["op"] in ("balance", "router"):
        return _prepare_router(case, g)
    V, H, K = case["V"], case["H"], case["K"]
    if case["bits"] == 16:
        head = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16) * 0.02
    else:  # codes of all values, weights of about the same spread around zero
        words = torch.randint(-2 ** 31, 2 ** 31, (V, H // 8), generator=g, device="cuda",
                              dtype=torch.int32)
        scales = (torch.rand(V, H // 64, generator=g, device="cuda") * 0.002 + 0.0035).bfloat16()
        head = (words, scales, (-7.5 * scales.float()).bfloat16())
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn(T, H, generator=g, device="cuda")
    # a trained model's rows lean towards their next token, some far and some not at all
    first = ids[:, 0].long()
    row = head[first].float() if case["bits"] == 16 else _dequant(tuple(m[first] for m in head))
    lean = torch.rand(T, 1, generator=g, device="cuda") * 12.0
    x = (x + lean * row / row.norm(dim=1, keepdim=True).clamp(min=1e-6)).bfloat16()
    weights = None
    if K > 1:  # probabilities in falling order that sum to a little under one
        weights = torch.softmax(torch.randn(T, K, generator=g, device="cuda").mul(2.0)
                                .sort(dim=1, descending=True).values, -1) * 0.97
    if case["skip"]:
        out = torch.rand(T, generator=g, device="cuda") < case["skip"]
        ids[out] = -1
    s = dict(case=case, x=x, head=head, ids=ids[:, 0].contiguous() if K == 1 else ids,
             weights=weights)
    if case["op"] == "grad":  # a mean over the tokens that count; the loss's own pass came before
        n = int((ids[:, 0] >= 0).sum())
        s["g"] = torch.full((T,), 1.0 / max(n, 1), device="cuda")
        s["lse"] = torch.empty(T, device="cuda")
        W = _weights(head)
        for a in range(0, T, 1024):
            s["lse"][a:a + 1024] = torch.logsumexp(x[a:a + 1024].float() @ W.t(), -1)
    return s


def _prepare_router(case, g):
    T, E, k = case["T"], case["E"], case["k"]
    popular = torch.randn(E, generator=g, device="cuda") * 0.7  # some experts are liked by most
    logits = torch.randn(T, E, generator=g, device="cuda") * 1.5 + popular
    inds = logits.topk(k, dim=1).indices.to(torch.int32)
    mask = None
    if case["skip"]:
        mask = torch.rand(T, generator=g, device="cuda") >= case["skip"]
    s = dict(case=case, logits=logits, inds=inds, mask=mask)
    if case["op"] == "router":
        s["dw"] = torch.randn(T, k, generator=g, device="cuda") / T
        if case["balance"]:  # what the balance loss's own pass gave
            keep = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
            s["counts"] = torch.bincount(inds[keep].long().view(-1), minlength=E).to(torch.int32)
            s["tokens"] = keep.sum().view(1).to(torch.int32)
            s["weight"] = 0.01
            if own:
                from lagunalab_b200 import ops
                s["stats"] = ops.router_balance(logits, inds, case["score"], mask)
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from lagunalab_b200 import ops
        if op == "loss":
            return ops.head_loss(s["x"], s["head"], s["ids"], s["weights"])
        if op == "grad":
            return ops.head_loss_grad(s["x"], s["head"], s["ids"], s["lse"], s["g"], s["weights"],
                                      dw=case["bits"] == 16)
        if op == "balance":
            return tuple(ops.router_balance(s["logits"], s["inds"], case["score"], s["mask"]))
        return ops.router_grad(s["logits"], s["inds"], s["dw"], case["norm"], case["score"],
                               s.get("stats"), s.get("weight", 0.0), s["mask"])
    if op == "loss":
        return _loss(s)
    if op == "grad":
        return _grad(s)
    return _balance(s) if op == "balance" else _router(s)


def _dequant(mat):
    """The bf16 weights of a 4-bit head, in 32 bits."""
    words, scales, biases = mat
    shift = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    codes = ((words[..., None] >> shift) & 15).flatten(-2).float()
    codes = codes.view(*scales.shape, 64)
    return (codes * scales.float()[..., None] + biases.float()[..., None]).flatten(-2) \
        .bfloat16().float()


def _weights(head):
    return _dequant(head) if isinstance(head, tuple) else head.float()


def _targets(s):
    """Ids [T, K] (64 bits, left-out ones at 0) and their weights [T, K] (0 where left out)."""
    ids = s["ids"].view(s["case"]["T"], -1).long()
    w = torch.ones_like(ids, dtype=torch.float32) if s["weights"] is None else s["weights"]
    return ids.clamp(min=0), torch.where(ids >= 0, w, 0.0)


def _loss(s):
    ids, w = _targets(s)
    z = s["x"].float() @ _weights(s["head"]).t()
    top = z.amax(1, keepdim=True)
    lse = top + (z - top).exp().sum(1, keepdim=True).log()
    return (w * (lse - z.gather(1, ids))).sum(1), lse.view(-1)


def _grad(s):
    ids, w = _targets(s)
    x, W = s["x"].float(), _weights(s["head"])
    p = ((x @ W.t()) - s["lse"][:, None]).exp()
    dz = p.mul_(w.sum(1, keepdim=True)).scatter_add_(1, ids, -w).mul_(s["g"][:, None])
    dx = (dz @ W).bfloat16()
    return dx, (dz.t() @ x).bfloat16() if s["case"]["bits"] == 16 else None


def _scores(logits, score):
    """(scores as the router takes them, the same divided by their sum)"""
    if score == "softmax":
        e = (logits - logits.amax(1, keepdim=True)).exp()
        p = e / e.sum(1, keepdim=True)
        return p, p
    p = 1.0 / (1.0 + (-logits).exp())
    return p, p / p.sum(1, keepdim=True)


def _keep(s):
    T = s["case"]["T"]
    return torch.ones(T, dtype=torch.bool, device=s["logits"].device) if s["mask"] is None \
        else s["mask"]


def _balance(s):
    E, keep = s["case"]["E"], _keep(s)
    _, q = _scores(s["logits"], s["case"]["score"])
    n = keep.sum()
    probs = torch.where(keep[:, None], q, 0.0).sum(0) / n.clamp(min=1)
    hit = torch.zeros(E + 1, dtype=torch.int32, device=q.device)  # the last: tokens left out
    at = torch.where(keep[:, None], s["inds"], E).long().view(-1)
    counts = hit.index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:E]
    loss = E * (counts * probs).sum() / counts.sum().clamp(min=1)
    return loss.view(1), counts, probs, n.view(1).to(torch.int32)


def _router(s):
    case, keep = s["case"], _keep(s)
    sc, q = _scores(s["logits"], case["score"])
    i = s["inds"].long()
    dw = s["dw"]
    if case["norm"]:
        picked = sc.gather(1, i)
        total = picked.sum(1, keepdim=True)
        dw = (dw - (dw * picked).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(sc).scatter_add_(1, i, dw)
    if case["balance"]:
        share = s["counts"].float() / s["counts"].sum().clamp(min=1)
        dq = s["weight"] * case["E"] * share / s["tokens"].clamp(min=1)
        dq = dq - (q * dq).sum(1, keepdim=True)
        ds = ds + (dq if case["score"] == "softmax" else dq / sc.sum(1, keepdim=True))
    if case["score"] == "softmax":
        dl = sc * (ds - (sc * ds).sum(1, keepdim=True))
    else:
        dl = ds * sc * (1.0 - sc)
    return torch.where(keep[:, None], dl, 0.0)


# ---- the operators' definition in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "balance":
        return _exact_balance(s)
    if case["op"] == "router":
        return _exact_router(s)
    T, K, x = case["T"], case["K"], s["x"].double()
    W = s["head"].double() if case["bits"] == 16 else _codes64(s["head"])
    ids = s["ids"].view(T, K)
    w = (torch.ones(T, K, device="cuda") if s["weights"] is None else s["weights"]).double()
    w = w * (ids >= 0)
    at = ids.long() * (ids >= 0)
    step = max(1, int(2e9 / (8 * case["V"])))
    loss, lse = torch.empty(2, T, dtype=torch.float64, device="cuda")
    dx = torch.empty_like(x)
    dW = torch.zeros_like(W) if case["bits"] == 16 and case["op"] == "grad" else None
    for a in range(0, T, step):
        b = min(T, a + step)
        z = x[a:b] @ W.T
        if case["op"] == "loss":
            lse[a:b] = torch.logsumexp(z, 1)
            loss[a:b] = ((lse[a:b, None] - z.gather(1, at[a:b])) * w[a:b]).sum(1)
            continue
        dz = torch.exp(z - s["lse"][a:b, None].double()) * w[a:b].sum(1)[:, None]
        for j in range(K):
            r = torch.arange(b - a, device="cuda")
            dz[r, at[a:b, j]] -= w[a:b, j]
        dz *= s["g"][a:b, None].double()
        dx[a:b] = dz @ W
        if dW is not None:
            dW.addmm_(dz.T, x[a:b])
    return (loss, lse) if case["op"] == "loss" else (dx, dW)


def _codes64(head):
    words, scales, biases = head
    cols = [(words >> (4 * i)).bitwise_and(15).double() for i in range(8)]
    codes = torch.stack(cols, dim=2).view(words.shape[0], -1)
    W = codes * scales.double().repeat_interleave(64, 1) + biases.double().repeat_interleave(64, 1)
    return W.float().to(torch.bfloat16).double()  # scale * code + bias has at most 20 bits


def _exact_balance(s):
    case = s["case"]
    keep = _keep(s)
    z = s["logits"][keep].double()
    q = torch.softmax(z, 1) if case["score"] == "softmax" else torch.sigmoid(z)
    q = q / q.sum(1, keepdim=True)
    n = z.shape[0]
    probs = q.sum(0) / max(n, 1)
    picks = s["inds"][keep].flatten().tolist()
    counts = [0] * case["E"]
    for e in picks:
        counts[e] += 1
    f = torch.tensor(counts, dtype=torch.float64, device="cuda") / max(len(picks), 1)
    return (case["E"] * (f @ probs)).view(1), None, probs, None


def _exact_router(s):
    """By automatic differentiation of sum(dw * w) + weight * balance loss."""
    case, keep = s["case"], _keep(s)
    z = s["logits"].double().requires_grad_()
    sc = torch.softmax(z, 1) if case["score"] == "softmax" else torch.sigmoid(z)
    w = sc.gather(1, s["inds"].long())
    if case["norm"]:
        w = w / w.sum(1, keepdim=True)
    total = (w * s["dw"].double())[keep].sum()
    if case["balance"]:
        q = (sc / sc.sum(1, keepdim=True))[keep]
        f = s["counts"].double() / s["counts"].sum().clamp(min=1)
        total = total + s["weight"] * case["E"] * (q.sum(0) / max(q.shape[0], 1) * f).sum()
    if z.shape[0] and total.requires_grad:
        total.backward()
    return z.grad if z.grad is not None else torch.zeros_like(z)
