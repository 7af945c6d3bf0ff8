"""The router's balance loss and the gradient of its logits against 64 bits.

Bounds: an fp32 score is off by at most 2^-20 relative (exponential of an argument up to 16 rounded to 2^-24 of it, a
division's approximation, a sum of up to 256 terms); T tokens' sum adds (T / 16 + 24) 2^-24 (16 warps a CTA add
their tokens one by one). A gradient is a sum of products of scores, each term within 2^-17 of the terms'
absolute sum."""
import pytest
import torch

from lagunalab_b200 import ops

pytestmark = pytest.mark.gpu


def make(T, E, k, seed=0, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(T, E, generator=g, device="cuda") * std
    inds = logits.topk(k, 1).indices.to(torch.int32)
    return logits, inds, torch.randn(T, k, generator=g, device="cuda"), \
        torch.rand(T, generator=g, device="cuda") > 0.3


def scores(z, fn):
    return torch.softmax(z, 1) if fn == "softmax" else torch.sigmoid(z)


def balance64(logits, inds, fn, mask):
    keep = torch.ones(logits.shape[0], dtype=torch.bool) if mask is None else mask.cpu()
    z, i = logits.cpu().double()[keep], inds.cpu().long()[keep]
    E = z.shape[1]
    s = scores(z, fn)
    probs = (s / s.sum(1, keepdim=True)).sum(0) / max(z.shape[0], 1)
    i = i.flatten()
    counts = torch.bincount(i[(i >= 0) & (i < E)], minlength=E)
    loss = E * (counts.double() @ probs) / max(int(counts.sum()), 1)
    return loss, counts, probs, z.shape[0]


def check_balance(logits, inds, fn, mask):
    loss, counts, probs, n = balance64(logits, inds, fn, mask)
    got = ops.router_balance(logits, inds, fn, mask)
    assert torch.equal(got.counts.cpu().long(), counts) and int(got.tokens) == n
    rel = 2.0 ** -20 + (logits.shape[0] / 16 + 24) * 2.0 ** -24
    assert ((got.probs.cpu().double() - probs).abs() <= rel * probs + 1e-37).all()
    assert abs(float(got.loss) - float(loss)) <= (rel + 2.0 ** -18) * float(loss)
    return got


def grad64(logits, inds, dw, norm, fn, mask, weight):
    z = logits.cpu().double().requires_grad_()
    T, E = z.shape
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
    i = inds.cpu().long()
    ok = (i >= 0) & (i < E)
    s = scores(z, fn)
    w = torch.where(ok, s.gather(1, i.clamp(0, E - 1)), 0.0)
    if norm:
        w = w / torch.where(ok.any(1, keepdim=True), w.sum(1, keepdim=True), 1.0)
    total = (w.sum() + z.sum()) * 0
    if dw is not None:
        total = total + (w * dw.cpu().double())[keep].sum()
    if weight is not None:
        loss, counts, _, n = balance64(logits, inds, fn, mask)
        q = (s / s.sum(1, keepdim=True))[keep]
        total = total + weight * E * (q.sum(0) / max(n, 1)) @ counts.double() / max(int(counts.sum()), 1)
    total.backward()
    return z.grad


def check_grad(logits, inds, dw, norm, fn, mask, weight):
    bal = None if weight is None else ops.router_balance(logits, inds, fn, mask)
    got = ops.router_grad(logits, inds, dw, norm, fn, bal, weight or 0.0, mask).cpu().double()
    want = grad64(logits, inds, dw, norm, fn, mask, weight)
    # the terms' absolute sum: each |ds| is at most (|dw| + sum |dw| w) / sum of the picks' scores
    T, E = want.shape
    s = scores(logits.cpu().double(), fn)
    i = inds.cpu().long()
    p = torch.where((i >= 0) & (i < E), s.gather(1, i.clamp(0, E - 1)), 0.0)
    mass = torch.zeros(T, 1, dtype=torch.float64)
    if dw is not None:
        most = 2 * dw.cpu().double().abs().sum(1, keepdim=True)
        mass = mass + (most / p.sum(1, keepdim=True).clamp(min=1e-300) if norm else most)
    if weight is not None:
        share = bal.counts.cpu().double()
        share = weight * E * share / max(float(share.sum()), 1) / max(int(bal.tokens), 1)
        mass = mass + 2 * share.max() / (1.0 if fn == "softmax" else s.sum(1, keepdim=True))
    bound = 2.0 ** -17 * mass * (s if fn == "softmax" else s * (1 - s)) + 1e-37
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
    assert (got[~keep] == 0).all()
    assert ((got - want).abs()[keep] <= bound[keep]).all()
    return got


SIZES = [(1, 1, 1), (1, 128, 8), (3, 5, 5), (16, 64, 8), (64, 32, 4), (65, 33, 2), (1000, 129, 8),
         (4097, 256, 32), (777, 65, 3)]


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
@pytest.mark.parametrize("masked", [False, True])
def test_balance(T, E, k, fn, masked):
    logits, inds, _, mask = make(T, E, k, T + E)
    check_balance(logits, inds, fn, mask if masked else None)


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
@pytest.mark.parametrize("norm,with_dw,weight", [(True, True, None), (False, True, 0.01), (True, True, 0.5),
                                                 (True, False, 1.0)])
def test_grad(T, E, k, fn, norm, with_dw, weight):
    logits, inds, dw, mask = make(T, E, k, T + E)
    check_grad(logits, inds, dw if with_dw else None, norm, fn, mask if T % 2 else None, weight)


def test_even_routing_has_loss_one():
    logits = torch.zeros(64, 16, device="cuda")
    inds = (torch.arange(64, device="cuda")[:, None] * 2 + torch.arange(2, device="cuda")) % 16
    got = ops.router_balance(logits, inds.to(torch.int32), "softmax")
    assert float(got.loss) == 1 and (got.counts == 8).all()


@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
def test_masked_rows_may_hold_anything(fn):
    logits, inds, dw, mask = make(300, 40, 4)
    want = ops.router_balance(logits, inds, fn, mask)
    gw = ops.router_grad(logits, inds, dw, True, fn, want, 0.1, mask)
    logits[~mask] = float("nan")
    logits[(~mask).nonzero()[::2, 0]] = float("inf")
    inds[~mask] = 2 ** 31 - 1
    dw[~mask] = float("nan")
    got = ops.router_balance(logits, inds, fn, mask)
    gg = ops.router_grad(logits, inds, dw, True, fn, got, 0.1, mask)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(gw, gg)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_no_token_is_kept(T):
    logits, inds, dw, _ = make(T, 40, 4)
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    got = ops.router_balance(logits, inds, mask=mask)
    assert all((t == 0).all() for t in got)
    assert (ops.router_grad(logits, inds, dw, balance=got, balance_weight=1.0, mask=mask) == 0).all()


def test_no_tokens():
    logits, inds, dw, _ = make(4, 40, 4)
    got = ops.router_balance(logits[:0], inds[:0])
    assert all((t == 0).all() for t in got)
    assert ops.router_grad(logits[:0], inds[:0], dw[:0]).shape == (0, 40)


@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
def test_picks_outside_the_experts_and_picked_twice(fn):
    logits, inds, dw, mask = make(90, 20, 6)
    inds[::3, 1] = -1
    inds[1::3, 2] = 20
    inds[2::3, 3:] = inds[2::3, :1]  # the same expert four times
    inds[5] = -1
    check_balance(logits, inds, fn, mask)
    for norm in (True, False):
        check_grad(logits, inds, dw, norm, fn, None, 0.3)


@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
def test_far_logits(fn):
    """Scores near 0 and 1, and an expert ruled out by -inf."""
    logits, inds, dw, _ = make(64, 48, 4, std=12.0)
    logits[:, 7] = float("-inf")
    inds = logits.topk(4, 1).indices.to(torch.int32)
    got = ops.router_balance(logits, inds, fn)
    loss, counts, probs, _ = balance64(logits, inds, fn, None)
    assert torch.equal(got.counts.cpu().long(), counts) and float(got.probs[7]) == 0
    # arguments up to 100: exp2's is rounded to 2^-24 of 144
    assert ((got.probs.cpu().double() - probs).abs() <= 2.0 ** -16 * probs + 1e-37).all()
    g = ops.router_grad(logits, inds, dw, True, fn, got, 0.1)
    assert g.isfinite().all() and (g[:, 7] == 0).all()


@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
def test_weights_of_one_pick_have_no_gradient(fn):
    logits, inds, dw, _ = make(300, 20, 1)
    assert (ops.router_grad(logits, inds, dw, True, fn) == 0).all()
    logits, inds, dw, _ = make(300, 1, 1)  # one expert: its share is 1 whatever its logit
    bal = ops.router_balance(logits, inds, "softmax")
    assert (ops.router_grad(logits, inds, dw, False, "softmax", bal, 0.3) == 0).all()


@pytest.mark.parametrize("E,k", [(7, 6), (60, 4), (128, 8), (250, 20)])
@pytest.mark.parametrize("weight", [None, 0.5])
@pytest.mark.parametrize("norm,fn", [(True, "sigmoid"), (True, "softmax"), (False, "softmax")])
def test_one_share_near_one(E, k, weight, norm, fn):
    """A pick whose share is nearly all of it. Each gradient is a score times a sum of differences from the largest
    share's value; a score is off by 2^-17 relative (arguments up to 40), the sums' other roundings by less: 2^-15 of
    the differences' absolute sum. Differences from the mean itself would be off by 2^-24 of the values."""
    logits, inds, dw, _ = make(200, E, k)
    if fn == "sigmoid":
        logits = logits - 12
    logits[torch.arange(200, device="cuda"), inds[:, 0].long()] += 12
    bal = None if weight is None else ops.router_balance(logits, inds, fn)
    got = ops.router_grad(logits, inds, dw, norm, fn, bal, weight or 0.0).cpu().double()
    want = grad64(logits, inds, dw, norm, fn, None, weight)
    s, i, d = scores(logits.cpu().double(), fn), inds.cpu().long(), dw.cpu().double()
    tail = s if fn == "softmax" else torch.sigmoid(-logits.cpu().double()) * s
    total = s.sum(1, keepdim=True)
    if norm:
        p = s.gather(1, i)
        w, d = p / p.sum(1, keepdim=True), (d - d[:, :1]).abs()
        part = torch.zeros_like(s).scatter_(1, i, (d + (w * d).sum(1, keepdim=True)) / p.sum(1, keepdim=True))
        h = torch.zeros_like(s)
    else:
        part, h = torch.zeros_like(s), torch.zeros_like(s).scatter_(1, i, d)
    dq = torch.zeros(E, dtype=torch.float64)
    if weight is not None:
        dq = weight * E * bal.counts.cpu().double() / int(bal.counts.sum()) / 200
    top = s.argmax(1, keepdim=True)
    own = 2.0 ** -22 * dq + 2.0 ** -23 * h.abs()  # of dq and of its sum with dw; none for the largest share
    own = (own + own.gather(1, top)).scatter(1, top, 0.0)
    h = h + dq
    h = (h - h.gather(1, top)).abs()
    both = [a + (s * a).sum(1, keepdim=True) / total for a in (h, own)]
    if fn == "sigmoid":
        both = [a / total for a in both]
    # the formula's own roundings: an expert that is not picked has exactly 0 where 64 bits leave a sum that cancels, off
    # by 2^-53 of each of up to 2 k terms of up to 2 |dw| / sum s (sum s > 0.5 here) and their own few roundings
    exact = 2.0 ** -47 * dw.cpu().double().abs().sum(1, keepdim=True)
    assert ((got - want).abs() <= tail * (2.0 ** -15 * (part + both[0]) + 2 * both[1] + exact) + 1e-37).all()


def test_strides_streams_and_graphs():
    logits, inds, dw, mask = make(500, 40, 4)
    bal = ops.router_balance(logits, inds, mask=mask)
    want = tuple(bal) + (ops.router_grad(logits, inds, dw, balance=bal, balance_weight=0.1, mask=mask),)

    def run(lg, ii, d, m):
        b = ops.router_balance(lg, ii, mask=m)
        return tuple(b) + (ops.router_grad(lg, ii, d, balance=b, balance_weight=0.1, mask=m),)

    got = run(logits.t().contiguous().t(), torch.cat([inds, inds], 1)[:, :4], dw.t().contiguous().t(),
              torch.stack([mask, mask], 1)[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    both = []
    for st in side:
        with torch.cuda.stream(st):
            both.append(run(logits, inds, dw, mask))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in both for a, b in zip(want, r))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run(logits, inds, dw, mask)
        graphs.append((gr, out))
    new = make(500, 40, 4, seed=5)
    for a, b in zip((logits, inds, dw, mask), new):
        a.copy_(b)
    for gr, _ in graphs:
        gr.replay()
    want = run(*new)
    assert all(torch.equal(a, b) for _, r in graphs for a, b in zip(want, r))


def test_repeatable():
    logits, inds, dw, _ = make(20000, 128, 8)
    a, b = (ops.router_balance(logits, inds) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals():
    logits, inds, dw, mask = make(8, 16, 2)
    bal = ops.router_balance(logits, inds)
    bad = [dict(logits=logits.bfloat16()), dict(logits=logits[0]), dict(inds=inds.long()), dict(inds=inds[:3]),
           dict(score_fn="relu"), dict(mask=mask[:3]), dict(mask=mask.int()), dict(logits=logits.cpu()),
           dict(inds=inds.cpu()), dict(inds=inds[:, :0]), dict(inds=inds.repeat(1, 17)),
           dict(logits=torch.zeros(8, 257, device="cuda"))]
    base = dict(logits=logits, inds=inds)
    for b in bad:
        with pytest.raises(ValueError):
            ops.router_balance(**{**base, **b})
        with pytest.raises(ValueError):
            ops.router_grad(**{**base, "dw": dw, **b})
    for b in (dict(), dict(dw=dw[:, :1]), dict(dw=dw.half()), dict(balance=ops.router_balance(logits[:, :9], inds)),
              dict(dw=dw, balance=bal._replace(tokens=bal.counts))):
        with pytest.raises(ValueError):
            ops.router_grad(**base, **b)
