"""The operators together, as a step that fits a pruned model's head and a router to a reference again: the head's
loss against stored probabilities and its gradients, the routing, its balance loss and its gradient; held to automatic
differentiation in 64 bits of the same step."""
import pytest
import torch

from lagunalab_b200 import ops

pytestmark = pytest.mark.gpu


def _step(x, head, ids, p, g, gate, bias, dw, k, mask, weight):
    loss, lse = ops.head_loss(x, head, ids, p)
    dx, dhead = ops.head_loss_grad(x, head, ids, lse, g, p)
    inds, w, logits = ops.router_topk(x, gate, bias, k)
    bal = ops.router_balance(logits, inds, mask=mask)
    dl = ops.router_grad(logits, inds, dw, balance=bal, balance_weight=weight, mask=mask)
    return loss, dx, dhead, inds, bal, dl, dl.t() @ x.float()


@pytest.mark.parametrize("T", [40, 300])
def test_step(T):
    H, V, E, k, K, weight = 256, 1200, 32, 4, 6, 0.05
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = rnd(T, H).bfloat16()
    head = (rnd(V, H) * 0.05).bfloat16()
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda", dtype=torch.int32)
    p = torch.softmax(rnd(T, K), -1)
    gate, bias = rnd(E, H) * 0.05, rnd(E) * 0.1
    mask = torch.rand(T, generator=g, device="cuda") > 0.25
    ids[~mask] = -1
    gr = mask.float() / mask.sum()
    dw = rnd(T, k) / T
    args = (x, head, ids, p, gr, gate, bias, dw, k, mask, weight)
    loss, dx, dhead, inds, bal, dl, dgate = _step(*args)

    x64, h64, g64 = (t.double().requires_grad_() for t in (x, head, gate))
    lp = torch.log_softmax(x64 @ h64.T, -1)
    ce = -(p.double() * lp.gather(1, ids.long().clamp(min=0)) * (ids >= 0)).sum(1)
    (ce * gr.double()).sum().backward()
    # dz, rounded to bf16 (2^-8), in products that are rounded to bf16 (2^-8): against the terms' absolute sums
    dz = (torch.softmax(x64 @ h64.T, -1) * (p * (ids >= 0)).sum(1, keepdim=True).double()).detach()
    dz.scatter_add_(1, ids.long().clamp(min=0), -(p * (ids >= 0)).double())
    dz = dz.abs() * gr.double()[:, None] * 2.0 ** -8 * 1.1
    for got, want, bound in ((dx, x64.grad, dz @ head.double().abs()), (dhead, h64.grad, dz.T @ x.double().abs())):
        assert ((got.double() - want).abs() <= bound + 2.0 ** -8 * want.abs() + 1e-30).all()

    z = x.double() @ g64.T
    s = torch.sigmoid(z)
    picked = s.gather(1, inds.long())
    w = picked / picked.sum(1, keepdim=True)
    q = (s / s.sum(1, keepdim=True))[mask]
    f = bal.counts.double() / bal.counts.sum()
    total = (w * dw.double())[mask].sum() + weight * E * (q.mean(0) * f).sum()
    total.backward()
    assert abs(float(bal.loss) - float((E * (q.mean(0) * f).sum()).detach())) < 1e-5
    assert torch.equal(bal.counts.cpu(), torch.bincount(inds[mask].flatten().long(), minlength=E).int().cpu())
    # fp32 logits and scores: 2^-14 of the gradient's terms through a product of T fp32 rows
    bound = 2.0 ** -14 * (dl.abs().t() @ x.float().abs()) + 1e-7 * dl.abs().max()
    assert ((dgate.double() - g64.grad).abs() <= bound.double()).all()


def test_captured_step_replayed():
    """The whole step in a graph, with other inputs at the replay, while another stream runs the same step."""
    T, H, V, E, k = 150, 128, 900, 16, 2
    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
        mask = torch.rand(T, generator=g, device="cuda") > 0.25
        return [rnd(T, H).bfloat16(), (rnd(V, H) * 0.05).bfloat16(),
                torch.randint(-1, V, (T, 3), generator=g, device="cuda", dtype=torch.int32),
                torch.rand(T, 3, generator=g, device="cuda"), rnd(T), rnd(E, H) * 0.05, rnd(E) * 0.1, rnd(T, k), k,
                mask, 0.1]
    a, b = inputs(1), inputs(2)
    _step(*a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(*a)
    want = _step(*b)
    for s, d in zip(b, a):
        if isinstance(d, torch.Tensor):
            d.copy_(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = _step(*b)
    graph.replay()
    torch.cuda.synchronize()
    flat = lambda o: [t for v in o for t in (v if isinstance(v, tuple) else (v,))]
    for u, v, w in zip(flat(want), flat(out), flat(other)):
        assert torch.equal(u, v) and torch.equal(u, w)
