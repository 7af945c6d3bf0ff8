"""The head's gradient at tokens that the model is nearly sure of, where a target's S p - w is a small difference.

There an error of z against lse is one of dz itself. Both take a heavy target's logit from the same fp32 sum, whose
error delta (at most 72 2^-24 sum |x w|: a lane's 64 terms and 5 joins) then only scales 1 - p, as the others' own
errors do (bz: (H + 4) 2^-24 sum |x w|, the tensor cores'). What is left besides dz's rounding to bf16:
lse's rounding, |lse| 2^-24, as much again from the largest logit's log2(e) multiple in its tile's exponentials, and
2^-22 from each of two exponentials near 1 and at most 8 2^-24 from additions of sums near 1: 2^-20 together."""
import pytest
import torch

from lagunalab_b200 import ops
from tests._head_util import E32, EBF, dequant64, within

pytestmark = pytest.mark.gpu

H = 2048


def exact(x, W, ids, weights, g):
    """dz of ids [T, K], and its bound."""
    x, W, at, w = x.double().cpu(), W.double().cpu(), ids.long().cpu(), weights.double().cpu()
    z = x @ W.T
    lse = torch.logsumexp(z, 1, keepdim=True)
    S = w.sum(1, keepdim=True)
    dz = S * torch.exp(z - lse)
    dz.scatter_add_(1, at, -w)
    bz = (H + 4) * E32 * (x.abs() @ W.abs().T)
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    delta = 72 * E32 * (x.abs() @ W.abs().T).amax(1, keepdim=True)
    rel = EBF + 2.0 ** -12 + delta + torch.where(hot > 0, 0.0, bz).amax(1, keepdim=True)
    b = rel * dz.abs() + hot * S * (2 * lse.abs() * E32 + 2.0 ** -20)
    g = g.double().cpu()[:, None]
    return dz * g, b * g.abs(), x, W


def check(x, head, W, ids, weights, g, dw):
    _, lse = ops.head_loss(x, head, ids, weights)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=dw)
    T = x.shape[0]
    w = torch.ones(T, 1) if weights is None else weights.view(T, -1)
    dz, b, X, W64 = exact(x, W, ids.view(T, -1), w, g)
    for got, l, bl, m in ((gx, dz, b, W64), (gw, dz.T, b.T, X)):
        if got is not None:
            want = l @ m
            within(got, want, (bl @ m.abs() + (l.shape[1] + 4) * E32 * (l.abs() @ m.abs())) * (1 + EBF)
                   + EBF * want.abs())
    return dz


def sure(T, rest, bits, repeat=1):
    """T tokens that are nearly alike, and a head in which ids 5 .. 5 + repeat - 1 share all but about `rest` of their
    probability: (x, head, the weights that it stands for). Their products with x are all of one sign."""
    g = torch.Generator(device="cuda").manual_seed(T)
    base = torch.rand(1, H, generator=g, device="cuda") + 0.5
    x = (base * (1 + 0.02 * torch.randn(T, H, generator=g, device="cuda"))).bfloat16()
    W = torch.randn(24, H, generator=g, device="cuda") * 2e-4
    W -= (W @ base.T) / (base @ base.T) * base
    z = torch.log(torch.tensor((24 - repeat) * (1 - rest) / (rest * repeat)))
    W[5:5 + repeat] = z / H + (z / H) * (base - 1) * 0.5
    if bits == 4:
        head = ops.quantize(W, 64, 4)
        W = dequant64(head)
    else:
        head = W = W.bfloat16()
    return x, head, W


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T", [6, 240])  # one CTA a tile, a pair
@pytest.mark.parametrize("rest", [1e-2, 1e-3, 1e-4, 1e-5, 3e-6])
def test_one_target(bits, T, rest):
    x, head, W = sure(T, rest, bits)
    ids = torch.full((T,), 5, dtype=torch.int32, device="cuda")
    g = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) + 0.5
    dz = check(x, head, W, ids, None, g, bits == 16)
    assert rest / 8 < dz[:, 5].abs().max() < rest * 8
    weights = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) + 0.1
    check(x, head, W, ids, weights, g, bits == 16)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rest", [1e-3, 1e-4, 1e-5])
def test_shares_that_are_met(bits, rest):
    """Two ids of equal logits with half of the weight each, one of them listed twice, and a place that is left out."""
    T = 9
    x, head, W = sure(T, rest, bits, repeat=2)
    ids = torch.tensor([6, -1, 5, 6], dtype=torch.int32, device="cuda").repeat(T, 1)
    weights = torch.tensor([0.25, 7.0, 0.5, 0.25], device="cuda").repeat(T, 1)
    g = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) + 0.5
    _, lse = ops.head_loss(x, head, ids, weights)
    gx, _ = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=False)
    keep = [0, 2, 3]
    dz, b, _, W64 = exact(x, W, ids[:, keep], weights[:, keep], g)
    want = dz @ W64
    within(gx, want, (b @ W64.abs() + (dz.shape[1] + 4) * E32 * (dz.abs() @ W64.abs())) * (1 + EBF)
           + EBF * want.abs())
