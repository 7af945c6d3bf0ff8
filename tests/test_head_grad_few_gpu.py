"""The head's gradient of few tokens: dz is kept with what its rounding to bf16 left, so that the results' own rounding
is nearly all of their error.

dz is within 2^-18 of itself then (two roundings of at most 2^-9, and a factor of 2 for their difference's), and of what
reference()'s bound holds besides the rounding."""
import pytest
import torch

from lagunalab_b200 import ops
from tests._head_util import E32, EBF, reference, within
from tests.test_head_loss_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,V,H", [(1, 300, 64), (2, 1003, 192), (17, 130, 64), (33, 257, 320), (40, 3001, 512),
                                   (63, 700, 64), (64, 2000, 128)])
@pytest.mark.parametrize("K", [1, 7])
@pytest.mark.parametrize("bits", [16, 4])
def test_few_tokens(T, V, H, K, bits):
    x, head, W, ids, weights, g = make(T, V, H, bits=bits, K=K, skip=0.2, seed=T + K)
    if K == 1:  # a weight of its own a token, so that a target's dz is not 1 in units of the largest
        weights = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)) + 0.1
    _, lse = ops.head_loss(x, head, ids, weights)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=bits == 16)
    r = reference(x, W, ids, weights, g)
    # reference()'s dz again, for the part of its bound that is dz's rounding
    X, W64, at = x.double().cpu(), W.double().cpu(), ids.long().cpu().view(T, -1)
    w = torch.where(at >= 0, weights.double().cpu().view(T, -1), 0.0)
    g64 = g.double().cpu()[:, None]
    dz = torch.softmax(X @ W64.T, 1) * (g64 * w.sum(1, keepdim=True))
    dz.scatter_add_(1, at.clamp(min=0), -(g64 * w))
    X = torch.where((at >= 0).any(1, keepdim=True), X, 0.0)
    less = EBF - 2.0 ** -18
    for got, name, l, m in ((gx, "dx", dz, W64), (gw, "dw", dz.T, X)):
        if got is not None:
            bound = r["b" + name] - less * (l.abs() @ m.abs()) + 4 * (l.shape[1] + 8) * E32 * (l.abs() @ m.abs())
            within(got, r[name], bound)
