"""Weights and g of very different sizes in the head's gradient with several targets."""
import pytest
import torch

from lagunalab_b200 import ops
from tests._head_util import reference, within
from tests.test_head_loss_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
def test_a_token_whose_weights_are_all_zero(bits):
    """Its g may be any size above the others' g w: it adds nothing."""
    x, head, W, ids, weights, g = make(70, 300, 64, bits=bits, K=3, seed=1)
    weights[5] = 0
    weights[6] = 0
    _, lse = ops.head_loss(x, head, ids, weights)
    g *= 1e-12
    calm = g.clone()
    calm[5:7] = 0
    g[5], g[6] = 3e38, -1e30
    want = ops.head_loss_grad(x, head, ids, lse, calm, weights, dw=bits == 16)
    got = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=bits == 16)
    assert (got[0][5:7] == 0).all() and torch.equal(got[0], want[0])
    assert bits == 4 or torch.equal(got[1], want[1])


@pytest.mark.parametrize("K", [2, 7])
@pytest.mark.parametrize("small,large", [(1e-40, 1e36), (1e-37, 1e33), (1e-33, 1e30), (1e-30, 3e36)])
def test_tiny_weights_and_a_large_factor(K, small, large):
    x, head, W, ids, weights, g = make(150, 300, 64, K=K, skip=0.2, seed=K)
    weights, g = weights * small, g * large
    _, lse = ops.head_loss(x, head, ids, weights)
    r = reference(x, W, ids, weights, g)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights)
    within(gx, r["dx"], r["bdx"])
    within(gw, r["dw"], r["bdw"])
    # beside tokens of ordinary weights
    weights[::2] = torch.rand(75, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    g[::2] /= large
    _, lse = ops.head_loss(x, head, ids, weights)
    r = reference(x, W, ids, weights, g)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights)
    within(gx, r["dx"], r["bdx"])
    within(gw, r["dw"], r["bdw"])
