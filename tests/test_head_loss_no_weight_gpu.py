"""Targets whose weights are all 0: their logits are not summed again, so that lse does not depend on which they are."""
import pytest
import torch

from lagunalab_b200 import ops
from tests.test_head_loss_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,V,bits", [(40, 900, 16), (200, 900, 16), (40, 900, 4), (200, 900, 4)])
@pytest.mark.parametrize("K", [1, 64])
def test_lse_does_not_depend_on_ids_without_weight(T, V, bits, K):
    x, head, W, ids, _, g = make(T, V, 2048, bits=bits, K=K, seed=T, std=0.1)
    other = (ids + 37) % V
    nothing = torch.zeros(ids.shape, device="cuda")
    a, b = (ops.head_loss(x, head, i, nothing) for i in (ids, other))
    assert (a[0] == 0).all() and (b[0] == 0).all() and torch.equal(a[1], b[1])
    gx, gw = ops.head_loss_grad(x, head, ids, a[1], g, nothing, dw=bits == 16)
    assert not gx.any() and (gw is None or not gw.any())
