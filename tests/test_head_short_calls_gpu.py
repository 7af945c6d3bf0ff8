"""Many short calls of the head's loss and gradient one behind the other: kernels whose CTAs have a tile or two each and
end at once, by one CTA a tile and by pairs, next to kernels of other sizes."""
import pytest
import torch

from lagunalab_b200 import ops
from tests.test_head_loss_gpu import make

pytestmark = pytest.mark.gpu

SIZES = [(1, 300, 64, 16, 1), (40, 1200, 256, 16, 6), (128, 257, 72, 16, 1), (129, 600, 64, 16, 3),
         (300, 90, 512, 16, 2), (3, 64, 64, 4, 1), (40, 5000, 128, 4, 6), (90, 3000, 2048, 4, 1), (200, 700, 256, 4, 2)]


def run(x, head, W, ids, weights, g):
    loss, lse = ops.head_loss(x, head, ids, weights)
    dx, dw = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=not isinstance(head, tuple))
    return [t for t in (loss, lse, dx, dw) if t is not None]


def test_short_calls():
    sets = [make(T, V, H, bits=bits, K=K, skip=0.3, seed=T) for T, V, H, bits, K in SIZES]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    for r in range(40):
        got = [run(*s) for s in sets]
        assert all(torch.equal(a, b) for w, o in zip(want, got) for a, b in zip(w, o)), r
