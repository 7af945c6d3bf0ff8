"""lse where one logit is most of the softmax, whether it is a target or not.

A target's logit is summed again in fp32 for lse. A token with the same row but without that target (none, or another)
has the same lse: both take the largest logit from one fp32 sum, and differ by their roundings alone, each
|lse| 2^-24 twice and 2^-20 (see test_head_grad_confident_gpu.py), and by the tensor cores' errors of the other
logits, bz times their share `rest` of the softmax. The tensor cores' own sum would be off by 1e-5 and more."""
import pytest
import torch

from lagunalab_b200 import _lib, ops
from tests._head_util import E32
from tests.test_head_grad_confident_gpu import H, sure

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T", [6, 90, 240, 600])  # from the codes in two forms, products by one CTA a tile and by pairs
@pytest.mark.parametrize("rest", [0.6, 0.3, 1e-2, 1e-4])
@pytest.mark.parametrize("K", [1, 3])
def test_lse_without_the_target(bits, T, rest, K):
    x, head, W = sure(T, rest, bits)
    ids = torch.full((T, K), -1, dtype=torch.int32, device="cuda")
    ids[:, K // 2] = 5
    _, want = ops.head_loss(x, head, ids)
    bz = ((H + 4) * E32 * (x.double().abs() @ W.double().abs().T.cuda())).cpu()
    bz[:, 5] = 0
    bound = 2 * (2 * want.double().cpu().abs() * E32 + 2.0 ** -20) + 2 * rest * bz.amax(1)
    for other in (-1, 9):
        ids[:, K // 2] = other
        for top in (False, True):
            loss, lse = ops.head_loss(x, head, ids, top=top)[:2]
            assert ((lse - want).double().cpu().abs() <= bound).all()
            row = W[9].double().cuda()
            z, bz9 = x.double() @ row, 72 * E32 * (x.double().abs() @ row.abs())  # an fp32 sum as well
            assert (loss == 0).all() if other < 0 else \
                ((loss.double() - (lse.double() - z)).abs() <= 2.0 ** -20 + bz9 + 2 * E32 * lse.abs()).all()
    assert _lib.lib().lg_head_loss_workspace_bytes(8192, 2048, 100352, 1, 16, 0) < 64 << 20


def test_one_id_and_few():
    """A vocabulary of one id, and of fewer than a block: the largest logit is always near."""
    for V in (1, 3, 33):
        x, head, W = sure(40, 0.3, 16)
        W = W[:V].contiguous()
        loss, lse = ops.head_loss(x, W, torch.full((40,), -1, dtype=torch.int32, device="cuda"))
        want = torch.logsumexp(x.double().cpu() @ W.double().cpu().T, 1)
        bz = 72 * E32 * (x.double().cpu().abs() @ W.double().cpu().abs().T).amax(1)
        bound = 2.0 ** -18 + 2 * E32 * want.abs() + bz
        assert ((lse.double().cpu() - want).abs() <= bound).all() and (loss == 0).all()
