"""The loss of tokens that the model is nearly sure of, at large logits: it is a small difference of lse and the target's
logit, and does not have their roundings.

The target's logit comes from one fp32 sum, whose error only scales 1 - p (72 2^-24 sum |x w|), as the others' own errors
do ((H + 4) 2^-24 sum |x w|, the tensor cores', and 2^-24 of the logit in the exponentials' arguments, twice). Besides:
2^-22 from each of two exponentials near 1 and at most 8 2^-24 from additions of sums near 1, together 2^-20."""
import pytest
import torch

from lagunalab_b200 import ops
from tests._head_util import E32, dequant64
from tests.test_head_grad_confident_gpu import H, sure

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("T", [6, 90, 240, 600])
@pytest.mark.parametrize("rest", [1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("shift", [0, 50, 200])
def test_loss(bits, T, rest, shift):
    x, head, W = sure(T, rest, bits)
    if shift:  # as much for every id
        W = W.float().cuda() + shift / H
        if bits == 4:
            head = ops.quantize(W, 64, 4)
            W = dequant64(head)
        else:
            head = W = W.bfloat16()
    ids = torch.full((T,), 5, dtype=torch.int32, device="cuda")
    z = x.double().cpu() @ W.double().cpu().T
    size = x.double().cpu().abs() @ W.double().cpu().abs().T
    want = torch.logsumexp(z - z[:, 5:6], 1)
    rel = (72 + H + 4 + 2) * E32 * size.amax(1)
    bound = 2.0 ** -20 + 2 * want * (rel + 2.0 ** -20)
    for top in (False, True):
        loss, lse = ops.head_loss(x, head, ids, top=top)[:2]
        assert ((loss.double().cpu() - want).abs() <= bound).all()
