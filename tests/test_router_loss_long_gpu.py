"""The router's balance loss and gradient where a warp takes more than one turn of tokens, against 64 bits.

Bound of the mean shares, which are sums of positive terms: 2^-20 for a score (an exponential of an argument up to 16, a
division's approximation, a sum of up to 256 terms), and 2^-24 for each addition that a term goes through: the turns
of its lane (T tokens over C CTAs of 32 warps of 32 / G tokens, at least two a trip), up to 2 joins of tokens beside one
another, 32 warps, the CTAs of its slice, the slices, and 2 for the mean. The loss adds its own sum over experts (2^-18).
The gradient's bound is that of the short batches: a token's gradient has no sum over tokens."""
import pytest
import torch

from lagunalab_b200 import ops
from tests.test_router_loss_gpu import balance64, check_grad, make

pytestmark = pytest.mark.gpu

# one CTA with several trips; more tokens than a trip of 144 CTAs, for each number of lanes a token; a join of two trips
SIZES = [(250, 128, 8), (256, 256, 32), (200, 66, 9), (10007, 200, 3), (20000, 256, 32), (40000, 128, 8), (80001, 64, 8),
         (30001, 61, 2)]


def relative(T, E, k):
    G = 8 if E <= 64 and k <= 8 else 16 if E <= 128 and k <= 16 else 32
    C = 1 if T <= 256 else min(144, -(-T // 64))
    S = 1024 // (-(-E // 32) * 32)
    turns = 2 * -(-T // (2 * C * 32 * (32 // G)))
    return 2.0 ** -20 + (turns + 2 + 32 + -(-C // S) + S + 2) * 2.0 ** -24


def data(T, E, k):
    """Picks with some outside the experts and some twice, as well."""
    logits, inds, dw, mask = make(T, E, k, T)
    if k > 1:
        inds[::5, 1] = inds[::5, 0]
        inds[1::7, 0] = -1
        inds[2::7, k - 1] = E
    return logits, inds, dw, mask


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
@pytest.mark.parametrize("masked", [False, True])
def test_balance(T, E, k, fn, masked):
    logits, inds, _, mask = data(T, E, k)
    mask = mask if masked else None
    loss, counts, probs, n = balance64(logits, inds, fn, mask)
    got = ops.router_balance(logits, inds, fn, mask)
    assert torch.equal(got.counts.cpu().long(), counts) and int(got.tokens) == n
    rel = relative(T, E, k)
    assert ((got.probs.cpu().double() - probs).abs() <= rel * probs).all()
    assert abs(float(got.loss) - float(loss)) <= (rel + 2.0 ** -18) * float(loss)


@pytest.mark.parametrize("T,E,k", SIZES[3:])
@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
@pytest.mark.parametrize("norm,with_dw,weight,masked", [(True, True, 0.5, True), (False, True, 0.01, False),
                                                        (True, True, None, False), (False, True, None, True),
                                                        (True, False, 1.0, True)])
def test_grad(T, E, k, fn, norm, with_dw, weight, masked):
    logits, inds, dw, mask = data(T, E, k)
    check_grad(logits, inds, dw if with_dw else None, norm, fn, mask if masked else None, weight)
