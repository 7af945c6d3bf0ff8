"""Tokens whose scores (or whose picks' scores) are all so small that they are 0 in fp32, while the quotients that the
balance loss and its gradient are made of are not. Bounds as for other logits: exponentials of differences here.

Sums of 2^-80 and more are not taken again: a score below 2^-126 is then 0 where its share is up to 2^-46, and each
gradient of shares is off by that times the sum of its differences (check_picks)."""
import pytest
import torch

from lagunalab_b200 import ops
from tests.test_router_loss_gpu import check_balance, check_grad, grad64, make, scores

pytestmark = pytest.mark.gpu


def far64(logits, inds, dw, norm, mask, weight):
    """(mean shares, gradient of the logits, its bound) of sigmoid scores from their logarithms in 64 bits, in which no
    quotient of two scores underflows: the formula and the bound of check_balance and check_grad."""
    z, i = logits.cpu().double(), inds.cpu().long()
    T, E = z.shape
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
    ls, rest = torch.nn.functional.logsigmoid(z), torch.sigmoid(-z)
    q = torch.exp(ls - torch.logsumexp(ls, 1, keepdim=True))
    probs = q[keep].sum(0) / max(int(keep.sum()), 1)
    grad, bound = torch.zeros_like(z), torch.zeros_like(z)
    if dw is not None:
        d = dw.cpu().double()
        lp = ls.gather(1, i)
        most = 2 * d.abs().sum(1, keepdim=True)
        if norm:
            all_ = torch.logsumexp(lp, 1, keepdim=True)
            w = torch.exp(lp - all_)
            grad.scatter_add_(1, i, w * (d - (w * d).sum(1, keepdim=True)))
            bound += most * torch.exp(ls - all_)
        else:
            grad.scatter_add_(1, i, torch.exp(lp) * d)
            bound += most * torch.exp(ls)
    if weight is not None:
        counts = torch.bincount(i[keep].flatten(), minlength=E).double()
        dq = weight * E * counts / max(float(counts.sum()), 1) / max(int(keep.sum()), 1)
        grad += q * (dq - (q * dq).sum(1, keepdim=True))
        bound += 2 * dq.max() * q
    zero = ~keep[:, None]
    return probs, (grad * rest).masked_fill(zero, 0), (2.0 ** -17 * bound * rest + 1e-37).masked_fill(zero, 0)


SIZES = [(40, 20, 3), (300, 128, 8), (90, 200, 20), (301, 61, 2)]


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("low", [50, 87, 100, 3000])
def test_scores_that_underflow(T, E, k, low):
    """Sigmoids of logits far below 0, in some tokens or all."""
    for every in (1, 3):
        logits, inds, dw, mask = make(T, E, k, T)
        logits[::every] -= low
        got = ops.router_balance(logits, inds, "sigmoid", mask)
        probs, _, _ = far64(logits, inds, None, True, mask, None)
        rel = 2.0 ** -20 + (T / 16 + 24) * 2.0 ** -24
        assert ((got.probs.cpu().double() - probs).abs() <= rel * probs + 1e-37).all()
        if low < 700:  # the scores themselves are numbers in 64 bits
            check_balance(logits, inds, "sigmoid", mask)
        for norm, with_dw, weight in ((False, True, None), (True, True, None), (True, True, 0.5), (False, True, 0.5),
                                      (True, False, 1.0)):
            d = dw if with_dw else None
            g = ops.router_grad(logits, inds, d, norm, "sigmoid", None if weight is None else got, weight or 0.0, mask)
            _, want, bound = far64(logits, inds, d, norm, mask, weight)
            assert ((g.cpu().double() - want).abs() <= bound).all()
            if low < 700:
                check_grad(logits, inds, d, norm, "sigmoid", mask, weight)


def check_picks(logits, inds, dw, norm, fn, mask, weight):
    """check_grad, with 2^-46 of the differences' sums for shares of scores that are 0 in fp32."""
    bal = None if weight is None else ops.router_balance(logits, inds, fn, mask)
    got = ops.router_grad(logits, inds, dw, norm, fn, bal, weight or 0.0, mask).cpu().double()
    want = grad64(logits, inds, dw, norm, fn, mask, weight)
    E = logits.shape[1]
    s, i, keep = scores(logits.cpu().double(), fn), inds.cpu().long(), mask.cpu()
    p = torch.where((i >= 0) & (i < E), s.gather(1, i.clamp(0, E - 1)), 0.0)
    most = 2 * dw.cpu().double().abs().sum(1, keepdim=True)
    mass = most / p.sum(1, keepdim=True).clamp(min=1e-300) if norm else most
    lost = 2.0 ** -46 * most
    if weight is not None:
        share = bal.counts.cpu().double()
        share = weight * E * share / max(float(share.sum()), 1) / max(int(bal.tokens), 1)
        mass = mass + 2 * share.max() / (1.0 if fn == "softmax" else s.sum(1, keepdim=True))
        lost = lost + 2.0 ** -46 * 2 * share.max()
    bound = 2.0 ** -17 * mass * (s if fn == "softmax" else s * (1 - s)) + lost
    assert (got[~keep] == 0).all()
    assert ((got - want).abs()[keep] <= bound[keep]).all()


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
@pytest.mark.parametrize("low", [60, 90, 200])
def test_picks_that_underflow(T, E, k, fn, low):
    """Picks far below the token's other scores, one of them twice and one outside the experts."""
    logits, _, dw, mask = make(T, E, k, T)
    inds = (torch.arange(k, device="cuda") * 2 % E).repeat(T, 1).to(torch.int32)
    if k > 2:
        inds[::2, 2] = inds[::2, 0]
        inds[1::2, 1] = E
    logits.scatter_add_(1, inds.long().clamp(max=E - 1), torch.full((T, k), -float(low), device="cuda"))
    for norm, weight in ((True, None), (True, 0.5), (False, None), (False, 0.5)):
        check_picks(logits, inds, dw, norm, fn, mask, weight)


def test_one_not_a_number_stays_its_own():
    """Without norm and without a balance loss a sigmoid's gradient is each score's own."""
    logits, inds, dw, _ = make(50, 30, 4)
    want = ops.router_grad(logits, inds, dw, False)
    logits[7, 3] = float("nan")
    got = ops.router_grad(logits, inds, dw, False)
    assert got[7, 3].isnan()
    got[7, 3] = want[7, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("fn", ["sigmoid", "softmax"])
def test_every_logit_of_minus_infinity(fn):
    """Shares of nothing are not numbers, in the 64-bit form as here; a sigmoid's own gradient is 0."""
    logits, inds, dw, _ = make(10, 30, 4)
    logits[4] = float("-inf")
    got = ops.router_grad(logits, inds, dw, False, fn).cpu()
    want = grad64(logits, inds, dw, False, fn, None, None)
    assert (got.isnan() == want.isnan()).all() and (fn == "softmax" or (got[4] == 0).all())
