"""The head's loss and gradient in 64 bits, with bounds of what fp32 sums and bf16 operands may be off.

A product of H bf16 pairs is exact term by term; its fp32 sum is off by at most H 2^-24 sum |x w| (dz_z).
exp2's approximation and its argument's rounding are within 2^-20 of a term for |z| < 8 (the argument
is rounded to 2^-24 of at most 16), a sum of exponentials goes through at most 60 additions, so that lse is off
by at most dz_z + 2^-17. dz takes that relative to its softmax term, and 2^-8 relative from its rounding to
bf16; the products with W or x add H 2^-24 as above, the result's rounding 2^-8 relative."""
import torch

E32, EBF = 2.0 ** -24, 2.0 ** -8


def dequant64(head):
    q, s, b = (t.cpu() for t in head)
    codes = torch.stack([(q >> (4 * i)) & 15 for i in range(8)], -1).flatten(1).double()
    w = codes * s.double().repeat_interleave(64, 1) + b.double().repeat_interleave(64, 1)
    return w.to(torch.bfloat16).double()


def reference(x, W, ids, weights, g=None):
    """dict of loss, lse, dx, dw, top in 64 bits and their bounds (bloss, ...). Rows of x without a target count as
    zeros for dw."""
    x, W = x.double().cpu(), W.double().cpu()
    T, H = x.shape
    V = W.shape[0]
    ids = ids.view(T, -1).long().cpu()
    w = torch.ones(ids.shape) if weights is None else weights.cpu().view(ids.shape)
    ok = (ids >= 0) & (ids < V)
    w = torch.where(ok, w.double(), 0.0)
    at = ids.clamp(0, V - 1)
    z = x @ W.T
    bz = (H + 4) * E32 * (x.abs() @ W.abs().T)
    lse = torch.logsumexp(z, 1)
    blse = bz.amax(1) + 2.0 ** -17
    loss = torch.where(w != 0, w * (lse[:, None] - z.gather(1, at)), 0.0).sum(1)
    has = ok.any(1)
    loss = torch.where(has, loss, 0.0)
    bloss = (w.abs() * (2 * blse[:, None] + (ids.shape[1] + 2) * E32
                        * (lse[:, None] - z.gather(1, at)).abs())).sum(1)
    bloss = torch.where(has, bloss, 0.0)
    loss = torch.where((ids >= V).any(1), float("nan"), loss)
    r = dict(loss=loss, lse=lse, bloss=bloss, blse=blse + 2 * E32 * lse.abs(), top=z.argmax(1))
    if g is not None:
        g = g.double().cpu()
        p = torch.exp(z - lse[:, None]) * (g * w.sum(1))[:, None]
        dz = p.clone()
        dz.scatter_add_(1, at, -(g[:, None] * w))
        dz = torch.where(has[:, None], dz, 0.0)
        bdz = p.abs() * (2 * blse[:, None] + bz + 8 * E32) + EBF * dz.abs() \
            + torch.zeros_like(p).scatter_add_(1, at, 64 * E32 * (g[:, None] * w).abs())
        bdz = torch.where(has[:, None], bdz, 0.0)
        xz = torch.where(has[:, None], x, 0.0)
        for name, l, bl, m in (("dx", dz, bdz, W), ("dw", dz.T, bdz.T, xz)):
            r[name] = l @ m
            r["b" + name] = (bl @ m.abs() + (l.shape[1] + 4) * E32 * (l.abs() @ m.abs())) * (1 + EBF) \
                + EBF * r[name].abs() + 1e-37
    return r


def within(got, want, bound):
    got, want = got.double().cpu(), want.cpu()
    assert (got.isnan() == want.isnan()).all()
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by up to " \
        f"{((got - want).abs() / bound.clamp(min=1e-300)).nan_to_num().max():.3g} of the bound"
