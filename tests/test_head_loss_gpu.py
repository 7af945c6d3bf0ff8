"""The head's cross entropy without logits and its gradient against 64 bits, over sizes that end inside
tiles, both kinds of head, several targets a token, left-out tokens, strides, streams and graphs."""
import pytest
import torch

from lagunalab_b200 import _lib, ops
from tests._head_util import dequant64, reference, within

pytestmark = pytest.mark.gpu


def make(T, V, H, bits=16, K=1, skip=0.0, seed=0, std=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W = torch.randn(V, H, generator=g, device="cuda") * std
    if bits == 4:
        head = ops.quantize(W, 64, 4)
        W = dequant64(head)
    else:
        head = W = W.bfloat16()
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, V, (T, K), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.rand(T, K, generator=g, device="cuda") < skip] = -1
    weights = torch.rand(T, K, generator=g, device="cuda") if K > 1 else None
    gr = torch.randn(T, generator=g, device="cuda")
    return x, head, W, ids[:, 0].contiguous() if K == 1 else ids, weights, gr


def from_codes(T, H, V):
    """Whether the 4-bit loss of these sizes reads the codes themselves: no workspace of V H bf16 then."""
    return _lib.lib().lg_head_loss_workspace_bytes(T, H, V, 1, 4, 0) < V * H


def check(x, head, W, ids, weights, g, dw=True):
    r = reference(x, W, ids, weights, g)
    loss, lse = ops.head_loss(x, head, ids, weights)
    within(loss, r["loss"], r["bloss"])
    within(lse, r["lse"], r["blse"])
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=dw)
    within(gx, r["dx"], r["bdx"])
    if dw:
        within(gw, r["dw"], r["bdw"])
    return r, loss, lse, gx, gw


@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (1, 257, 64), (2, 5, 72), (64, 512, 256), (127, 255, 136),
                                   (128, 256, 64), (129, 1000, 200), (300, 5003, 128), (257, 513, 264),
                                   (5, 40000, 64), (700, 300, 520)])
def test_bf16_head(T, V, H):
    check(*make(T, V, H, seed=T + V))


@pytest.mark.parametrize("T,V,H", [(1, 300, 64), (37, 1003, 128), (200, 257, 320), (520, 700, 192)])
@pytest.mark.parametrize("K", [1, 64])
def test_4bit_head(T, V, H, K):
    x, head, W, ids, weights, g = make(T, V, H, bits=4, K=K, skip=0.2, seed=K + T)
    check(x, head, W, ids, weights, g, dw=False)


@pytest.mark.parametrize("T,V,H,K", [(1, 1, 64, 1), (1, 33, 512, 1), (16, 31, 128, 2), (17, 129, 448, 1),
                                     (31, 4740, 64, 1), (32, 700, 1024, 64), (33, 40000, 576, 3),
                                     (64, 5003, 512, 1), (65, 20000, 192, 1), (100, 9001, 2048, 64),
                                     (128, 40001, 1536, 1), (128, 300, 4096, 64), (129, 40001, 512, 1),
                                     (255, 3001, 192, 5), (256, 700, 512, 1), (384, 5000, 320, 2),
                                     (385, 5000, 320, 2), (64, 30001, 1024, 2), (129, 50001, 1024, 1),
                                     (255, 60001, 1088, 5), (384, 90001, 2048, 1)])
def test_4bit_head_of_few_tokens(T, V, H, K):
    """Both forms of the 4-bit loss. From the codes, in passes of up to 128 tokens: a CTA's ids in up to three tiles, its
    last of one to four blocks, groups of scales that come eight at a time (H % 512 == 0) or one by one."""
    if V * H > 1e6:
        assert from_codes(T, H, V) == (T <= 32 or T <= 384 and V * H > 15e6 and H >= 576)
    x, head, W, ids, weights, _ = make(T, V, H, bits=4, K=K, skip=0.2, seed=V, std=0.02)
    ids.view(T, K)[T // 2] = V - 1
    r = reference(x, W, ids, weights)
    loss, lse, top = ops.head_loss(x, head, ids, weights, top=True)
    within(loss, r["loss"], r["bloss"])
    within(lse, r["lse"], r["blse"])
    z = x.double().cpu() @ W.double().cpu().T
    assert (z.amax(1) - z.gather(1, top.long().cpu()[:, None])[:, 0] <= 2 * r["blse"]).all()
    loss, lse = ops.head_loss(x, head, ids, weights)  # without ids of maxima the sums have other references
    within(loss, r["loss"], r["bloss"])
    within(lse, r["lse"], r["blse"])
    again = ops.head_loss(x, head, ids, weights)
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)


@pytest.mark.parametrize("T,H,codes", [(7, 64, True), (40, 64, False), (40, 2048, True), (90, 64, False),
                                       (90, 2048, True)])
def test_4bit_top_of_equal_logits_is_the_lowest_id(T, H, codes):
    assert from_codes(T, H, 6000) == codes
    rows = torch.zeros(6000, H, device="cuda")
    rows[[37, 300, 301, 5990]] = 1
    x = torch.ones(T, H, dtype=torch.bfloat16, device="cuda")
    x[1] = -1
    top = ops.head_loss(x, ops.quantize(rows, 64, 4), torch.zeros(T, dtype=torch.int32, device="cuda"),
                        top=True)[2]
    assert top[1] == 0 and (top[[0, 2, T - 1]] == 37).all()


@pytest.mark.parametrize("T,V,H,codes", [(5, 3000, 128, True), (60, 3000, 128, False), (128, 3000, 128, False),
                                         (60, 9001, 2048, True), (128, 9001, 2048, True)])
def test_4bit_head_with_tokens_that_hold_nan(T, V, H, codes):
    assert from_codes(T, H, V) == codes
    x, head, W, ids, _, _ = make(T, V, H, bits=4)
    want = ops.head_loss(x, head, ids)
    x[3] = float("nan")
    got = ops.head_loss(x, head, ids)
    keep = torch.arange(T, device="cuda") != 3
    assert got[0][3].isnan() and all(torch.equal(a[keep], b[keep]) for a, b in zip(want, got))


@pytest.mark.parametrize("T,V,K", [(1, 64, 64), (33, 100, 2), (130, 900, 5), (260, 3, 17), (64, 2000, 63)])
def test_several_targets(T, V, K):
    """Few ids, so that the same one is listed twice or more."""
    check(*make(T, V, 64, K=K, skip=0.3, seed=K))


def test_targets_with_unit_weights_are_a_sum_of_losses():
    x, head, W, ids, _, g = make(50, 200, 64, K=3)
    check(x, head, W, ids, None, g)
    loss, lse = ops.head_loss(x, head, ids)
    one = sum(ops.head_loss(x, head, ids[:, j].contiguous())[0].double() for j in range(3))
    assert (loss.double() - one).abs().max() < 8 * 2 ** -24 * one.max()


def test_one_target_with_a_weight():
    x, head, W, ids, _, g = make(70, 300, 64, skip=0.2)
    weights = torch.rand(70, device="cuda")
    check(x, head, W, ids, weights, g)
    a, b = ops.head_loss(x, head, ids.view(70, 1), weights.view(70, 1)), ops.head_loss(x, head, ids, weights)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("K", [1, 3])
@pytest.mark.parametrize("in_weights", [False, True])
def test_a_common_factor_is_not_rounded(K, in_weights):
    """g (or the weights) a constant just below the middle between two bf16 numbers. dz / g is K p - 1 at a target, which
    rounds to -1 (K p < 2^-9, half a step below 1), an error of K p; elsewhere an error of 2^-8 K p.
    -g itself would be off by 2^-8 g: as much again as the result's rounding allows."""
    c, V, T = 1 + 2 ** -8 * 0.99, 3001, 150
    x, head, W, _, _, _ = make(T, V, 128, std=0.02, seed=3)
    x = x * 0.5
    ids = torch.randperm(V, device="cuda")[:T * K].view(T, K).int()
    ones, cs = torch.ones(T, K, device="cuda"), torch.full((T, K), c, device="cuda")
    weights, g = (cs, ones[:, 0].contiguous()) if in_weights else (ones, cs[:, 0].contiguous())
    _, lse = ops.head_loss(x, head, ids, weights)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights)
    X, W64 = x.double().cpu(), W.double().cpu()
    at = ids.long().cpu()
    c = float(torch.tensor(c, dtype=torch.float32))
    p = torch.softmax(X @ W64.T, 1)
    assert K * p.max() < 2 ** -9
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    dz, off = c * (K * p - hot), c * K * p * (hot + 2 ** -8 + 2 ** -12) + c * hot * 2 ** -18
    for got, l, b, m in ((gx, dz, off, W64), (gw, dz.T, off.T, X)):
        want = l @ m
        within(got, want, b @ m.abs() + 2 ** -8 * want.abs() * (1 + 2 ** -8) + 2 ** -18 * (l.abs() @ m.abs()))


def test_gradients_of_every_scale():
    """g of any size: tiny, huge, zeros, one infinite (its own row and dW are not finite)."""
    x, head, W, ids, _, g = make(70, 300, 64)
    _, lse = ops.head_loss(x, head, ids)
    one = ops.head_loss_grad(x, head, ids, lse, g)
    for e in (-60, 60):
        for a, b in zip(ops.head_loss_grad(x, head, ids, lse, g * 2.0 ** e), one):
            assert torch.equal(a.float(), b.float() * 2.0 ** e)
    for a in ops.head_loss_grad(x, head, ids, lse, torch.zeros_like(g)):
        assert not a.any()
    far = torch.zeros_like(g)
    far[3] = float("inf")
    gx, gw = ops.head_loss_grad(x, head, ids, lse, far)
    assert not gx[3].isfinite().any() and not gx[:3].any() and not gx[4:].any()


@pytest.mark.parametrize("K", [1, 7])
def test_tokens_without_a_target_may_hold_anything(K):
    x, head, W, ids, weights, g = make(200, 700, 128, K=K)
    clean = x.clone()
    out = torch.arange(0, 200, 3, device="cuda")
    ids[out] = -1
    clean[out] = 0
    x[out[::2]] = float("nan")
    x[out[1::2]] = float("inf")
    r, loss, lse, gx, gw = check(clean, head, W, ids, weights, g)
    loss2, lse2 = ops.head_loss(x, head, ids, weights)
    assert torch.equal(loss, loss2) and (loss[out] == 0).all() and lse2[out].isnan().all()
    gx2, gw2 = ops.head_loss_grad(x, head, ids, lse2, g, weights)
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2) and (gx2[out] == 0).all()


def test_every_token_left_out():
    x, head, W, ids, _, g = make(130, 300, 64)
    ids.fill_(-1)
    loss, lse = ops.head_loss(x, head, ids)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g)
    assert (loss == 0).all() and (gx == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("K", [1, 4])
def test_an_id_past_the_vocabulary(K):
    """Its token's loss is NaN; in the gradient it counts as left out."""
    x, head, W, ids, weights, g = make(140, 300, 64, K=K)
    ids.view(140, K)[17, 0] = 300
    ids.view(140, K)[18, 0] = 2 ** 31 - 1
    check(x, head, W, ids, weights, g)


def test_a_nan_row_stays_its_own():
    x, head, W, ids, _, g = make(140, 600, 64)
    r, loss, lse, gx, _ = check(x, head, W, ids, None, g)
    x[9] = float("nan")
    loss2, lse2 = ops.head_loss(x, head, ids)
    gx2, _ = ops.head_loss_grad(x, head, ids, lse2, g, dw=False)
    keep = torch.arange(140, device="cuda") != 9
    assert loss2[9].isnan() and gx2[9].isnan().all()
    assert torch.equal(loss[keep], loss2[keep]) and torch.equal(gx[keep], gx2[keep])


def test_large_logits():
    """Logits of several hundred: the maximum is taken out before the exponentials."""
    x, head, W, ids, _, g = make(130, 700, 256, std=4.0)
    loss, lse = ops.head_loss(x, head, ids)
    r = reference(x, W, ids, None)
    # the exponential's argument is up to |z| log2(e), rounded to 2^-24 of itself
    far = r["lse"].abs().max() * 2 ** -21
    within(loss, r["loss"], r["bloss"] + far)
    within(lse, r["lse"], r["blse"] + far)


@pytest.mark.parametrize("T,V", [(1, 300), (200, 1000), (3, 1)])
def test_top(T, V):
    x, head, W, ids, _, _ = make(T, V, 64)
    r = reference(x, W, ids, None)
    loss, lse, top = ops.head_loss(x, head, ids, top=True)
    z = x.double().cpu() @ W.double().cpu().T
    got = z.gather(1, top.long().cpu()[:, None])[:, 0]
    assert (z.amax(1) - got <= 2 * r["blse"]).all()  # the largest, or one as large within fp32
    a, b = ops.head_loss(x, head, ids)
    assert torch.equal(a, loss) and torch.equal(b, lse)


def test_top_of_equal_logits_is_the_lowest_id():
    head = torch.zeros(900, 64, dtype=torch.bfloat16, device="cuda")
    head[[37, 300, 301, 899]] = 1
    x = torch.ones(150, 64, dtype=torch.bfloat16, device="cuda")
    x[1] = -1
    top = ops.head_loss(x, head, torch.zeros(150, dtype=torch.int32, device="cuda"), top=True)[2]
    assert top[1] == 0 and (top[[0, 2, 149]] == 37).all()


def test_strides_and_alignment():
    x, head, W, ids, _, g = make(140, 500, 64)
    want = ops.head_loss(x, head, ids)
    gw = ops.head_loss_grad(x, head, ids, want[1], g)
    wide = torch.full((140, 80), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:72] = x
    odd = torch.full((140 * 65 + 1,), float("nan"), dtype=torch.bfloat16, device="cuda")[1:].view(140, 65)
    odd[:, :64] = x
    tall = torch.full((500, 96), float("nan"), dtype=torch.bfloat16, device="cuda")
    tall[:, :64] = head
    cases = [(wide[:, 8:72], head), (odd[:, :64], head), (x.t().contiguous().t(), head),
             (x, tall[:, :64]), (x, head.t().contiguous().t())]
    for a, b in cases:
        got = ops.head_loss(a, b, ids)
        gg = ops.head_loss_grad(a, b, ids, got[1], g)
        assert all(torch.equal(u, v) for u, v in zip(want + gw, got + gg))
    every = torch.stack([ids, ids], 1)[:, 0]  # a column
    assert torch.equal(ops.head_loss(x, head, every)[0], want[0])
    same = x[:1].expand(140, 64)  # a broadcast row
    got = ops.head_loss(same, head, ids)[1]
    assert (got == got[0]).all()


def test_no_tokens():
    x, head, W, ids, _, g = make(4, 300, 64)
    loss, lse, top = ops.head_loss(x[:0], head, ids[:0], top=True)
    gx, gw = ops.head_loss_grad(x[:0], head, ids[:0], lse, g[:0])
    assert loss.shape == lse.shape == top.shape == (0,) and gx.shape == (0, 64) and (gw == 0).all()
    gx, gw = ops.head_loss_grad(x[:0], head, ids[:0], lse, g[:0], dw=False)
    assert gx.shape == (0, 64) and gw is None


def test_one_gradient_alone():
    x, head, W, ids, _, g = make(150, 400, 128)
    lse = ops.head_loss(x, head, ids)[1]
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g)
    assert torch.equal(ops.head_loss_grad(x, head, ids, lse, g, dw=False)[0], gx)
    assert torch.equal(ops.head_loss_grad(x, head, ids, lse, g, dx=False)[1], gw)


def _many(T, V, H, K, dw, bits=16):
    """Sizes at which the vocabulary is taken in several pieces; the check runs on some rows."""
    x, head, W, ids, weights, g = make(T, V, H, bits=bits, K=K, skip=0.1, seed=V)
    loss, lse = ops.head_loss(x, head, ids, weights)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights, dw=dw)
    some = torch.tensor([0, 1, 127, 128, T // 2, T - 1], device="cuda")
    r = reference(x[some], W, ids[some], None if weights is None else weights[some], g[some])
    within(loss[some], r["loss"], r["bloss"])
    within(lse[some], r["lse"], r["blse"])
    within(gx[some], r["dx"], r["bdx"])
    if dw:  # columns of the vocabulary on either side of the pieces' ends
        z = x.double() @ W.double().cuda().T
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
        id2 = ids.view(T, -1).long()
        w = (torch.ones_like(id2, dtype=torch.float64) if weights is None else weights.double()) * (id2 >= 0)
        dz = p * w.sum(1, keepdim=True)
        dz.scatter_add_(1, id2.clamp(min=0), -w)
        dz *= g.double()[:, None]
        want = dz.T @ x.double()
        bound = (2 ** -8 + 2 ** -10) * (dz.abs().T @ x.double().abs()) + 2 ** -8 * want.abs()
        within(gw, want.cpu(), bound.cpu())


@pytest.mark.parametrize("T,V,K", [(8195, 40007, 1), (8195, 36000, 3)])
def test_vocabulary_in_pieces(T, V, K):
    _many(T, V, 64, K, True)


@pytest.mark.parametrize("T,V,H", [(1024, 1, 8), (1100, 130, 264), (2050, 300, 72), (4757, 380, 136), (3000, 5000, 64)])
def test_many_tokens_over_few_ids(T, V, H):
    """dW's contraction in parts, as its tiles alone would leave most SMs idle."""
    check(*make(T, V, H, K=2, skip=0.3, seed=V))


def test_many_tokens_over_few_ids_in_pieces():
    _many(600000, 500, 64, 1, True)


@pytest.mark.parametrize("T,V", [(257, 140001), (390, 140001)])
def test_4bit_vocabulary_in_pieces(T, V):
    _many(T, V, 2048, 2, False, bits=4)


def test_repeatable():
    x, head, W, ids, weights, g = make(300, 5000, 256, K=8)
    first = None
    for _ in range(4):
        loss, lse = ops.head_loss(x, head, ids, weights)
        out = (loss, lse) + ops.head_loss_grad(x, head, ids, lse, g, weights)
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, out))
        first = out


def test_two_streams_at_once():
    sets = [make(200 + 57 * i, 3000, 128, K=1 + 3 * i, seed=i) for i in range(2)]
    want = []
    for x, head, W, ids, weights, g in sets:
        loss, lse = ops.head_loss(x, head, ids, weights)
        want.append((loss, lse) + ops.head_loss_grad(x, head, ids, lse, g, weights))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for st, (x, head, W, ids, weights, g) in zip(streams, sets):
            with torch.cuda.stream(st):
                loss, lse = ops.head_loss(x, head, ids, weights)
                got.append((loss, lse) + ops.head_loss_grad(x, head, ids, lse, g, weights))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captured_graphs_replayed_with_new_inputs():
    x, head, W, ids, weights, g = make(150, 2000, 128, K=4)
    graphs = []
    ops.head_loss(x, head, ids, weights)
    for _ in range(2):  # two graphs: neither has the other's workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            loss, lse = ops.head_loss(x, head, ids, weights)
            out = (loss, lse) + ops.head_loss_grad(x, head, ids, lse, g, weights)
        graphs.append((gr, out))
    y = make(150, 2000, 128, K=4, skip=0.5, seed=9)
    x.copy_(y[0]), ids.copy_(y[3]), weights.copy_(y[4]), g.copy_(y[5])
    for gr, _ in graphs:
        gr.replay()
    loss, lse = ops.head_loss(x, head, ids, weights)
    want = (loss, lse) + ops.head_loss_grad(x, head, ids, lse, g, weights)
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_gradient_against_differences():
    """d loss / d x along a direction, from fp32-accurate losses at two points on either side."""
    x, head, W, ids, weights, g = make(40, 300, 64, K=3)
    loss, lse = ops.head_loss(x, head, ids, weights)
    gx, gw = ops.head_loss_grad(x, head, ids, lse, g, weights)
    d = torch.randn(40, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * 0.25
    a, b = (x + d).bfloat16(), (x - d).bfloat16()
    step = (a.double() - b.double())
    la, lb = (ops.head_loss(p, head, ids, weights)[0].double() for p in (a, b))
    want = g.double() * (la - lb)
    got = (gx.double() * step).sum(1)
    # third-order term: at most |g| S max|step . (W_v - W_u)|^3 / 24 (the softmax's third cumulant is
    # below a sixth of the spread cubed); rounding: 2^-8 of the gradient's terms and fp32 of the losses
    spread = (step @ W.double().cuda().T)
    spread = spread.amax(1) - spread.amin(1)
    r = reference(x, W, ids, weights, g)
    middle = ((a.double() + b.double()) / 2 - x.double()).abs() @ W.double().cuda().abs().amax(0)
    bound = g.abs().double() * weights.sum(1).double() * (spread ** 3 / 24 + 2 * middle * spread) \
        + (r["bdx"].cuda() * step.abs()).sum(1) + 2 * g.abs().double() * r["bloss"].cuda() * 2
    assert ((got - want).abs() <= bound).all()


def test_refusals():
    x, head, W, ids, _, g = make(4, 300, 64)
    lse = torch.zeros(4, device="cuda")
    q = ops.quantize(head.float(), 64, 4)
    bad = [(x.float(), head, ids), (x[0], head, ids), (x, head.float(), ids), (x, head[:, :32], ids),
           (x, head, ids.long()), (x, head, ids[:3]), (x, head[:0], ids), (x, q[:2] + (q[2][:3],), ids),
           (x, head, ids.view(4, 1).expand(4, 65)), (x, head, ids.view(4, 1)[:, :0]),
           (x[:, :12].contiguous(), head[:, :12].contiguous(), ids), (x.cpu(), head, ids),
           (x, head.cpu(), ids), (x, head, ids.cpu())]
    for a in bad:
        with pytest.raises(ValueError):
            ops.head_loss(*a)
        with pytest.raises(ValueError):
            ops.head_loss_grad(*a, lse, g)
    with pytest.raises(ValueError):
        ops.head_loss(x, head, ids, torch.ones(4, 2, device="cuda"))
    with pytest.raises(ValueError, match="4-bit"):
        ops.head_loss_grad(x, q, ids, lse, g)
    with pytest.raises(ValueError, match="neither"):
        ops.head_loss_grad(x, head, ids, lse, g, dx=False, dw=False)
    with pytest.raises(ValueError, match="lse"):
        ops.head_loss_grad(x, head, ids, lse[:3], g)
    with pytest.raises(ValueError, match="g must"):
        ops.head_loss_grad(x, head, ids, lse, g.double())


@pytest.mark.parametrize("T", [20, 200])
def test_4bit_scales_of_every_size(T):
    """Scales that the packed fma takes and others (0, 2^-133, 2^-5 and more, negative) in one head, some groups
    beside one another: the weights are bf16(scale * code + bias) all the same."""
    g = torch.Generator(device="cuda").manual_seed(7)
    V, H = 700, 512
    q = torch.randint(-2 ** 31, 2 ** 31, (V, H // 8), generator=g, device="cuda", dtype=torch.int32)
    s = torch.rand(V, H // 64, generator=g, device="cuda") * 0.01
    for at, v in enumerate([0.0, 2.0 ** -133, 2.0 ** -126, 0.0312, 2.0 ** -5, 0.11, -0.004, -0.2]):
        s[at * 64:at * 64 + 40, at] = v
    s = s.bfloat16()
    b = (torch.randn(V, H // 64, generator=g, device="cuda") * 0.03).bfloat16()
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    W = dequant64((q, s, b))
    assert torch.equal(ops.dequantize(q, s, b).cpu().double(), W)
    gr = torch.randn(T, generator=g, device="cuda")
    r = reference(x, W, ids, None, gr)
    loss, lse = ops.head_loss(x, (q, s, b), ids)
    far = r["lse"].abs().max() * 2 ** -21
    within(loss, r["loss"], r["bloss"] + far)
    within(lse, r["lse"], r["blse"] + far)
    within(ops.head_loss_grad(x, (q, s, b), ids, lse, gr, dw=False)[0], r["dx"], r["bdx"])


@pytest.mark.parametrize("T,H,codes", [(9, 64, True), (50, 64, True), (128, 64, False), (50, 1024, True),
                                       (128, 1024, True)])
@pytest.mark.parametrize("order", [1, -1])
def test_4bit_logits_far_above_those_before(T, H, codes, order):
    """Logits that rise (or fall) by hundreds along the vocabulary: the reference of the exponentials has to follow,
    within a CTA's tiles and between CTAs."""
    V = 40000
    assert from_codes(T, H, V) == codes
    g = torch.Generator(device="cuda").manual_seed(T)
    steps = order * torch.linspace(-900, 900, V // 32, device="cuda").repeat_interleave(32)
    rows = (torch.randn(V, H, generator=g, device="cuda") * 0.1 + (steps / H)[:, None])
    head = ops.quantize(rows, 64, 4)
    W = dequant64(head)
    x = (1 + 0.1 * torch.randn(T, H, generator=g, device="cuda")).bfloat16()
    x[1] *= -1  # this token's logits go the other way
    ids = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    ids[:2] = torch.tensor([0, V - 1])
    r = reference(x, W, ids, None)
    far = 1000 * 2 ** -21  # the exponentials' arguments: up to 1,500, rounded to 2^-24 of that
    for top in (False, True):
        loss, lse = ops.head_loss(x, head, ids, top=top)[:2]
        within(loss, r["loss"], r["bloss"] + far)
        within(lse, r["lse"], r["blse"] + far)
