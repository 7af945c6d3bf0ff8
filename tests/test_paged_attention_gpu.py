"""Attention over a paged K/V cache (packed prompts and streams with a shared prefix; the SDPA
branch of Attention.__call__, laguna_mlx/laguna.py:102-107, for many sequences) against the
definition in 64 bits.

Tolerance, derived: with weights w_j >= 0 summing to 1 the kernel's output differs from
sum w_j v_j by (a) each exp weight rounded to bf16, relative 2^-8 at most, so at most
2^-8 sum w_j |v_j| in the numerator; (b) the fp32 errors of scores, exponentials and sums: a score
of magnitude s carries an error of at most 128 * 2^-24 * sum |q k| * scale, below 2^-10 for these
inputs' scores, which moves every weight by less than 2^-10 relative and the output by less than
2 * 2^-10 sum w_j |v_j|; (c) the rounding of the output to bf16, 2^-8 |o| at most, and the rounding after the
gate, as much again. Hence |out - exact| <= (2^-8 + 2^-9 + 2 * 2^-8) A = 3.5 * 2^-8 A with A = sum w_j
|v_j| * |gate| >= |o|; the bound is 2^-6 A (4 * 2^-8), plus 1e-30 for zeros."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def _case(new, kv, Hq, Hkv, R, seed=0, shared=0, junk=float("nan"), pad=0, extra=3):
    """Random inputs: pages in a random order with ``extra`` unused ones, junk in every row that
    no sequence holds, ``pad`` rows of q behind the last token. ``shared``: rows [0, shared) are the
    same rows for all (whole pages by id, the rest copied)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // R) for n in kv]
    first = shared // R
    total = first + sum(max(0, n - first) for n in need) + extra
    ids = torch.randperm(total, generator=g).tolist()
    pre, rest = ids[:first], ids[first:]
    M = max(need + [1])
    table = torch.full((len(kv), M), -7, dtype=torch.int32)
    k = torch.full((total, Hkv, R, D), junk)
    v = torch.full((total, Hkv, R, D), junk)
    rows = torch.randn(2, shared, Hkv, D, generator=g)
    for b, n in enumerate(need):
        own = [rest.pop() for _ in range(max(0, n - first))]
        pages = (pre + own)[:n]
        table[b, :n] = torch.tensor(pages, dtype=torch.int32)
        x = torch.randn(2, kv[b], Hkv, D, generator=g)
        s = min(shared, kv[b])
        x[:, :s] = rows[:, :s]
        for j, p in enumerate(pages):
            m = min(R, kv[b] - j * R)
            if j < first and m < R:
                continue  # a short stream inside a shared page: another stream fills it
            k[p, :, :m] = x[0, j * R:j * R + m].transpose(0, 1)
            v[p, :, :m] = x[1, j * R:j * R + m].transpose(0, 1)
    for j in range(first):
        k[pre[j]] = rows[0, j * R:(j + 1) * R].transpose(0, 1)
        v[pre[j]] = rows[1, j * R:(j + 1) * R].transpose(0, 1)
    T = sum(new) + pad
    q = torch.randn(T, Hq, D, generator=g)
    gate = torch.rand(T, Hq, generator=g) * 2
    c = lambda t: t.to(torch.bfloat16).cuda()
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32).cuda()
    return c(q), c(k), c(v), table.cuda(), cu, torch.tensor(kv, dtype=torch.int32).cuda(), c(gate)


def _exact(q, k, v, table, new, kv, scale, gate, window):
    """(out, A) in 64 bits."""
    Hq, Hkv, R = q.shape[1], k.shape[1], k.shape[2]
    G = Hq // Hkv
    q = q.double()
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    for b, n in enumerate(new):
        ids = table[b, :-(-kv[b] // R)].long()
        kk = k[ids].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :kv[b]]
        vv = v[ids].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :kv[b]]
        for i in range(n):
            p = kv[b] - n + i
            lo = max(0, p - window + 1) if window else 0
            if p < lo:
                continue
            for h in range(Hkv):
                qs = q[at + i, h * G:(h + 1) * G]
                w = torch.softmax(qs @ kk[h, lo:p + 1].T * scale, -1)
                out[at + i, h * G:(h + 1) * G] = w @ vv[h, lo:p + 1]
                A[at + i, h * G:(h + 1) * G] = w @ vv[h, lo:p + 1].abs()
        at += n
    if gate is not None:
        out, A = out * gate.double()[..., None], A * gate.double().abs()[..., None]
    return out, A


def _near(got, out, A, rows, bound=2 ** -6):
    err = (got[:rows].double() - out[:rows]).abs() - (bound * A[:rows] + 1e-30)
    assert not torch.isnan(got[:rows]).any()
    assert float(err.max()) <= 0, float(err.max())


PROMPTS = [
    # new tokens, rows held, Hq, Hkv, R, window
    ([1], [1], 1, 1, 16, 0),
    ([5, 1, 33], [5, 1, 33], 8, 1, 64, 0),
    ([17, 0, 40], [300, 0, 41], 32, 4, 64, 0),
    ([3, 200], [130, 457], 4, 4, 32, 0),
    ([129], [129], 16, 1, 128, 0),
    ([300], [300], 2, 2, 16, 0),
    ([64, 31, 2], [64, 159, 2], 10, 2, 16, 0),
    ([7], [1025], 14, 2, 128, 0),
    ([90, 260], [90, 900], 8, 2, 64, 1),
    ([90, 260], [90, 900], 8, 2, 64, 33),
    ([257], [700], 3, 3, 32, 128),
    ([4, 6], [2, 0], 4, 2, 16, 0),  # more new tokens than rows: some see no key
    ([513], [513], 6, 2, 64, 200),
]


@pytest.mark.parametrize("new,kv,Hq,Hkv,R,window", PROMPTS)
@pytest.mark.parametrize("gated", [False, True])
def test_prompts(new, kv, Hq, Hkv, R, window, gated):
    from lagunalab_b200 import ops
    q, k, v, table, cu, kvt, gate = _case(new, kv, Hq, Hkv, R, seed=Hq + R, pad=3)
    gate = gate if gated else None
    plan = ops.prompt_plan(cu, kvt, q.shape[0], Hq, Hkv, R, window=window)
    mark = torch.full_like(q, 7.0)
    got = ops.prompt_attention(q, k, v, table, plan, D ** -0.5, gate=gate, out=mark)
    out, A = _exact(q, k, v, table, new, kv, D ** -0.5, gate, window)
    T = sum(new)
    _near(got, out, A, T)
    assert (got[T:] == 7).all()  # rows of no sequence stay as they were


STREAMS = [
    # rows held, Hq, Hkv, R, prefix, window
    ([1], 1, 1, 16, 0, 0),
    ([300], 32, 4, 64, 0, 0),
    ([5, 0, 130, 1], 8, 2, 32, 0, 0),
    ([140, 129, 1000, 131], 16, 2, 64, 128, 0),
    ([70, 65, 66, 400], 8, 1, 16, 65, 0),
    ([70, 20, 0, 400], 10, 2, 16, 50, 0),  # a stream shorter than the prefix, and one without rows
    ([2100] * 3, 4, 4, 128, 2099, 0),
    ([300, 500, 280], 16, 1, 32, 256, 100),
    ([300, 500, 280, 257], 7, 1, 32, 256, 280),
    (list(range(129, 129 + 40)), 8, 1, 64, 128, 0),
    (list(range(200, 200 + 300)), 2, 2, 64, 192, 0),
]


@pytest.mark.parametrize("kv,Hq,Hkv,R,prefix,window", STREAMS)
@pytest.mark.parametrize("gated", [False, True])
def test_streams(kv, Hq, Hkv, R, prefix, window, gated):
    from lagunalab_b200 import ops
    new = [1 if n else 0 for n in kv]
    q, k, v, table, _, kvt, gate = _case([1] * len(kv), kv, Hq, Hkv, R, seed=Hq + R, shared=prefix)
    gate = gate if gated else None
    plan = ops.stream_plan(kvt, Hq, Hkv, R, prefix=prefix, window=window)
    got = ops.stream_attention(q, k, v, table, plan, D ** -0.5, gate=gate)
    out, A = torch.zeros_like(q).double(), torch.zeros_like(q).double()
    live = [b for b, n in enumerate(new) if n]
    o, a = _exact(q[live], k, v, table[live], [1] * len(live), [kv[b] for b in live], D ** -0.5,
                  gate[live] if gated else None, window)
    out[live], A[live] = o, a
    _near(got, out, A, len(kv))


def test_many_short_sequences_of_random_lengths():
    from lagunalab_b200 import ops
    r = random.Random(1)
    new = [r.randint(0, 9) for _ in range(1500)]
    kv = [n + r.randint(0, 30) for n in new]
    q, k, v, table, cu, kvt, _ = _case(new, kv, 2, 1, 16, seed=3)
    plan = ops.prompt_plan(cu, kvt, q.shape[0], 2, 1, 16)
    got = ops.prompt_attention(q, k, v, table, plan, 0.1)
    out, A = _exact(q, k, v, table, new, kv, 0.1, None, 0)
    _near(got, out, A, sum(new))


def test_strided_q_and_pages_of_a_pool():
    """q as columns of a wider projection, K and V as planes of one pool."""
    from lagunalab_b200 import ops
    new, kv, Hq, Hkv, R = [37, 5], [100, 5], 8, 2, 32
    q, k, v, table, cu, kvt, _ = _case(new, kv, Hq, Hkv, R, seed=5)
    wide = torch.full((q.shape[0], Hq + 5, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:2 + Hq] = q
    pool = torch.stack([v, k, v], 1)  # [P, 3, Hkv, R, D]
    plan = ops.prompt_plan(cu, kvt, q.shape[0], Hq, Hkv, R)
    want = ops.prompt_attention(q, k, v, table, plan, D ** -0.5)
    got = ops.prompt_attention(wide[:, 2:2 + Hq], pool[:, 1], pool[:, 2], table, plan, D ** -0.5)
    assert torch.equal(got, want)


def test_large_scores_and_infinite_junk():
    """Scores of magnitude hundreds (the running maximum moves far), infinities behind the rows."""
    from lagunalab_b200 import ops
    new, kv = [140, 1], [700, 260]
    q, k, v, table, cu, kvt, _ = _case(new, kv, 8, 1, 64, seed=9, junk=float("inf"))
    ramp = torch.linspace(0.1, 6, k.shape[0], device="cuda")[:, None, None, None]
    k = (k.float() * ramp).to(torch.bfloat16)
    q = (q.float() * 4).to(torch.bfloat16)
    plan = ops.prompt_plan(cu, kvt, 141, 8, 1, 64)
    got = ops.prompt_attention(q, k, v, table, plan, D ** -0.5)
    out, A = _exact(q, k, v, table, new, kv, D ** -0.5, None, 0)
    _near(got, out, A, 141)


def test_pages_outside_the_pool_give_nan():
    from lagunalab_b200 import ops
    new, kv = [20, 20], [200, 200]
    q, k, v, table, cu, kvt, _ = _case(new, kv, 4, 1, 64, seed=2, junk=0.0)
    plan = ops.prompt_plan(cu, kvt, 40, 4, 1, 64)
    want = ops.prompt_attention(q, k, v, table, plan, 0.1)
    for bad in (-1, k.shape[0], 1 << 30):
        t = table.clone()
        t[1, 1] = bad
        got = ops.prompt_attention(q, k, v, t, plan, 0.1)
        assert torch.equal(got[:20], want[:20]) and torch.isnan(got[20:]).all()
    # a length that the table row cannot hold
    plan = ops.prompt_plan(cu, kvt + torch.tensor([0, 100], dtype=torch.int32, device="cuda"), 40, 4,
                           1, 64)
    got = ops.prompt_attention(q, k, v, table, plan, 0.1)
    assert torch.equal(got[:20], want[:20]) and torch.isnan(got[20:]).all()


def test_update_in_a_captured_graph():
    """A plan and its attention replayed from a graph for lengths that grow on the device."""
    from lagunalab_b200 import ops
    kv = [100, 37, 64]
    q, k, v, table, _, kvt, _ = _case([1] * 3, [n + 100 for n in kv], 8, 2, 32, seed=4)
    kvt.copy_(torch.tensor(kv, dtype=torch.int32))
    plan = ops.stream_plan(kvt, 8, 2, 32)
    ops.stream_attention(q, k, v, table, plan, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update()
        out = ops.stream_attention(q, k, v, table, plan, 0.1)
        kvt.add_(1)
    for step in range(70):
        graph.replay()
    now = [n + 69 for n in kv]
    want, A = _exact(q, k, v, table, [1] * 3, now, 0.1, None, 0)
    _near(out, want, A, 3)


def test_the_same_call_gives_the_same_bits():
    from lagunalab_b200 import ops
    new, kv = [700, 3, 41], [2000, 900, 41]
    q, k, v, table, cu, kvt, _ = _case(new, kv, 16, 2, 64, seed=6)
    plan = ops.prompt_plan(cu, kvt, q.shape[0], 16, 2, 64)
    a = ops.prompt_attention(q, k, v, table, plan, D ** -0.5)
    for _ in range(5):
        assert torch.equal(ops.prompt_attention(q, k, v, table, plan, D ** -0.5), a)


def test_streams_of_their_own():
    """Two calls on two CUDA streams, a plan each."""
    from lagunalab_b200 import ops
    runs = []
    for i in range(2):
        new, kv = [300 + i, 5], [800, 700 - i]
        q, k, v, table, cu, kvt, _ = _case(new, kv, 8, 1, 64, seed=20 + i)
        plan = ops.prompt_plan(cu, kvt, q.shape[0], 8, 1, 64)
        runs.append((q, k, v, table, plan))
    want = [ops.prompt_attention(*r, 0.1) for r in runs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                got[i].append(ops.prompt_attention(*runs[i], 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_runs_of_one_tile_segments():
    """Many row tiles a CTA, each with one key tile that ends inside a page: the next one's loads
    are under way while this one's rows are cleared."""
    from lagunalab_b200 import ops
    r = random.Random(2)
    kv = [r.randint(1, 127) for _ in range(2500)]
    q, k, v, table, cu, kvt, _ = _case([1] * len(kv), kv, 4, 4, 128, seed=8)
    plan = ops.prompt_plan(cu, kvt, q.shape[0], 4, 4, 128)
    for _ in range(5):
        got = ops.prompt_attention(q, k, v, table, plan, 0.1)
    out, A = _exact(q, k, v, table, [1] * len(kv), kv, 0.1, None, 0)
    _near(got, out, A, len(kv))
    assert plan.status() == 0


@pytest.mark.parametrize("Hq,Hkv,new,kv", [(8, 1, [140, 3], [700, 300]), (4, 4, [1, 1], [513, 900]),
                                           (3, 3, [2], [640])])
def test_scores_that_climb(Hq, Hkv, new, kv):
    """Every 64 keys score 32 (2^46) or, for some rows, 8 above the ones before: the running
    reference has to follow at each step, in either half of a key tile. The step's part of a score is
    exact (small integers times powers of two); the other 127 terms' magnitudes sum to about 127 *
    0.64 * 0.25 = 20, and the running sum stays below 512, so a score's error is at most 128 * 2^-24 *
    512 = 2^-8 and a weight's, relative, too; numerator and sum together move by 2 * 2^-8 A. With the
    3.5 * 2^-8 A of above that is 5.5 * 2^-8 A, below the 2^-5 A that is allowed here."""
    from lagunalab_b200 import ops
    q, k, v, table, cu, kvt, _ = _case(new, kv, Hq, Hkv, 64, seed=12, junk=float("nan"))
    # one dim carries the climb, exactly: powers of two times small integers
    k = torch.nan_to_num(k.float())
    q[..., 0] = torch.where(torch.arange(q.shape[0], device="cuda")[:, None] % 3 == 0, 8.0, 32.0)
    for b, n in enumerate(kv):
        for page in range(-(-n // 64)):
            k[table[b, page].long(), :, :, 0] = float(page)
    k[..., 1:] *= 0.25
    k = k.to(torch.bfloat16)
    plan = ops.prompt_plan(cu, kvt, q.shape[0], Hq, Hkv, 64)
    got = ops.prompt_attention(q, k, v, table, plan, 1.0)
    out, A = _exact(q, k, v, table, new, kv, 1.0, None, 0)
    _near(got, out, A, sum(new), 2 ** -5)
    assert plan.status() == 0


@pytest.mark.parametrize("Hq,R", [(4, 16), (16, 32), (1, 64), (7, 128)])
def test_one_kv_head_and_one_key_tile(Hq, R):
    """With one kv head a row tile's key tiles go to two halves, of which one has none here and runs
    ahead of the loads; products in between leave shared memory full of other values."""
    from lagunalab_b200 import ops
    r = random.Random(Hq)
    junk = torch.randn(2048, 2048, device="cuda").to(torch.bfloat16)
    for k in range(40):
        new = [r.randint(3, 25) for _ in range(r.randint(8, 30))]
        q, kp, v, table, cu, kvt, _ = _case(new, new, Hq, 1, R, seed=k)
        plan = ops.prompt_plan(cu, kvt, q.shape[0], Hq, 1, R)
        got = []
        for _ in range(10):
            junk @ junk
            got.append(ops.prompt_attention(q, kp, v, table, plan, 0.1))
        assert all(torch.equal(g, got[0]) for g in got[1:])
        if k < 3:
            out, A = _exact(q, kp, v, table, new, new, 0.1, None, 0)
            _near(got[0], out, A, sum(new))
        assert not torch.isnan(got[0]).any()


def test_a_plan_of_other_sizes_is_refused_on_the_device():
    """Through the C interface, which cannot look into the plan: nothing is written, the plan's status
    says so. (The Python surface refuses before.)"""
    from lagunalab_b200 import _lib, ops
    q, k, v, table, cu, kvt, _ = _case([20, 7], [90, 7], 4, 2, 32, seed=1)
    out = torch.full_like(q, 7.0)
    plan = ops.prompt_plan(cu, kvt, 27, 4, 2, 32)

    def call(T, Hq, Hkv, R, B):
        ks = k.stride()
        _lib.call("lg_prompt_attention", q.data_ptr(), q.stride(0), q.stride(1), T, Hq, Hkv, D,
                  k.data_ptr(), v.data_ptr(), k.shape[0], R, ks[0], ks[1], ks[2], table.data_ptr(),
                  B, table.shape[1], 0.1, None, out.data_ptr(), plan.ptr, 1 << 40,
                  torch.cuda.current_stream().cuda_stream)

    for bad in ((26, 4, 2, 32, 2), (27, 2, 2, 32, 2), (27, 4, 1, 32, 2), (27, 4, 2, 16, 2),
                (27, 4, 2, 32, 1)):
        call(*bad)
        assert (out == 7).all() and plan.status() == 10
        plan.update()
    call(27, 4, 2, 32, 2)
    assert plan.status() == 0 and not (out == 7).any()
    with pytest.raises(ValueError, match="plan is for"):
        ops.stream_attention(q, k, v, table, plan, 0.1)
    with pytest.raises(ValueError, match="plan is for"):
        ops.prompt_attention(q[:26], k, v, table, plan, 0.1)
    with pytest.raises(ValueError, match="rows"):
        ops.prompt_attention(q, k, v, table[:1], plan, 0.1)
    with pytest.raises(ValueError, match="shares memory"):
        ops.prompt_attention(q, k, v, table, plan, 0.1, out=q)
    with pytest.raises(ValueError, match="gate"):
        ops.prompt_attention(q, k, v, table, plan, 0.1, gate=torch.ones(27, 4, device="cuda"))
    with pytest.raises(ValueError, match="bf16"):
        ops.prompt_attention(q.float(), k, v, table, plan, 0.1)
    with pytest.raises(ValueError, match="strides"):
        ops.prompt_attention(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), table, plan, 0.1)


def test_offsets_past_32_bits():
    """Pages, tokens and output rows whose element offsets pass 2^31."""
    from lagunalab_b200 import ops
    P, Hq, Hkv, R, n, B = 17000, 32, 8, 128, 128, 4375
    kv = torch.full((2, P, Hkv, R, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    for p in (0, P - 2, P - 1):
        kv[:, p] = torch.randn(2, Hkv, R, D, generator=g, device="cuda").to(torch.bfloat16)
    assert kv[0].numel() > 2 ** 31 and n * B * Hq * D > 2 ** 31
    q = torch.randn(n * B, Hq, D, generator=g, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([[0, P - 1], [P - 1, P - 2]], dtype=torch.int32, device="cuda")
    table = rows.repeat(B // 2 + 1, 1)[:B].contiguous()
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    lens = torch.full((B,), 200, dtype=torch.int32, device="cuda")
    plan = ops.prompt_plan(cu, lens, n * B, Hq, Hkv, R)
    got = ops.prompt_attention(q, kv[0], kv[1], table, plan, D ** -0.5)
    assert plan.status() == 0
    for b in (0, 1, B - 2, B - 1):
        at = slice(b * n, (b + 1) * n)
        out, A = _exact(q[at], kv[0], kv[1], table[b:b + 1], [n], [200], D ** -0.5, None, 0)
        _near(got[at], out, A, n)
