"""The paged cache (``paged``, ``ops.pages_*``, the paged attention; no counterpart in the reference)
where a caller's lists, lengths and plans leave the ordinary path: decode steps past the reserved
rows, and states that an operation has to refuse as a whole."""
import pytest
import torch

from tests.test_streams_gpu import _model, _prompts

pytestmark = pytest.mark.gpu


def _t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _step_tokens(n, step):
    return _t([(7 * s + 31 * step) % 512 for s in range(n)])


@pytest.mark.parametrize("prefix", [0, 70])
def test_a_stream_without_a_page_sits_the_step_out(prefix):
    """Stream 1 is freed and stream 2 runs past its reserved rows while their Decoder goes on: their
    lengths stay, their logits are NaN, the others' steps give the bits that they give when every
    stream has its pages; after a reserve stream 2 goes on with the bits that it gives when it never
    had to wait."""
    from lagunalab_b200 import paged
    _, model, _, _ = _model("full")
    prompt = _prompts([70], 5)[0].tolist()

    def start(rows):  # rows reserved for streams 0, 1, 2
        cache = paged.PagedCache(model, 4, 40, 16, max_rows=96)
        paged.prefill(model, cache, [3], [prompt])
        cache.fork([3] * 3, [0, 1, 2])
        cache.reserve([0, 1, 2], rows)
        return cache, paged.Decoder(model, cache, [0, 1, 2], prefix=prefix)

    cache, dec = start([90, 90, 80])
    full, ref = start([90, 90, 96])
    want = [ref.step(_step_tokens(3, i)).clone() for i in range(13)]
    for i in range(3):
        assert torch.equal(dec.step(_step_tokens(3, i)), want[i])
    cache.free([1])
    for i in range(3, 13):  # stream 2 has rows 70..79
        got = dec.step(_step_tokens(3, i))
        assert cache.lens.tolist() == [71 + i, 0, min(71 + i, 80), 70]
        assert torch.equal(got[0], want[i][0])
        assert torch.isnan(got[1]).all()
        assert torch.equal(got[2], want[i][2]) if i < 10 else torch.isnan(got[2]).all()
        assert dec.wrote.tolist() == [True, False, i < 10]
    cache.reserve([2], [96])
    got = dec.step(_step_tokens(3, 10))
    assert torch.equal(got[2], want[10][2]) and cache.lens.tolist() == [84, 0, 81, 70]
    # the freed stream starts from nothing, as a fresh one does
    other = _prompts([9], 8)[0].tolist()
    a = paged.prefill(model, cache, [1], [other])
    fresh = paged.PagedCache(model, 1, 4, 16)
    assert torch.equal(a, paged.prefill(model, fresh, [0], [other]))
    # past the table's last column, where the last page is there
    for i in range(11, 30):
        dec.step(_step_tokens(3, i))
    assert cache.lens.tolist()[2] == 96 and dec.wrote.tolist()[2] is False


def test_a_replayed_step_leaves_a_freed_stream_out():
    """A step captured while all streams had pages gives the bits of eager steps after one is freed, and
    after pages that were missing have come."""
    from lagunalab_b200 import paged
    _, model, _, _ = _model("sliding")
    prompts = [p.tolist() for p in _prompts([37, 30, 20], 9)]
    runs = []
    for _ in range(2):
        cache = paged.PagedCache(model, 3, 12, 32)
        paged.prefill(model, cache, [0, 1, 2], prompts)  # two, one and one page
        runs.append((cache, paged.Decoder(model, cache, [0, 1, 2])))
    (cache, dec), (cache_e, eager) = runs
    tok = _step_tokens(3, 0)
    assert torch.equal(dec.step(tok), eager.step(tok))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = dec.step(tok)
    for i in range(1, 12):
        for c in (cache, cache_e):
            if i == 6:
                c.free([2])
            if i == 9:
                c.reserve([1], [64])
        tok.copy_(_step_tokens(3, i))
        graph.replay()
        want = eager.step(tok)
        assert torch.equal(torch.nan_to_num(logits), torch.nan_to_num(want))
        assert torch.equal(dec.wrote, eager.wrote)
        assert torch.isnan(logits).all(1).tolist() == (~dec.wrote).tolist()
        assert dec.wrote.tolist() == [True, i < 2 or i >= 9, i < 6]
        assert cache.lens.tolist() == cache_e.lens.tolist()
    assert cache.lens.tolist() == [49, 35, 0] and torch.equal(cache.pool, cache_e.pool)


class _Pool:
    """Streams of a small pool, and whether a refused operation left all of it alone."""

    def __init__(self, S, M, P, R, rows):
        from lagunalab_b200 import ops
        i = dict(dtype=torch.int32, device="cuda")
        self.pool = torch.randn(2, P, 1, R, 128, device="cuda").to(torch.bfloat16)
        self.table = torch.full((S, M), -1, **i)
        self.lens, self.refs = torch.zeros(S, **i), torch.zeros(P, **i)
        ids = _t(list(range(len(rows))))
        assert ops.pages_reserve(self.table, self.refs, ids, _t(rows), R).tolist()[0] == 0
        self.lens[:len(rows)] = _t(rows)

    def state(self):
        return [t.clone() for t in (self.pool, self.table, self.lens, self.refs)]

    def fork(self, src, dst):
        from lagunalab_b200 import ops
        return ops.pages_fork(self.pool, self.table, self.lens, self.refs, _t(src),
                              _t(dst)).tolist()

    def refused(self, src, dst, code):
        before = self.state()
        assert self.fork(src, dst) == [code, 0]
        assert all(torch.equal(a, b) for a, b in zip(before, self.state()))


@pytest.mark.parametrize("page", [-1, 40, 1 << 30])
@pytest.mark.parametrize("col", [0, 2, 5, 6])  # whole pages, the last whole one, the part-filled one
def test_a_fork_of_rows_without_a_page_is_refused(page, col):
    p = _Pool(8, 9, 40, 16, [33, 6 * 16 + 5, 16])
    good = p.table[1, col].item()
    p.table[1, col] = page
    p.refused([1], [3], 4)
    p.refused([0, 2, 1, 1, 0], [3, 4, 5, 6, 7], 4)
    p.table[1, col] = good
    assert p.fork([0, 2, 1, 1, 0], [3, 4, 5, 6, 7]) == [0, 4]
    assert p.table[5, :6].tolist() == p.table[1, :6].tolist()


def test_a_fork_looks_at_every_source_of_a_long_list():
    """More children than a CTA has threads and sources of very different lengths; the one whole
    page that is missing is the last, the longest, an early or a middle source's."""
    S, M, R, n = 4000, 40, 16, 1500
    rows = [(7 * i) % 48 + 1 for i in range(n)]
    rows[700] = 39 * R + 3
    p = _Pool(S, M, 8000, R, rows)
    src, dst = list(range(n)), list(range(n, 2 * n))
    for s in (n - 1, 700, 4, 1100):
        last = rows[s] // R - 1
        good = p.table[s, last].item()
        p.table[s, last] = -1
        p.refused(src, dst, 4)
        p.table[s, last] = good
    assert p.fork(src, dst) == [0, sum(r % R > 0 for r in rows)]


def test_of_several_faults_the_lowest_code_is_told():
    """Whatever their places in the list: a stream out of range (2) or that holds pages (2), a length
    past the table (3), a page that is missing (4)."""
    S, M, R, n = 2400, 4, 16, 1200
    p = _Pool(S, M, 2000, R, [20] * 900)
    p.lens[5], p.table[7, 0] = M * R + 1, -1
    for i in (0, 40, 800, 1199):
        for j in (1, 30, 900, 1198):
            src, dst = [9] * n, list(range(1000, 1000 + n))
            src[i], src[j] = 7, 5
            p.refused(src, dst, 3)
            src[j] = 9
            p.refused(src, dst, 4)
            dst[j] = 8
            p.refused(src, dst, 2)
            dst[j], src[j] = 1000 + j, -1
            p.refused(src, dst, 2)
    # nothing is free either: 900 streams hold 1,800 pages, 200 are left for 1,200 children
    p.lens[5], p.table[7, 0] = 20, 1999
    p.refused([9] * n, list(range(1000, 1000 + n)), 1)


@pytest.mark.parametrize("S,M", [(65536, 32769), (65536, 65537)])
def test_a_reserve_of_more_pages_than_32_bits_count(S, M):
    """Sums of 2^31 + 2^16 and of 2^32 + 2^16 pages, which are negative or 2^16 in 32 bits."""
    from lagunalab_b200 import ops
    table = torch.full((S, M), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(70000, dtype=torch.int32, device="cuda")
    ids = torch.arange(S, dtype=torch.int32, device="cuda")
    rows = torch.full((S,), M * 16, dtype=torch.int32, device="cuda")
    assert ops.pages_reserve(table, refs, ids, rows, 16).tolist() == [1, 0]
    assert int(table.max()) == -1 and not refs.any()
    rows[1:] = 0  # one stream alone
    rows[0] = 16 * min(M, 60000) - 5
    assert ops.pages_reserve(table, refs, ids, rows, 16).tolist() == [0, min(M, 60000)]
    assert int(refs.sum()) == min(M, 60000) and int((table >= 0).sum()) == min(M, 60000)


def test_a_reserve_of_as_many_rows_as_32_bits_count():
    from lagunalab_b200 import ops
    table = torch.full((2, 2 ** 24 + 1), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(10, dtype=torch.int32, device="cuda")
    call = lambda r: ops.pages_reserve(table, refs, _t([1]), _t([r]), 128).tolist()
    for r in (2 ** 31 - 1, 2 ** 31 - 127, 2 ** 31 - 128):
        assert call(r) == [1, 0]
        assert int(table.max()) == -1 and not refs.any()
    assert call(10 * 128) == [0, 10]


def test_a_refused_call_leaves_the_plan_good():
    """A call of other sizes (through the C interface, which cannot look into the plan) writes nothing;
    the calls of the plan's own sizes that follow give their rows, with waits of every length: short
    parts, parts of many key tiles, last tiles that end inside a page."""
    from lagunalab_b200 import _lib, ops
    from tests.test_paged_attention_gpu import D, _case
    for new, kv, Hq, Hkv in (([20, 7], [90, 7], 4, 2), ([3000, 1, 700], [8001, 20001, 701], 32, 4),
                             ([1], [60001], 3, 3)):
        q, k, v, table, cu, kvt, _ = _case(new, kv, Hq, Hkv, 32, seed=1)
        T, ks = q.shape[0], k.stride()
        plan = ops.prompt_plan(cu, kvt, T, Hq, Hkv, 32)
        want = ops.prompt_attention(q, k, v, table, plan, 0.1)
        out = torch.full_like(q, 7.0)
        for _ in range(3):
            _lib.call("lg_prompt_attention", q.data_ptr(), q.stride(0), q.stride(1), T, Hq, Hkv, D,
                      k.data_ptr(), v.data_ptr(), k.shape[0], 32, ks[0], ks[1], ks[2],
                      table.data_ptr(), len(new) - 1 or 2, table.shape[1], 0.1, None,
                      out.data_ptr(), plan.ptr, 1 << 40, torch.cuda.current_stream().cuda_stream)
            assert (out == 7).all() and plan.status() == 10
            for _ in range(5):
                assert torch.equal(ops.prompt_attention(q, k, v, table, plan, 0.1), want)
        assert plan.status() == 10
        assert plan.update().status() == 0
