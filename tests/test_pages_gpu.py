"""The page operations of a paged K/V cache (reserve, fork, free, compact; no counterpart in the
reference, whose caches hold one sequence, laguna_mlx/cache.py:66-157) against a host model of
the same bookkeeping: tables, counts and lengths exactly, and every row of every plane."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Host:
    """The bookkeeping in Python lists."""

    def __init__(self, S, M, P, R):
        self.M, self.P, self.R = M, P, R
        self.table = [[-1] * M for _ in range(S)]
        self.lens, self.refs = [0] * S, [0] * P

    def take(self, n):
        free = [p for p in range(self.P) if self.refs[p] == 0][:n]
        assert len(free) == n
        for p in free:
            self.refs[p] = 1
        return free

    def reserve(self, ids, rows):
        for s, r in zip(ids, rows):
            have = sum(p >= 0 for p in self.table[s])
            new = self.take(max(0, -(-r // self.R) - have))
            self.table[s][have:have + len(new)] = new

    def fork(self, pool, src, dst):
        old = pool.clone()
        for s, d in zip(src, dst):
            n = self.lens[s]
            whole, part = divmod(n, self.R)
            row = self.table[s][:whole]
            for p in row:
                self.refs[p] += 1
            if part:
                new = self.take(1)[0]
                pool[..., new, :, :part, :] = old[..., self.table[s][whole], :, :part, :]
                row = row + [new]
            self.table[d] = row + [-1] * (self.M - len(row))
            self.lens[d] = n

    def free(self, ids):
        for s in ids:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s], self.lens[s] = [-1] * self.M, 0

    def compact(self, pool):
        n = sum(r > 0 for r in self.refs)
        holes = [p for p in range(n) if self.refs[p] == 0]
        name = dict(zip([p for p in range(n, self.P) if self.refs[p] > 0], holes))
        for a, b in name.items():
            pool[..., b, :, :, :] = pool[..., a, :, :, :]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[name.get(p, p) for p in row] for row in self.table]


class Device:
    def __init__(self, S, M, P):
        i = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((S, M), -1, **i)
        self.lens, self.refs = torch.zeros(S, **i), torch.zeros(P, **i)


def _t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _same(h, d):
    assert d.table.tolist() == h.table
    assert d.lens.tolist() == h.lens
    assert d.refs.tolist() == h.refs


@pytest.mark.parametrize("S,M,P,R,shape,dtype", [
    (7, 5, 40, 16, (2, 3), torch.bfloat16), (3, 1, 3, 64, (1, 1), torch.bfloat16),
    (40, 9, 1500, 32, (1, 2), torch.int32), (5, 70, 300, 128, (6, 1), torch.bfloat16)])
def test_random_life_of_a_pool(S, M, P, R, shape, dtype):
    """Streams come, grow, fork, go; the pool is compacted now and then."""
    from lagunalab_b200 import ops
    rng = random.Random(S * M)
    planes, H = shape
    D = 128 if dtype == torch.bfloat16 else 32
    pool = torch.randint(0, 1 << 15, (planes, P, H, R, D), dtype=torch.int32, device="cuda")
    pool = pool.to(dtype) if dtype == torch.int32 else pool.to(torch.int16).view(dtype)
    ref = pool.clone()
    h, d = Host(S, M, P, R), Device(S, M, P)
    for step in range(60):
        empty = [s for s in range(S) if not h.lens[s] and h.table[s][0] < 0]
        held = [s for s in range(S) if h.lens[s]]
        free = sum(r == 0 for r in h.refs)
        what = rng.choice(["grow", "grow", "fork", "fork", "free", "compact"])
        if what == "grow":
            ids = rng.sample(range(S), rng.randint(1, S))
            rows = [rng.randint(h.lens[s], M * R) for s in ids]
            need = sum(max(0, -(-r // R) - sum(p >= 0 for p in h.table[s])) for s, r in zip(ids, rows))
            st = ops.pages_reserve(d.table, d.refs, _t(ids), _t(rows), R)
            if need > free:
                assert st.tolist() == [1, 0]
            else:
                assert st.tolist() == [0, need]
                h.reserve(ids, rows)
                for s, r in zip(ids, rows):
                    h.lens[s] = r
                d.lens[torch.tensor(ids, device="cuda")] = _t(rows)
        elif what == "fork" and held and empty:
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(held) for _ in dst]
            need = sum(h.lens[s] % R > 0 for s in src)
            st = ops.pages_fork(pool, d.table, d.lens, d.refs, _t(src), _t(dst))
            if need > free:
                assert st.tolist() == [1, 0]
            else:
                assert st.tolist() == [0, need]
                h.fork(ref, src, dst)
        elif what == "free":
            ids = rng.sample(range(S), rng.randint(1, max(1, S // 2)))
            assert ops.pages_free(d.table, d.lens, d.refs, _t(ids)).tolist() == [0, len(ids)]
            h.free(ids)
        elif what == "compact":
            n = sum(r > 0 for r in h.refs)
            moved = sum(r > 0 for r in h.refs[n:])
            assert ops.pages_compact(pool, d.table, d.refs).tolist() == [0, moved]
            h.compact(ref)
        _same(h, d)
        view = torch.int32 if dtype == torch.int32 else torch.int16
        assert torch.equal(pool.view(view), ref.view(view)), (step, what)


def test_refusals_change_nothing():
    from lagunalab_b200 import ops
    S, M, P, R = 6, 4, 12, 16
    d = Device(S, M, P)
    pool = torch.randn(2, P, 1, R, 128, device="cuda").to(torch.bfloat16)
    assert ops.pages_reserve(d.table, d.refs, _t([0, 1]), _t([40, 16]), R).tolist() == [0, 4]
    d.lens[:2] = _t([40, 16])
    before = [t.clone() for t in (pool, d.table, d.lens, d.refs)]

    def refused(status, code):
        assert status.tolist() == [code, 0]
        assert all(torch.equal(a, b) for a, b in zip(before, (pool, d.table, d.lens, d.refs)))

    fork = lambda s, t: ops.pages_fork(pool, d.table, d.lens, d.refs, _t(s), _t(t))
    res = lambda i, r: ops.pages_reserve(d.table, d.refs, _t(i), _t(r), R)
    refused(fork([0, 0], [2, 2]), 2)      # a child twice
    refused(fork([0], [1]), 2)            # a child that holds pages
    refused(fork([0, 2], [2, 3]), 2)      # a child that is a source too
    refused(fork([6], [2]), 2)
    refused(fork([0], [-1]), 2)
    refused(res([2, 2], [1, 1]), 2)
    refused(res([0, 6], [1, 1]), 2)
    refused(res([2], [M * R + 1]), 3)
    refused(res([2], [-1]), 3)
    refused(res([2, 3, 4], [M * R, M * R, 1]), 1)
    refused(ops.pages_free(d.table, d.lens, d.refs, _t([0, 0])), 2)
    refused(ops.pages_free(d.table, d.lens, d.refs, _t([7])), 2)
    d.table[0, 2] = P  # a part-filled last page outside the pool
    before[1] = d.table.clone()
    refused(fork([0], [2]), 4)


def test_empty_lists_and_empty_streams():
    from lagunalab_b200 import ops
    S, M, P, R = 3, 2, 4, 32
    d = Device(S, M, P)
    pool = torch.zeros(1, P, 1, R, 128, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.pages_reserve(d.table, d.refs, none, none, R).tolist() == [0, 0]
    assert ops.pages_free(d.table, d.lens, d.refs, none).tolist() == [0, 0]
    assert ops.pages_fork(pool, d.table, d.lens, d.refs, none, none).tolist() == [0, 0]
    assert ops.pages_compact(pool, d.table, d.refs).tolist() == [0, 0]
    assert ops.pages_fork(pool, d.table, d.lens, d.refs, _t([0]), _t([1])).tolist() == [0, 0]
    assert ops.pages_free(d.table, d.lens, d.refs, _t([0, 1, 2])).tolist() == [0, 3]
    assert d.table.tolist() == [[-1] * M] * S and d.refs.tolist() == [0] * P


def test_lists_longer_than_a_cta():
    """More streams in one call than a CTA has threads, free pages far into the pool, and the same
    operations captured into a graph and replayed."""
    from lagunalab_b200 import ops
    rng = random.Random(5)
    S, M, P, R, n = 3600, 2, 9000, 16, 1500
    pool = torch.randint(0, 1 << 15, (1, P, 1, R, 4), dtype=torch.int32, device="cuda")
    ref = pool.clone()
    h, d = Host(S, M, P, R), Device(S, M, P)
    order = rng.sample(range(S), 2 * n)
    src, dst = order[:n], order[n:]
    rows = [rng.randint(0, M * R) for _ in src]
    need = sum(-(-r // R) for r in rows)
    assert ops.pages_reserve(d.table, d.refs, _t(src), _t(rows), R).tolist() == [0, need]
    h.reserve(src, rows)
    for s, r in zip(src, rows):
        h.lens[s] = r
    d.lens[torch.tensor(src, device="cuda")] = _t(rows)
    _same(h, d)
    parents = [rng.choice(src) for _ in dst]
    ids = [_t(parents), _t(dst), _t(src[::2])]
    kept = [t.clone() for t in (pool, d.table, d.lens, d.refs)]

    def life():
        return (ops.pages_fork(pool, d.table, d.lens, d.refs, ids[0], ids[1]),
                ops.pages_free(d.table, d.lens, d.refs, ids[2]),
                ops.pages_compact(pool, d.table, d.refs))

    first = [st.tolist() for st in life()]
    h.fork(ref, parents, dst)
    h.free(src[::2])
    live = sum(r > 0 for r in h.refs)
    assert first == [[0, sum(h.lens[s] % R > 0 for s in dst)], [0, len(src[::2])],
                     [0, sum(r > 0 for r in h.refs[live:])]]
    h.compact(ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = life()
    for replays in range(3):
        _same(h, d)
        assert torch.equal(pool, ref)
        for t, k in zip((pool, d.table, d.lens, d.refs), kept):
            t.copy_(k)
        graph.replay()
        assert [st.tolist() for st in again] == first


def test_a_pool_past_32_bit_offsets():
    """Planes more than 2^32 bytes apart: a fork and a compaction move the last plane's rows."""
    from lagunalab_b200 import ops
    planes, P, R = 3, 9000, 128
    pool = torch.zeros(planes, P, 1, R, 1024, dtype=torch.bfloat16, device="cuda")
    d = Device(2, 2, P)
    d.refs[:] = 1
    d.refs[7], d.refs[11] = 0, 0
    d.table[0, 0] = P - 1
    d.lens[0] = 100
    pool[:, P - 1, 0] = torch.randn(planes, R, 1024, device="cuda").to(torch.bfloat16)
    want = pool[:, P - 1, 0].clone()
    assert ops.pages_fork(pool, d.table, d.lens, d.refs, _t([0]), _t([1])).tolist() == [0, 1]
    assert d.table[1].tolist() == [7, -1] and d.lens[1].item() == 100
    assert torch.equal(pool[:, 7, 0, :100], want[:, :100])
    assert not pool[:, 7, 0, 100:].any()
    assert ops.pages_compact(pool, d.table, d.refs).tolist() == [0, 1]
    assert d.table[0].tolist() == [11, -1]
    assert torch.equal(pool[:, 11, 0], want)
