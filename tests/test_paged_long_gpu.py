"""Paged attention where one CTA's part spans many columns of the table (the loader holds 32 at a time)
and many turns of the ring of key tiles: tables of randomly permuted pages over thousands of rows, in
all forms of a row tile, against the definition in 64 bits.

Tolerance: the one of tests/test_paged_attention_gpu.py, 2^-6 A of which 3.5 * 2^-8 A are taken by
the roundings to bf16 and the errors of the scores. What grows with the rows are the fp32 sums. The
weights' sum: at most 481 key tiles and 128 keys within one, (481 + 128) 2^-24 < 2^-14 relative. The
output: eight products of 16 keys a key tile, each of which adds to the sum with an error of at most
three steps of it (the products lined up, then cut off), 481 * 8 * 3 * 2^-23 A = 0.36 * 2^-8 A.
Together 3.9 * 2^-8 A, and the bound is 4 * 2^-8 A."""
import pytest
import torch

from tests.test_paged_attention_gpu import D, _exact, _near

pytestmark = pytest.mark.gpu


def _inputs(new, kv, Hq, Hkv, R, prefix, seed):
    """Pages that sequences share in different orders, a last page of each one's own with NaN past its
    rows; the first prefix / R columns are the same for all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, need = len(kv), [-(-n // R) for n in kv]
    P = max(need) + 5
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)
    k, v = r(P + B, Hkv, R, D), r(P + B, Hkv, R, D)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(P, generator=g, device="cuda")
    first, rest = order[:prefix // R], order[prefix // R:]
    for b, n in enumerate(need):
        own = rest[torch.randperm(len(rest), generator=g, device="cuda")]
        table[b, :n] = torch.cat([first, own])[:n].to(torch.int32)
        table[b, n - 1] = P + b
        for t in (k, v):
            t[P + b, :, kv[b] - (n - 1) * R:] = float("nan")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return r(sum(new), Hq, D), k, v, table, i32([sum(new[:i]) for i in range(B + 1)]), i32(kv)


def _columns(segments, R):
    """Table columns that a CTA's share spans at least: (segments, key tiles each, cost of a tile)."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    cost = sum(n * (6 + t * w) for n, t, w in segments)
    return (cost / sms - 6) / max(w for _, _, w in segments) * 128 / R


# new tokens a sequence, sequences, rows held, Hq, Hkv, R
PROMPTS = [
    (512, 1, 12000, 32, 4, 16),  # pairs of row tiles
    (1000, 1, 20000, 32, 4, 128),
    (300, 2, 24000, 6, 3, 32),
    (10, 40, 12000, 32, 4, 16),  # two neighbouring heads
    (3, 80, 20000, 16, 2, 128),
    (16, 24, 9000, 8, 1, 16),  # halves of the key tiles
    (5, 64, 20000, 15, 3, 128),
    (1, 40, 7000, 3, 3, 64),
]


@pytest.mark.parametrize("n,B,rows,Hq,Hkv,R", PROMPTS)
def test_long_parts_of_prompts(n, B, rows, Hq, Hkv, R):
    from lagunalab_b200 import ops
    new, kv = [n] * B, [rows - 37 * b for b in range(B)]
    tq = 128 // (Hq // Hkv)
    pair = n > tq
    duo = not pair and Hkv % 2 == 0
    segments = [(Hkv // (1 + duo) * -(-n // (2 * tq)), m // 128, 4 if pair or duo else 2) for m in kv]
    assert _columns(segments, R) > 64  # at least two steps to the next 32 columns
    q, k, v, table, cu, kvt = _inputs(new, kv, Hq, Hkv, R, 0, seed=n + R)
    plan = ops.prompt_plan(cu, kvt, n * B, Hq, Hkv, R)
    got = ops.prompt_attention(q, k, v, table, plan, D ** -0.5)
    out, A = _exact(q, k, v, table, new, kv, D ** -0.5, None, 0)
    _near(got, out, A, n * B)
    assert plan.status() == 0


# streams, prefix, rows of its own, Hq, Hkv, R
STREAMS = [
    (64, 32768, 40, 32, 4, 16),  # prefix: pairs; own keys: two neighbouring heads
    (300, 40960, 30, 32, 4, 128),
    (200, 24576, 60, 12, 3, 16),  # own keys in halves
    (12, 60 * 1024, 90, 64, 8, 16),  # prefix: two neighbouring heads
    (9, 60 * 1024, 90, 28, 7, 16),  # prefix in halves
    (64, 0, 12000, 32, 4, 16),
    (64, 0, 20000, 8, 2, 64),
    (48, 0, 9000, 15, 5, 16),
    (96, 0, 20000, 5, 5, 128),
]


@pytest.mark.parametrize("B,prefix,own,Hq,Hkv,R", STREAMS)
def test_long_parts_of_streams(B, prefix, own, Hq, Hkv, R):
    from lagunalab_b200 import ops
    kv = [prefix + own - (29 * b) % (own // 2) for b in range(B)]
    tq = 128 // (Hq // Hkv)
    if prefix:  # the prefix's row tiles come first and have their CTAs to themselves
        pair = B > tq
        duo = not pair and Hkv % 2 == 0
        segments = [(Hkv // (1 + duo) * -(-B // (2 * tq)), prefix // 128, 4 if pair or duo else 2)]
    else:
        segments = [(Hkv // (2 - Hkv % 2), n // 128, 4 - Hkv % 2 * 2) for n in kv]
    assert _columns(segments, R) > 64
    q, k, v, table, _, kvt = _inputs([1] * B, kv, Hq, Hkv, R, prefix, seed=B + R)
    plan = ops.stream_plan(kvt, Hq, Hkv, R, prefix=prefix)
    got = ops.stream_attention(q, k, v, table, plan, D ** -0.5)
    out, A = _exact(q, k, v, table, [1] * B, kv, D ** -0.5, None, 0)
    _near(got, out, A, B)
    assert plan.status() == 0


def test_a_query_broadcast_over_heads_or_tokens():
    from lagunalab_b200 import ops
    q, k, v, table, cu, kvt = _inputs([7, 40], [300, 90], 8, 2, 32, 0, seed=3)
    plan = ops.prompt_plan(cu, kvt, 47, 8, 2, 32)
    for x in (q[:, :1].expand(47, 8, D), q[:1].expand(47, 8, D)):
        want = ops.prompt_attention(x.contiguous(), k, v, table, plan, D ** -0.5)
        assert torch.equal(ops.prompt_attention(x, k, v, table, plan, D ** -0.5), want)
