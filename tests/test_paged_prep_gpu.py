"""The attention prologue into cache pages (laguna_mlx/laguna.py:94-104 for packed tokens of several
sequences) gives the bits of the one-sequence prologue: q, gates, and every k and v row; rows that no
token has stay as they were."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per_head", [True, False])
@pytest.mark.parametrize("table_rope", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,R", [(32, 4, 128, 64), (6, 3, 64, 16), (5, 1, 256, 128),
                                        (8, 2, 128, 24)])
def test_bits_of_the_one_sequence_prologue(Hq, Hkv, D, R, table_rope, per_head):
    from lagunalab_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(Hq + D)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
    new, kv = [40, 1, 77], [40, 3 * R + 1, 90]  # the newest rows of each sequence
    M = max(-(-n // R) for n in kv) + 1
    P = 3 * M + 2
    table = torch.randperm(P, generator=g, device="cuda")[:3 * M].to(torch.int32).view(3, M)
    T = sum(new)
    order = random.Random(R).sample([(b, kv[b] - new[b] + i) for b in range(3)
                                     for i in range(new[b])], T)  # tokens in any order
    seq, pos = (torch.tensor([o[j] for o in order], dtype=torch.int32, device="cuda")
                for j in range(2))
    qkvg = r(T, (Hq + 2 * Hkv) * D + (Hq if per_head else Hq * D))
    qn, kn = 1 + 0.2 * r(D), 1 + 0.2 * r(D)
    rope = None
    if table_rope:
        half = 32 if D == 64 else D // 4
        rope = (torch.rand(half, generator=g, device="cuda"), 2 * half, 1.25)
    pool = torch.full((P, 2, Hkv, R, D), 3.0, dtype=torch.bfloat16, device="cuda")
    args = (Hq, Hkv, D, qn, kn, 1e-6, 1e4)
    q, gate = ops.attn_prep_pages(qkvg, *args, seq, pos, table, pool[:, 0], pool[:, 1],
                                  gate_per_head=per_head, rope=rope)
    want = torch.full_like(pool, 3.0)
    for b in range(3):
        at = sorted((p, t) for t, (s, p) in enumerate(order) if s == b)
        rows = torch.tensor([t for _, t in at], device="cuda")
        k, v = (torch.zeros(Hkv, M * R, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q1, gate1 = ops.attn_prep(qkvg[rows], *args, k, v, pos=at[0][0], gate_per_head=per_head,
                                  rope=rope)
        assert torch.equal(q[rows], q1.transpose(0, 1))
        assert torch.equal(gate[rows], gate1)
        for p, _ in at:
            page = table[b, p // R].long()
            want[page, 0, :, p % R], want[page, 1, :, p % R] = k[:, p], v[:, p]
    assert torch.equal(pool, want)


def test_a_token_without_a_page_leaves_no_row():
    from lagunalab_b200 import ops
    Hq, Hkv, D, R, P, M = 8, 2, 128, 16, 6, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    qkvg = torch.randn(8, (Hq + 2 * Hkv) * D + Hq, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = i32([[3, -1], [P, 1]])
    # a page, no page, past the table, a page outside the pool, sequences that are not there, before 0
    seq, pos = i32([0, 0, 0, 1, -1, 2, 1, 1]), i32([5, 16, 32, 3, 0, 0, -1, 2 ** 31 - 1])
    k, v = (torch.full((P, Hkv, R, D), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, gate = ops.attn_prep_pages(qkvg, Hq, Hkv, D, w, w, 1e-6, 1e4, seq, pos, table, k, v)
    assert torch.isfinite(q).all() and torch.isfinite(gate).all()
    for t in (k, v):
        assert not (t[3, :, 5] == 3).all()
        t[3, :, 5] = 3
        assert (t == 3).all()
