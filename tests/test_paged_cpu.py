"""The paged cache's entry points refuse bad arguments on the host, before any launch (no GPU needed:
the pointers are never dereferenced), and their plan and workspace sizes are host arithmetic."""
import ctypes

import pytest
import torch

from lagunalab_b200 import _lib, ops


def _fake(n=1):
    return ctypes.c_void_p(0x1000 * n)


def _attn(kind="prompt", q=None, q_tok=1024, q_head=128, T=5, Hq=8, Hkv=2, D=128, k=None, P=9, R=64,
          pg=2 * 64 * 128, hd=64 * 128, rw=128, table=None, B=2, M=4, scale=0.1, gate=None, out=None,
          plan=None, nb=1 << 40):
    f = lambda x: _fake() if x is None else x
    out = _fake(1000) if out is None else out
    a = [f(q), q_tok, q_head, T, Hq, Hkv, D, f(k), _fake(), P, R, pg, hd, rw, f(table)]
    b = [M, scale, gate, f(out), f(plan), nb, None]
    if kind == "prompt":
        return _lib.call("lg_prompt_attention", *a, B, *b)
    return _lib.call("lg_stream_attention", *a, *b)


@pytest.mark.parametrize("kind", ["prompt", "stream"])
@pytest.mark.parametrize("bad,match", [
    (dict(D=64), "head_dim"), (dict(Hq=34), "group"), (dict(Hq=7), "heads"), (dict(Hkv=0), "heads"),
    (dict(R=48), "rows"), (dict(R=256), "rows"), (dict(P=0), "pages"), (dict(M=0), "pages"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(q=ctypes.c_void_p(0)), "NULL"),
    (dict(table=ctypes.c_void_p(0)), "NULL"), (dict(out=ctypes.c_void_p(0)), "NULL"),
    (dict(q=ctypes.c_void_p(0x1008)), "multiples of 16"), (dict(q_tok=1025), "multiples of 16"),
    (dict(rw=132), "multiples of 16"), (dict(out=ctypes.c_void_p(0x1008)), "multiples of 16"),
    (dict(T=-1), "tokens"), (dict(T=1 << 30), "tokens"), (dict(out=_fake()), "shares memory"),
    (dict(q=_fake(3), out=_fake(2)), "shares memory")])
def test_attention_refuses(kind, bad, match):
    with pytest.raises(ValueError, match=match):
        _attn(kind, **bad)


@pytest.mark.parametrize("kind", ["prompt", "stream"])
def test_attention_needs_its_plan(kind):
    for bad in (dict(nb=256), dict(plan=ctypes.c_void_p(0x1010)), dict(plan=ctypes.c_void_p(0))):
        with pytest.raises(_lib.LagunaError) as e:
            _attn(kind, **bad)
        assert e.value.code == _lib.LG_ERR_WORKSPACE


def test_no_token_is_no_work():
    assert _attn("prompt", T=0) == _lib.LG_OK  # returns before it looks at any pointer


def test_plans_refuse():
    L = _lib.lib()
    plan = lambda B=3, T=9, Hq=8, Hkv=2, R=16, W=0, cu=_fake(), kv=_fake(), nb=1 << 40: _lib.call(
        "lg_prompt_plan", cu, kv, B, T, Hq, Hkv, R, W, _fake(), nb, None)
    for bad, match in ((dict(B=0), "sequences"), (dict(T=-1), "tokens"), (dict(Hq=9), "heads"),
                       (dict(R=8), "rows"), (dict(W=-1), "window"),
                       (dict(cu=ctypes.c_void_p(0)), "NULL"), (dict(kv=ctypes.c_void_p(0)), "NULL")):
        with pytest.raises(ValueError, match=match):
            plan(**bad)
    with pytest.raises(_lib.LagunaError) as e:
        plan(nb=64)
    assert e.value.code == _lib.LG_ERR_WORKSPACE
    with pytest.raises(ValueError, match="prefix"):
        _lib.call("lg_stream_plan", _fake(), 3, 8, 2, 16, -1, 0, _fake(), 1 << 40, None)
    a, b = L.lg_prompt_plan_bytes(64, 2, 8, 2), L.lg_prompt_plan_bytes(1 << 20, 2, 8, 2)
    assert 0 < a < b and a % 256 == 0
    assert 0 < L.lg_stream_plan_bytes(1, 8, 2) < L.lg_stream_plan_bytes(512, 8, 2)
    assert L.lg_prompt_plan_bytes(64, 2, 9, 2) == 0 and L.lg_stream_plan_bytes(0, 8, 2) == 0


def test_page_operations_refuse():
    S, M, P, R = 4, 3, 10, 16
    big = 1 << 30
    res = lambda **k: _lib.call("lg_pages_reserve", *({**dict(
        table=_fake(), refs=_fake(), S=S, M=M, P=P, R=R, ids=_fake(), rows=_fake(), n=2,
        status=_fake(), ws=_fake(), nb=big, st=None), **k}).values())
    free = lambda **k: _lib.call("lg_pages_free", *({**dict(
        table=_fake(), lens=_fake(), refs=_fake(), S=S, M=M, P=P, ids=_fake(), n=2, status=_fake(),
        st=None), **k}).values())
    fork = lambda **k: _lib.call("lg_pages_fork", *({**dict(
        pool=_fake(), planes=2, H=1, R=R, rb=256, table=_fake(), lens=_fake(), refs=_fake(), S=S, M=M,
        P=P, src=_fake(), dst=_fake(), n=2, status=_fake(), ws=_fake(), nb=big, st=None),
        **k}).values())
    comp = lambda **k: _lib.call("lg_pages_compact", *({**dict(
        pool=_fake(), planes=2, H=1, R=R, rb=256, table=_fake(), refs=_fake(), S=S, M=M, P=P,
        status=_fake(), ws=_fake(), nb=big, st=None), **k}).values())
    null = ctypes.c_void_p(0)
    for f, bads in ((res, [dict(table=null), dict(n=5), dict(n=-1), dict(ids=null), dict(R=0),
                           dict(P=0), dict(S=65537)]),
                    (free, [dict(lens=null), dict(n=5), dict(ids=null), dict(status=null)]),
                    (fork, [dict(pool=null), dict(pool=ctypes.c_void_p(0x1008)), dict(rb=8),
                            dict(planes=0), dict(n=5), dict(src=null), dict(status=null)]),
                    (comp, [dict(pool=null), dict(rb=24), dict(M=0), dict(status=null)])):
        for bad in bads:
            with pytest.raises(ValueError):
                f(**bad)
    for f in (res, fork, comp):
        with pytest.raises(_lib.LagunaError) as e:
            f(nb=16)
        assert e.value.code == _lib.LG_ERR_WORKSPACE


def test_prologue_refuses():
    call = lambda **k: _lib.call("lg_attn_prep_pages", *({**dict(
        qkvg=_fake(), T=2, Hq=4, Hkv=2, D=128, qn=_fake(), kn=_fake(), eps=1e-6, theta=1e4,
        seq=_fake(), pos=_fake(), table=_fake(), B=2, M=3, P=9, R=16, page=2 * 16 * 128, gate=1,
        q=_fake(), kp=_fake(), vp=_fake(), go=_fake(), inv=None, rot=0, ms=1.0, st=None),
        **k}).values())
    null = ctypes.c_void_p(0)
    for bad, match in ((dict(D=96), "head_dim"), (dict(R=0), "rows"), (dict(page=100), "pages"),
                       (dict(seq=null), "NULL"), (dict(kp=null), "NULL"), (dict(rot=96), "rotary"),
                       (dict(rot=64), "frequency")):
        with pytest.raises(ValueError, match=match):
            call(**bad)
    assert call(T=0) == _lib.LG_OK


def test_python_surface_refuses_cpu_tensors():
    t = torch.zeros(2, 3, dtype=torch.int32)
    one = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.pages_reserve(t, one, one, one, 16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.pages_fork(torch.zeros(1, 2, 1, 16, 128), t, one, one, one, one)
    with pytest.raises(ValueError, match="CUDA"):
        ops.stream_plan(one, 8, 2, 16)
