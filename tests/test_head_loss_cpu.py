"""What the head's loss and gradient refuse on the host, before anything looks at the pointers."""
import ctypes

import pytest

from lagunalab_b200 import _lib


def _fake(n=1):
    return ctypes.c_void_p(0x1000 * n)  # never dereferenced: the checks fail first


def _loss(x=_fake(), ldx=64, T=4, H=64, w=_fake(2), ldw=64, s=None, b=None, V=300, ids=_fake(3), K=1,
          loss=_fake(4), lse=_fake(5), ws=_fake(6), nb=1 << 40):
    return _lib.call("lg_head_loss", x, ldx, T, H, w, ldw, s, b, V, ids, None, K, loss, lse, None, ws, nb,
                     None)


def _grad(x=_fake(), ldx=64, T=4, H=64, w=_fake(2), ldw=64, s=None, b=None, V=300, ids=_fake(3), K=1,
          lse=_fake(5), g=_fake(5), dx=_fake(7), dw=_fake(8), ws=_fake(6), nb=1 << 40):
    return _lib.call("lg_head_loss_grad", x, ldx, T, H, w, ldw, s, b, V, ids, None, K, lse, g, dx, dw, ws,
                     nb, None)


BAD = [dict(T=-1), dict(V=0), dict(K=0), dict(K=65), dict(H=60), dict(H=0), dict(x=None), dict(w=None),
       dict(ids=None), dict(x=ctypes.c_void_p(0x1008)), dict(w=ctypes.c_void_p(0x1008)), dict(ldx=56),
       dict(ldx=68), dict(ldx=-64), dict(ldw=0), dict(ldw=68), dict(s=_fake(9)), dict(b=_fake(9)),
       dict(s=_fake(9), b=_fake(10), ldw=128), dict(s=_fake(9), b=_fake(10), H=72, ldx=72, ldw=72),
       dict(T=1 << 30, V=1 << 30)]


@pytest.mark.parametrize("bad", BAD + [dict(loss=None), dict(lse=None)])
def test_loss_refuses(bad):
    with pytest.raises(ValueError):
        _loss(**bad)


@pytest.mark.parametrize("bad", BAD + [dict(dx=None, dw=None), dict(lse=None), dict(g=None),
                                       dict(dx=ctypes.c_void_p(0x1008)), dict(dw=ctypes.c_void_p(0x1008)),
                                       dict(s=_fake(9), b=_fake(10))])
def test_gradient_refuses(bad):
    with pytest.raises(ValueError):
        _grad(**bad)


@pytest.mark.parametrize("call", [_loss, _grad])
def test_workspace(call):
    for bad in (dict(ws=None), dict(nb=100), dict(ws=ctypes.c_void_p(0x1010))):
        with pytest.raises(_lib.LagunaError) as e:
            call(**bad)
        assert e.value.code == _lib.LG_ERR_WORKSPACE


def test_workspace_sizes():
    L = _lib.lib()
    assert L.lg_head_loss_workspace_bytes(1, 64, 300, 1, 16, 0) % 256 == 0
    # a head of the benchmark's size: no [T, V] array in either
    assert L.lg_head_loss_workspace_bytes(8192, 2048, 100352, 1, 16, 0) < 64 << 20
    assert L.lg_head_loss_grad_workspace_bytes(8192, 2048, 100352, 1, 16, 1, 1) < 768 << 20
    assert L.lg_head_loss_grad_workspace_bytes(1, 2048, 100352, 64, 4, 1, 0) < 520 << 20  # a piece's weights


def test_which_form_a_4bit_loss_takes():
    """From the codes (a small workspace) for up to 32 tokens, and further where unpacking the weights costs more."""
    def codes(T, H, V):
        return _lib.lib().lg_head_loss_workspace_bytes(T, H, V, 1, 4, 0) < V * H
    assert all(codes(T, H, V) for T in (1, 32) for H in (64, 2048) for V in (6264, 100352))
    assert all(codes(T, 2048, 100352) for T in (33, 128, 129, 256, 384))
    assert not any(codes(T, 64, V) for T in (128, 384) for V in (6264, 77689))
    assert not any(codes(T, H, V) for T in (385, 8192) for H in (64, 2048) for V in (6264, 100352))
