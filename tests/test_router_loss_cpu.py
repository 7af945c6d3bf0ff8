"""What the router's balance loss and gradient refuse on the host, before anything looks at the pointers."""
import ctypes

import pytest

from lagunalab_b200 import _lib


def _fake(n=1):
    return ctypes.c_void_p(0x1000 * n)  # never dereferenced: the checks fail first


def _balance(logits=_fake(), inds=_fake(), T=4, E=16, k=2, fn=0, loss=_fake(), counts=_fake(), probs=_fake(),
             tokens=_fake(), ws=_fake(), nb=1 << 30):
    return _lib.call("lg_router_balance", logits, inds, None, T, E, k, fn, loss, counts, probs, tokens, ws, nb,
                     None)


def _grad(logits=_fake(), inds=_fake(), dw=_fake(), T=4, E=16, k=2, fn=0, counts=_fake(), tokens=_fake(),
          out=_fake()):
    return _lib.call("lg_router_grad", logits, inds, dw, None, T, E, k, 1, fn, counts, tokens, 0.1, out, None)


BAD = [dict(T=-1), dict(E=0), dict(E=257), dict(k=0), dict(k=33), dict(fn=2), dict(logits=None),
       dict(inds=None), dict(counts=None), dict(tokens=None)]


@pytest.mark.parametrize("bad", BAD + [dict(loss=None), dict(probs=None)])
def test_balance_refuses(bad):
    with pytest.raises(ValueError):
        _balance(**bad)


@pytest.mark.parametrize("bad", BAD + [dict(out=None), dict(dw=None, counts=None, tokens=None)])
def test_gradient_refuses(bad):
    with pytest.raises(ValueError):
        _grad(**bad)


def test_workspace():
    need = _lib.lib().lg_router_balance_workspace_bytes(4000, 16)
    for bad in (dict(ws=None), dict(nb=need - 1), dict(ws=ctypes.c_void_p(0x1010))):
        with pytest.raises(_lib.LagunaError) as e:
            _balance(T=4000, **bad)
        assert e.value.code == _lib.LG_ERR_WORKSPACE
