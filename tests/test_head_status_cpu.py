"""The status word of the head's product kernels: what the host refuses. (A wait that runs out is not provoked on a GPU.)"""
import pytest

from lagunalab_b200 import _lib


def test_status_needs_a_place():
    with pytest.raises(ValueError):
        _lib.call("lg_head_status", None, 1)
