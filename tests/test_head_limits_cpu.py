"""Token counts at the end of 32 bits are refused on the host: rounded up to tiles they would be negative."""
import pytest

from lagunalab_b200 import _lib
from tests.test_head_loss_cpu import _fake, _grad, _loss


@pytest.mark.parametrize("T", [2 ** 31 - 1024, 2 ** 31 - 127, 2 ** 31 - 1])
def test_too_many_tokens(T):
    for call in (_loss, _grad):
        with pytest.raises(ValueError):
            call(T=T, H=8, ldx=8, ldw=8, V=1)
        with pytest.raises(ValueError):
            call(T=T, s=_fake(9), b=_fake(10), **({"dw": None} if call is _grad else {}))
