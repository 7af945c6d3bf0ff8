"""The paged attention's strides are a tensor map's: a broadcast dimension (stride 0) or a negative
stride is refused on the host, before anything looks at the pointers."""
import pytest

from tests.test_paged_cpu import _attn


@pytest.mark.parametrize("kind", ["prompt", "stream"])
@pytest.mark.parametrize("bad", [dict(q_tok=0), dict(q_head=0), dict(pg=0), dict(hd=0), dict(rw=0),
                                 dict(q_tok=-1024), dict(q_head=-128), dict(pg=-2 * 64 * 128),
                                 dict(hd=-64 * 128), dict(rw=-128)])
def test_strides_of_a_tensor_map(kind, bad):
    with pytest.raises(ValueError, match="positive"):
        _attn(kind, **bad)
