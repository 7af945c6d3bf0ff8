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
