"""Replay scoring from the hidden rows, without logits: the same truncated KL and agreement as with logits, within
what the rounding of those to bf16 does, and each token's own loss."""
import numpy as np
import pytest
import torch

from tests._replay_util import CharTokenizer, write_capture
from tests.test_replay_gpu import _tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup(tmp_path_factory):
    from lagunalab_b200 import replay, synth
    d = tmp_path_factory.mktemp("refs")
    args, model, _, _ = _tiny()
    out = d / "s.npz"
    replay.build_ref(model, CharTokenizer(vocab=512), write_capture(d / "s.jsonl"), out, n_actions=1, max_new=2)
    other = synth.decoder(args, seed=5, std=0.05, norm_noise=0.1, router_bias_std=0.3)
    return model, other, out


@pytest.mark.parametrize("chunk", [2048, 16])
def test_fused_score(setup, chunk):
    """A logit rounded to bf16 is off by at most 2^-8 of it, so that a log-probability is off by at most 2^-7 of the
    largest logit; so is a KL, a mean of differences of them."""
    from lagunalab_b200 import replay
    model, other, out = setup
    ref = np.load(out)
    for m in (model, other):
        big = max(float(l.abs().max()) for _, h in replay._hidden(m, ref["ids"], ref["mask"], chunk, None)
                  for l in [m.lm_head(h).float()])
        want, got = replay.score(m, out, chunk=chunk), replay.score(m, out, chunk=chunk, fused=True)
        assert abs(want["kl_top64_mean"] - got["kl_top64_mean"]) <= 2 ** -7 * big
        assert got["assistant_tokens"] == want["assistant_tokens"] == len(ref["pos"])
    assert replay.score(model, out, fused=True)["top1_agree"] >= 0.9  # near-ties apart, the same model
    with pytest.raises(ValueError, match="forward"):
        replay.score(None, out, forward=lambda x, c: x, fused=True)


def test_nll_of_each_token(setup):
    from lagunalab_b200 import replay
    model, _, out = setup
    ref = np.load(out)
    pos, nll = replay.assistant_nll(model, ref["ids"], ref["mask"], chunk=32)
    assert (pos == ref["pos"]).all()
    W = model.lm_head.dequantize().double()
    for i, h in replay._hidden(model, ref["ids"], ref["mask"], 32, None):
        lp = torch.log_softmax(h.double() @ W.T, -1)
        nxt = torch.from_numpy(ref["ids"][pos[i:i + len(h)] + 1].astype(np.int64)).cuda()
        want = -lp.gather(1, nxt[:, None])[:, 0]
        # fp32 sums of 256 products, and the exponentials' 2^-17
        bound = 2.0 ** -16 + 2 * 260 * 2.0 ** -24 * (h.double().abs() @ W.abs().T).amax(1)
        assert ((nll[i:i + len(h)].double() - want).abs() <= bound).all()
