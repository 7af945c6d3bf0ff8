"""The status word of the head's product kernels stays 0 over every form: no wait of theirs runs out."""
import pytest
import torch

from lagunalab_b200 import ops
from tests.test_head_short_calls_gpu import SIZES, run
from tests.test_head_loss_gpu import make

pytestmark = pytest.mark.gpu


def test_no_wait_runs_out():
    ops.head_status()
    for T, V, H, bits, K in SIZES + [(700, 5000, 1024, 16, 1), (3000, 700, 128, 16, 2), (300, 5000, 1024, 4, 1)]:
        run(*make(T, V, H, bits=bits, K=K, seed=T))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(*make(20, 3000, 128, bits=4))
    assert ops.head_status(reset=False) == ops.head_status(torch.device("cuda", 0)) == 0
