"""The status words of kernels with bounded waits are read behind everything that runs, on torch's (non-blocking) streams too."""
import pytest
import torch

from nimllm_b200 import attention as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("status", [A.decode_tree_status, A.prefill_status, A.matvec_status])
def test_a_status_call_waits_for_side_streams(status):
    assert status() == 0                                   # the first call may load code, which waits by itself
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                     # cycles: 0.1 s
        done = torch.cuda.Event()
        done.record()
    assert not done.query()
    assert status(reset=False) == 0
    assert done.query()
