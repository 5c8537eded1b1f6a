"""CPU: calls over log-probabilities that were once taken and must be refused, and refused ones that must be taken, on the host and before anything is launched."""
import ctypes as C

import pytest
import torch

import gpu_cases as gc
from test_loss_args import AT, rows_of


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a machine without a GPU is meant: what is not refused goes no further than the launch")


@pytest.mark.parametrize("entropy", [None, AT])
def test_scores_refuse_a_workspace_that_is_too_small_or_misaligned(entropy):
    """None at all is a choice (a workgroup a row); one that cannot be used is a mistake, which the other calls refuse too."""
    m = gc.pkg()
    lib, r = m.lib(), rows_of(m, rows=2, vocab=151936, row_stride=151936)
    need = lib.ws_token_logprobs_workspace(C.byref(r))
    assert need > 0
    call = lambda work, size: lib.ws_token_logprobs(None, C.byref(r), AT, AT, entropy, work, size)  # noqa: E731
    assert call(AT, need - 1) == call(AT, 0) == call(AT + 4, need) == m.E_WORKSPACE
    assert call(None, 0) not in (m.E_WORKSPACE, m.E_INVALID) and call(AT, need) not in (m.E_WORKSPACE, m.E_INVALID) and call(None, need) not in (m.E_WORKSPACE, m.E_INVALID)
