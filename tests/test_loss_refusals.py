"""CPU: calls over log-probabilities that were once taken and must be refused, and refused ones that must be taken, on the host and before anything is launched."""
import ctypes as C

import pytest
import torch

import gpu_cases as gc
from test_loss_args import AT, policy_of, rows_of


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


# (gradient's place behind the logits in elements, stride of the logits, of the gradient, rows): vocab 100
APART = [(100, 200, 200, 4), (150, 300, 300, 4), (-100, 200, 200, 4), (-200, 300, 300, 4), (100 + 200, 200, 200, 4), (0, 100, 500, 1), (0, 500, 100, 1), (400, 100, 100, 4), (100, 100, 100, 1)]
OVER = [(99, 200, 200, 4), (101, 200, 200, 4), (-99, 200, 200, 4), (-101, 200, 200, 4), (100, 199, 199, 4), (299, 200, 200, 4), (100, 200, 201, 4), (0, 200, 201, 4), (99, 500, 500, 1), (-99, 100, 100, 1),
        (0, 1 << 63, 100, 3), (-400, 100, 1 << 62, 4), (400, 1 << 62, 100, 5)]


@pytest.mark.parametrize("dtype,each", [(0, 4), (1, 2)])
def test_gradients_between_the_rows_of_the_logits(dtype, each):
    """Memory that does not overlap the logits is taken, also between their rows; what overlaps them is refused, also where a matrix's size passes 64 bits."""
    m = gc.pkg()
    lib, p, at = m.lib(), policy_of(m), AT << 8
    for taken, places in ((True, APART), (False, OVER)):
        for off, stride, d_stride, rows in places:
            r = rows_of(m, logits=at, dtype=dtype, rows=rows, row_stride=stride)
            d = at + off * each
            codes = (lib.ws_token_logprobs_grad(None, C.byref(r), AT, AT, None, None, d, d_stride),
                     lib.ws_policy_loss_rows(None, C.byref(r), C.byref(p), AT, AT, None, d, d_stride, AT, 1 << 20))
            assert all((c != m.E_INVALID) == taken for c in codes), (off, stride, d_stride, rows, codes)


def test_sizes_past_32_bits_are_refused():
    """A C structure's entry keeps the lower 32 bits of a number: 2^32 + 3 rows would be three. (Tensors without memory: what is looked at first is the size.)"""
    m = gc.pkg()
    many = (1 << 32) + 3
    empty = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    ids, v, long = empty(3, dtype=torch.int32), empty(3), empty(many)
    calls = []
    for x in (empty(many, 1), empty(1, many), empty(1 << 20, 3), empty(3, 1 << 20)):
        calls += [lambda x=x: m.token_logprobs(x, ids), lambda x=x: m.token_logprobs_grad(x, ids, v), lambda x=x: m.policy_loss_rows(x, ids, v, v)]
    for x in (long, empty((1 << 30) + 1)):
        calls += [lambda x=x: m.policy_loss(x, x, x), lambda x=x: m.preference_loss(x, ids)]
    for i, call in enumerate(calls):
        with pytest.raises(m.WsError, match="at most"):
            call()
            raise AssertionError(i)
