"""CPU: what the entry points over log-probabilities refuse, on the host and before anything is launched, and the workspaces they ask for."""
import ctypes as C

import pytest
import torch

import gpu_cases as gc

AT = 1 << 20  # an address that nothing reads


def rows_of(m, **change):
    r = m.LossRows(logits=AT, dtype=m.DTYPE_F32, rows=4, vocab=100, row_stride=100, ids=AT, inv_t=AT)
    for k, v in change.items():
        setattr(r, k, v)
    return r


def policy_of(m, **change):
    p = m.Policy(old_logprob=AT, ref_logprob=AT, advantage=AT, weight=AT, clip_low=0.2, clip_high=0.2, dual_clip=0.0, kl_coef=0.1, entropy_coef=0.0)
    for k, v in change.items():
        setattr(p, k, v)
    return p


BAD_ROWS = [dict(logits=None), dict(logits=AT + 2), dict(dtype=2), dict(dtype=-1), dict(vocab=0), dict(vocab=1 << 20), dict(rows=1 << 20), dict(row_stride=99),
            dict(allow=AT, allow_stride=3), dict(allow=AT + 2, allow_stride=4), dict(dtype=1, logits=AT + 1)]


@pytest.mark.parametrize("change", BAD_ROWS)
def test_rows_that_are_refused(change):
    m = gc.pkg()
    lib, r, p = m.lib(), rows_of(m, **change), policy_of(m)
    far = AT << 20
    assert lib.ws_token_logprobs(None, C.byref(r), AT, AT, None, None, 0) == m.E_INVALID
    assert lib.ws_token_logprobs_grad(None, C.byref(r), AT, AT, None, None, far, 100) == m.E_INVALID
    assert lib.ws_policy_loss_rows(None, C.byref(r), C.byref(p), AT, AT, None, far, 100, AT, 1 << 20) == m.E_INVALID
    assert lib.ws_token_logprobs_workspace(C.byref(r)) == 0 and lib.ws_policy_loss_rows_workspace(C.byref(r)) == 0


def test_outputs_and_gradients_that_are_refused():
    m = gc.pkg()
    lib, r, far = m.lib(), rows_of(m), AT << 20
    assert lib.ws_token_logprobs(None, None, AT, AT, None, None, 0) == m.E_INVALID
    assert lib.ws_token_logprobs(None, C.byref(r), None, AT, None, None, 0) == m.E_INVALID
    assert lib.ws_token_logprobs(None, C.byref(r), AT, None, None, None, 0) == m.E_INVALID
    grad = lambda d, stride, stats=AT, entropy=None, d_entropy=None: lib.ws_token_logprobs_grad(None, C.byref(r), stats, AT, entropy, d_entropy, d, stride)  # noqa: E731
    assert grad(None, 100) == grad(far + 1, 100) == grad(far, 99) == grad(far, 100, stats=None) == grad(far, 100, d_entropy=AT) == m.E_INVALID
    for d, stride in ((AT, 101), (AT + 4, 100), (AT - 4, 100), (AT + 4 * 399, 100), (AT - 4 * 399, 100)):  # laid over the logits, but not on them
        assert grad(d, stride) == m.E_INVALID


BAD_POLICIES = [dict(old_logprob=None), dict(advantage=None), dict(clip_low=-0.1), dict(clip_low=1.1), dict(clip_low=float("nan")), dict(clip_high=-1e-9), dict(clip_high=float("nan")),
                dict(dual_clip=1.0), dict(spins=65537), dict(dual_clip=-2.0), dict(dual_clip=float("nan")), dict(kl_coef=float("nan")), dict(entropy_coef=float("nan")), dict(ref_logprob=None),
                dict(entropy_coef=0.01)]


@pytest.mark.parametrize("change", BAD_POLICIES)
def test_policies_that_are_refused(change):
    m = gc.pkg()
    lib, r, p, far = m.lib(), rows_of(m), policy_of(m, **change), AT << 20
    assert lib.ws_policy_loss_rows(None, C.byref(r), C.byref(p), AT, AT, None, far, 100, AT, 1 << 20) == m.E_INVALID
    assert lib.ws_policy_loss(None, 4, C.byref(p), AT, None, AT, AT, None, AT, 1 << 20) == m.E_INVALID


def test_policy_outputs_and_workspaces_that_are_refused():
    m = gc.pkg()
    lib, r, p, far = m.lib(), rows_of(m), policy_of(m), AT << 20
    ref = C.byref(r), C.byref(p)
    need = lib.ws_policy_loss_rows_workspace(ref[0])
    assert need >= 4 * 5 * 8
    assert lib.ws_policy_loss_rows(None, *ref, None, AT, None, far, 100, AT, need) == m.E_INVALID
    assert lib.ws_policy_loss_rows(None, *ref, AT, None, None, far, 100, AT, need) == m.E_INVALID
    assert lib.ws_policy_loss_rows(None, *ref, AT, AT, None, far, 100, AT, need - 1) == m.E_WORKSPACE
    assert lib.ws_policy_loss_rows(None, *ref, AT, AT, None, far, 100, None, need) == m.E_WORKSPACE
    assert lib.ws_policy_loss_rows(None, *ref, AT, AT, None, far, 100, AT + 4, need) == m.E_WORKSPACE
    r.ids = None
    assert lib.ws_policy_loss_rows(None, *ref, AT, AT, None, far, 100, AT, need) == m.E_INVALID
    many = 100000
    need = lib.ws_policy_loss_workspace(many)
    assert lib.ws_policy_loss_workspace(1) == lib.ws_policy_loss_workspace(0) == 0 and need > 0
    assert lib.ws_policy_loss(None, many, C.byref(p), AT, None, AT, AT, None, AT, need - 1) == m.E_WORKSPACE
    assert lib.ws_policy_loss(None, many, C.byref(p), None, None, AT, AT, None, AT, need) == m.E_INVALID
    assert lib.ws_policy_loss(None, many, C.byref(p), AT, None, None, AT, None, AT, need) == m.E_INVALID
    assert lib.ws_policy_loss(None, many, C.byref(p), AT, None, AT, None, None, AT, need) == m.E_INVALID
    assert lib.ws_policy_loss(None, 1 << 31, C.byref(p), AT, None, AT, AT, None, AT, 1 << 20) == m.E_INVALID


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("rows,words", [(1, 8), (2000, 8), (4096, 8), (5000, 6)])
def test_the_longest_rows_have_no_more_parts_than_can_meet(dtype, rows, words):
    """A wave looks at a row's parts, one a lane: 64 at most, each with six words and, where the rows' sums meet in the same launch, two for its mark."""
    m = gc.pkg()
    r = rows_of(m, dtype=dtype, rows=rows, vocab=1048575, row_stride=1048575)
    slots, second = (0 if rows == 1 else rows + (64 if rows > 64 else 0), 0) if words == 8 else (rows // 1024 + 1, rows * 5 * 8)
    sums = slots * 5 * 16
    parts = (m.lib().ws_policy_loss_rows_workspace(C.byref(r)) - sums - second) / (rows * words * 8)
    assert parts == int(parts) and 2 <= parts <= 64


@pytest.mark.parametrize("change", [dict(pairs=0), dict(pairs=1 << 31), dict(rows=1 << 31), dict(seq_off=None), dict(logprob=None), dict(loss=None), dict(pair_loss=None),
                                    dict(reward=None), dict(d_logprob=None), dict(beta=float("nan")), dict(label_smoothing=-0.1), dict(label_smoothing=1.5),
                                    dict(label_smoothing=float("nan"))])
def test_preferences_that_are_refused(change):
    m = gc.pkg()
    p = m.Preference(rows=10, pairs=2, seq_off=AT, logprob=AT, beta=0.1, loss=AT, pair_loss=AT, reward=AT, d_logprob=AT)
    need = m.lib().ws_preference_loss_workspace(2)
    assert need > 0 and m.lib().ws_preference_loss_workspace(1) == 0
    assert m.lib().ws_preference_loss(None, C.byref(p), AT, need - 1) == m.lib().ws_preference_loss(None, C.byref(p), None, need) == m.E_WORKSPACE
    for k, v in change.items():
        setattr(p, k, v)
    assert m.lib().ws_preference_loss(None, C.byref(p), AT, 1 << 20) == m.E_INVALID


def test_python_calls_refuse_host_tensors_before_they_reach_the_library():
    m = gc.pkg()
    x, ids, v = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    if torch.cuda.is_available():
        pytest.skip("a machine without a GPU is meant")
    for call in (lambda: m.token_logprobs(x, ids), lambda: m.token_logprobs_grad(x, ids, v), lambda: m.policy_loss_rows(x, ids, v, v), lambda: m.policy_loss(v, v, v),
                 lambda: m.preference_loss(v, ids), lambda: m.token_logprobs(x.half(), ids), lambda: m.token_logprobs(x[:, ::2], ids), lambda: m.token_logprobs(x[0], ids)):
        with pytest.raises(m.WsError):
            call()
