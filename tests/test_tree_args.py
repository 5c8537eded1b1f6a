"""CPU: what the calls over a cycle with a tree of drafts refuse, on the host and before anything is launched."""
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


def verify_of(m, **change):
    a = m.VerifyTree(n_seq=2, seq_off=AT, parent=AT, q=AT, q_words=144, q_off=AT, u_accept=AT, u_draw=AT, depth=3, n_accepted=AT, path=AT, chosen=AT, status=AT, logprob=AT)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def attention_of(m, cache=None, **change):
    layer = dict(k=AT, v=AT, dtype=1, pages=10, page_tokens=16, kv_heads=2, head_dim=64, k_page=2048, k_token=128, k_head=64, v_page=2048, v_token=128, v_head=64, table=AT, slots=3, slot_pages=4,
                 table_stride=4)
    layer.update(cache or {})
    a = m.TreeAttention(cache=m.CacheLayer(**layer), n_seq=2, rows=4, heads=8, q=AT, q_row=512, q_head=64, out=2 * AT, out_row=512, out_head=64, lse=AT, seq_off=AT, length=AT, mask=AT, scale=0.125)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def cache_of(m, **change):
    f = dict(k=AT, v=AT, dtype=1, layers=2, pages=10, page_tokens=16, kv_heads=2, head_dim=64, k_layer=20480, k_page=2048, k_token=128, k_head=64, v_layer=20480, v_page=2048, v_token=128, v_head=64, table=AT,
             slots=3, slot_pages=4, table_stride=4, held=AT, refs=AT, free=AT, n_free=AT)
    f.update(change)
    return m.Cache(**f)


@pytest.mark.parametrize("change", [dict(logits=None), dict(dtype=2), dict(vocab=0), dict(vocab=1 << 20), dict(rows=1 << 20), dict(row_stride=99), dict(allow=AT, allow_stride=3), dict(ids=None)])
def test_rows_that_verification_refuses(change):
    m = gc.pkg()
    assert m.lib().ws_verify_tree(None, C.byref(rows_of(m, **change)), C.byref(verify_of(m)), AT, 1 << 20) == m.E_INVALID
    assert m.lib().ws_verify_tree_workspace(C.byref(rows_of(m, **change)), C.byref(verify_of(m))) == 0


@pytest.mark.parametrize("change", [dict(n_seq=1 << 20), dict(seq_off=None), dict(q_off=None), dict(u_accept=None), dict(u_draw=None), dict(depth=0), dict(depth=65), dict(n_accepted=None), dict(path=None),
                                    dict(chosen=None), dict(status=None), dict(spins=65537), dict(hist="tokens alone")])
def test_verifications_that_are_refused(change):
    m = gc.pkg()
    if "hist" in change:
        change = dict(hist=m.History(tokens=AT, cap=10))
    assert m.lib().ws_verify_tree(None, C.byref(rows_of(m)), C.byref(verify_of(m, **change)), AT, 1 << 20) == m.E_INVALID


def test_verification_workspaces():
    m = gc.pkg()
    r, a = rows_of(m, vocab=151936, row_stride=151936), verify_of(m)
    need = m.lib().ws_verify_tree_workspace(C.byref(r), C.byref(a))
    assert need >= 2 * 2 * 32 + 4 * 16
    for at, size in ((None, need), (AT, need - 1), (AT + 4, need)):
        assert m.lib().ws_verify_tree(None, C.byref(r), C.byref(a), at, size) == m.E_WORKSPACE
    assert m.lib().ws_verify_tree(None, C.byref(r), None, AT, need) == m.lib().ws_verify_tree(None, None, C.byref(a), AT, need) == m.E_INVALID
    assert m.lib().ws_verify_tree(None, C.byref(r), C.byref(verify_of(m, n_seq=0)), None, 0) == 0  # nothing to do
    for dtype in (0, 1):  # the longest rows: as many parts as can meet
        for n_seq in (1, 300, 5000):
            r = rows_of(m, vocab=1048575, row_stride=1048575, dtype=dtype, rows=0)
            draw = m.lib().ws_verify_tree_workspace(C.byref(r), C.byref(verify_of(m, n_seq=n_seq)))
            parts = draw / (n_seq * 32)
            assert parts == int(parts) and 2 <= parts <= 64
            r.rows = 64 * n_seq
            parts = (m.lib().ws_verify_tree_workspace(C.byref(r), C.byref(verify_of(m, n_seq=n_seq))) - draw - r.rows * 16) / (r.rows * 32)
            assert parts == int(parts) and (parts == 0 or 2 <= parts <= 64)  # (where each row has one workgroup there are no words)


def test_stages_that_are_refused():
    m = gc.pkg()
    call = lambda **c: m.lib().ws_tree_stage(None, C.byref(m.TreeStage(**{**dict(n_seq=1, rows=4, seq_off=AT, mask=AT, position=AT, length=AT), **c})))  # noqa: E731
    assert m.lib().ws_tree_stage(None, None) == call(seq_off=None) == call(n_seq=1 << 20) == call(rows=1 << 20) == call(mask=AT + 4) == m.E_INVALID
    assert call(n_seq=0) == 0


@pytest.mark.parametrize("change", [dict(q=None), dict(out=None), dict(seq_off=None), dict(length=None), dict(heads=0), dict(heads=7), dict(heads=65536), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                    dict(scale=float("inf")), dict(q_row=511), dict(q_head=63), dict(q=AT + 8), dict(out_row=4), dict(out=AT + 2), dict(mask=AT + 4), dict(n_seq=1 << 20), dict(rows=1 << 20),
                                    dict(q_row=1 << 63), dict(q=AT, out=AT)])
def test_attention_that_is_refused(change):
    m = gc.pkg()
    assert m.lib().ws_tree_attention(None, C.byref(attention_of(m, **change)), AT, 1 << 40) == m.E_INVALID


@pytest.mark.parametrize("change", [dict(k=None), dict(v=AT + 8), dict(dtype=2), dict(pages=0), dict(page_tokens=0), dict(page_tokens=12), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264),
                                    dict(k_page=2047), dict(k_token=130), dict(v_head=1), dict(table=None), dict(slots=0), dict(slot_pages=0), dict(table_stride=3), dict(slot_pages=1 << 20),
                                    dict(slot_pages=1 << 19, table_stride=1 << 19, page_tokens=1 << 13)])
def test_caches_that_attention_refuses(change):
    m = gc.pkg()
    assert m.lib().ws_tree_attention(None, C.byref(attention_of(m, cache=change)), AT, 1 << 40) == m.E_INVALID


@pytest.mark.parametrize("change", [dict(k_page=1 << 35), dict(v_page=1 << 35), dict(k_token=1 << 35, k_page=1 << 36), dict(v_token=1 << 35)])
def test_attention_of_caches_whose_strides_are_not_supported(change):
    m = gc.pkg()
    assert m.lib().ws_tree_attention(None, C.byref(attention_of(m, cache=change)), AT, 1 << 40) == m.E_UNSUPPORTED


def test_attention_workspaces():
    m = gc.pkg()
    a = attention_of(m)
    need = m.lib().ws_tree_attention_workspace(C.byref(a))
    assert need > 0
    for at, size in ((None, need), (AT, need - 1), (AT + 8, need)):
        assert m.lib().ws_tree_attention(None, C.byref(a), at, size) == m.E_WORKSPACE
    assert m.lib().ws_tree_attention(None, None, AT, need) == m.E_INVALID
    assert m.lib().ws_tree_attention(None, C.byref(attention_of(m, n_seq=0)), None, 0) == m.lib().ws_tree_attention(None, C.byref(attention_of(m, rows=0)), None, 0) == 0


@pytest.mark.parametrize("change", [dict(k=None), dict(v=AT + 8), dict(dtype=-1), dict(layers=0), dict(pages=0), dict(page_tokens=3), dict(kv_heads=0), dict(head_dim=4), dict(k_layer=20481), dict(v_page=2047), dict(table=None),
                                    dict(slots=0), dict(slot_pages=0), dict(table_stride=3), dict(held=None), dict(refs=None), dict(free=None), dict(n_free=None), dict(k_layer=1 << 62)])
def test_caches_that_are_refused(change):
    m = gc.pkg()
    lib, c = m.lib(), C.byref(cache_of(m, **change))
    assert lib.ws_cache_reserve(None, c, AT, AT, 1, AT) == lib.ws_cache_fork(None, c, AT, AT, AT, 1, AT) == lib.ws_cache_release(None, c, AT, AT, 1, AT) == m.E_INVALID
    assert lib.ws_cache_keep(None, c, AT, 3, AT, AT, None, 1) == m.E_INVALID


def test_lists_that_are_refused():
    m = gc.pkg()
    lib, c = m.lib(), C.byref(cache_of(m))
    for n, a, b, s in ((1025, AT, AT, AT), (1, None, AT, AT), (1, AT, None, AT), (1, AT, AT, None)):
        assert lib.ws_cache_reserve(None, c, a, b, n, s) == m.E_INVALID
        assert lib.ws_cache_fork(None, c, a, b, AT, n, s) == m.E_INVALID
    assert lib.ws_cache_fork(None, c, AT, AT, None, 1, AT) == lib.ws_cache_release(None, c, None, AT, 1, None) == lib.ws_cache_release(None, c, AT, None, 1, None) == m.E_INVALID
    for path, depth, n_acc, length, n in ((None, 3, AT, AT, 1), (AT, 0, AT, AT, 1), (AT, 65, AT, AT, 1), (AT, 3, None, AT, 1), (AT, 3, AT, None, 1), (AT, 3, AT, AT, 1 << 20)):
        assert lib.ws_cache_keep(None, c, path, depth, n_acc, length, None, n) == m.E_INVALID
    assert lib.ws_cache_reserve(None, c, None, None, 0, None) == lib.ws_cache_fork(None, c, None, None, None, 0, None) == lib.ws_cache_release(None, c, None, None, 0, None) == 0
    assert lib.ws_cache_keep(None, c, None, 3, None, None, None, 0) == 0


def test_python_calls_refuse_host_tensors_before_they_reach_the_library():
    m = gc.pkg()
    if torch.cuda.is_available():
        pytest.skip("a machine without a GPU is meant")
    x, ids, off, u = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), torch.zeros(3, dtype=torch.float64)
    q, k, table = torch.zeros(3, 4, 64), torch.zeros(2, 16, 2, 64), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: m.tree_stage(off, 3), lambda: m.verify_tree(x, ids, off, u, u[:1]), lambda: m.tree_attention(q, k, k, table, ids[:1], off), lambda: m.tree_attention(q[0], k, k, table, ids[:1], off),
                 lambda: m.PagedCache(k[None], k[None], table, ids[:1], ids[:2], ids[:2], ids[:1])):
        with pytest.raises(m.WsError):
            call()


def test_what_a_row_sees_is_staged_as_it_is_written_out():
    """The plain implementation of the stage, by hand."""
    import tree_ref as tr
    mask, position = tr.stage([[-1, 0, 0, 1, 9, 4, 3]], [10])
    assert mask.tolist() == [1, 3, 5, 11, 16, 32, 75] and position.tolist() == [10, 11, 11, 12, 10, 10, 13]


def test_pages_by_hand():
    """The plain allocator of the tests: taken from the end, shared, given back the first uppermost."""
    import tree_ref as tr
    p = tr.Pages(4, 3, 6, 4)
    assert p.reserve([0, 1, 0, 2], [5, 13, 1, 4]) == [0, 1, 2, 0] and p.table[0] == [0, 1, -1] and p.table[2] == [2, -1, -1] and p.free == [5, 4, 3]
    assert p.fork([0, 0], [1, 3], [6, 8]) == [0, 0] and p.table[1] == [0, 3, -1] and p.table[3] == [0, 1, -1] and p.refs[:4] == [3, 2, 1, 1] and p.copies == [(1, 3, 2)]
    assert p.release([0, 1], [0, 0]) == [0, 0] and p.free == [5, 4, 3] and p.refs[:4] == [1, 1, 1, 0]
    assert p.release([3], [0]) == [0] and p.free == [5, 4, 3, 1, 0]


def test_histories_that_are_refused(monkeypatch):
    """Without slots a sequence's slot is its number: a history of fewer would be read, and written, behind its ends. One on another device would be too."""
    m = gc.pkg()

    class Reached(Exception):
        pass

    def library():
        raise Reached
    monkeypatch.setattr(m, "_device_of", lambda name, t: -1)  # (host tensors stand for device tensors)
    monkeypatch.setattr(m, "lib", library)
    n = 5
    off, ids, u = torch.arange(n + 1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32), torch.zeros(n, dtype=torch.float64)
    elsewhere = m.DeviceHistory(n, 8, "cpu")

    class Other:
        device = "cuda:1"
        get_device = staticmethod(lambda: 1)
    elsewhere.n_gen = Other
    for call in (lambda **c: m.tree_stage(off, n, **c), lambda **c: m.verify_tree(torch.zeros(n, 10), ids, off, u, u, **c)):
        for slots in (0, 1, n - 1):
            with pytest.raises(m.WsError, match="slot: missing"):
                call(hist=m.DeviceHistory(slots, 8, "cpu"))
        with pytest.raises(m.WsError, match="hist: on"):
            call(hist=elsewhere)
        with pytest.raises(m.WsError, match="slot: contiguous"):
            call(hist=m.DeviceHistory(n, 8, "cpu"), slot=ids[:4])
        for given in ({}, {"hist": m.DeviceHistory(n, 8, "cpu")}, {"hist": m.DeviceHistory(1, 8, "cpu"), "slot": ids}):
            with pytest.raises(Reached):
                call(**given)


def test_more_nodes_than_a_tree_has_are_refused(monkeypatch):
    """Who says that a sequence has more than 64 nodes would get rows that nothing has been written to."""
    m = gc.pkg()
    for nodes in (65, 1 << 20, (1 << 32) - 1):
        assert m.lib().ws_tree_attention(None, C.byref(attention_of(m, max_nodes=nodes)), AT, 1 << 40) == m.E_INVALID
        assert m.lib().ws_tree_attention_workspace(C.byref(attention_of(m, max_nodes=nodes))) == 0
    assert m.lib().ws_tree_attention_workspace(C.byref(attention_of(m, max_nodes=64))) > 0
    monkeypatch.setattr(m, "_device_of", lambda name, t: -1)  # (host tensors stand for device tensors)
    q, k, ids = torch.zeros(3, 4, 64), torch.zeros(2, 16, 2, 64), torch.zeros(3, dtype=torch.int32)
    for nodes in (-1, 65, 1 << 33):
        with pytest.raises(m.WsError, match="max_nodes"):
            m.tree_attention(q, k, k, ids[:2].view(1, 2), ids[:1], torch.tensor([0, 3], dtype=torch.int32), max_nodes=nodes)


BIG = 1 << 30


@pytest.mark.parametrize("change", [dict(out=BIG), dict(out=BIG + 16), dict(out=BIG + 3 * 1024), dict(out=BIG - 3 * 1024), dict(out=BIG + 512 * 2 - 16), dict(out=2 * BIG), dict(out=2 * BIG + 40960 - 16), dict(out=2 * BIG - 3 * 1024 - 16),
                                    dict(out=3 * BIG + 4096), dict(out_row=0), dict(out_head=0), dict(out_row=256), dict(out_row=504), dict(out_head=56), dict(out=BIG + 512, q_row=1024, out_row=1024, out_head=128),
                                    dict(out=BIG + 1024, q_row=1024, out_row=1032), dict(out=BIG + 128, q_row=1024, q_head=128, out_row=1024, out_head=136)])
def test_attention_whose_out_lies_over_what_it_reads(change):
    """q at BIG, K at 2 BIG, V at 3 BIG: out over one of them, or over itself, wherever they begin."""
    m = gc.pkg()
    a = attention_of(m, cache=dict(k=2 * BIG, v=3 * BIG), q=BIG, **{**dict(out=4 * BIG), **change})
    assert m.lib().ws_tree_attention(None, C.byref(a), AT, 1 << 40) == m.E_INVALID


@pytest.mark.parametrize("change", [dict(out=4 * BIG), dict(out=BIG + 4 * 1024), dict(out=BIG - 4 * 1024), dict(out=BIG + 1024, q_row=1024, out_row=1024), dict(out=BIG - 1024, q_row=1024, out_row=1024),
                                    dict(out=BIG + 128, q_row=1024, q_head=128, out_row=1024, out_head=128), dict(out=BIG + 512, q_row=64, q_head=512, out_row=64, out_head=512), dict(out_row=64, out_head=256),
                                    dict(rows=1, out_row=0), dict(q_row=0, q_head=0), dict(out=BIG + 1024, q_row=2048, out_row=1024, rows=1, n_seq=1)])
def test_outs_that_lie_apart(change):
    """out between the rows or the heads of q, before it, behind it: what is missing is the workspace."""
    m = gc.pkg()
    a = attention_of(m, cache=dict(k=2 * BIG, v=3 * BIG), q=BIG, **{**dict(out=4 * BIG), **change})
    assert m.lib().ws_tree_attention(None, C.byref(a), None, 0) == m.E_WORKSPACE


@pytest.mark.parametrize("change", [dict(page_tokens=1 << 20, kv_heads=128, head_dim=128), dict(kv_heads=65535, head_dim=(1 << 32) - 8, page_tokens=1 << 10), dict(head_dim=1 << 31, page_tokens=4),
                                    dict(page_tokens=1 << 20, slot_pages=1, table_stride=1, kv_heads=65528, head_dim=256)])
def test_pages_of_more_pieces_than_32_bits_count(change):
    m = gc.pkg()
    lib, c = m.lib(), C.byref(cache_of(m, **{**dict(k_token=0, v_token=0, k_head=0, v_head=0), **change}))
    assert lib.ws_cache_fork(None, c, AT, AT, AT, 1, AT) == lib.ws_cache_reserve(None, c, AT, AT, 1, AT) == lib.ws_cache_keep(None, c, AT, 3, AT, AT, None, 1) == m.E_INVALID
