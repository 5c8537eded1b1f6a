"""GPU: a cycle with a tree of drafts (ws_tree_stage, ws_verify_tree, ws_tree_attention) against plain implementations in 64 bits (tree_ref.py, where the tolerances are derived)."""
import math

import pytest
import torch

import gpu_cases as gc
import loss_ref as lr
import tree_ref as tr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def near(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    bad = ~((torch.isnan(got) & torch.isnan(want)) | (got == want) | ((got - want).abs() <= tol))
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError((what, i, float(got[i]), float(want[i]), float(tol[i]), int(bad.sum()), bad.numel()))


# ---- what a cycle begins with


@pytest.mark.parametrize("counts,kids", [([1], 1), ([64, 1, 0, 33], 2), ([64], 1), ([7] * 70, 4), ([64, 63, 2], 64)])
def test_stage(counts, kids):
    m = gc.pkg()
    g = torch.Generator().manual_seed(sum(counts) + kids)
    parents = tr.random_trees(counts, kids, g)
    if len(counts) == 4:  # nodes that are never reached, and what hangs below them
        parents[0][5], parents[3][2], parents[3][9] = -7, 2, 31
    n_seq, rows = len(counts), sum(counts)
    hist = m.DeviceHistory(n_seq + 3, 16, DEV)
    slot = torch.randperm(n_seq + 3, generator=g)[:n_seq].to(torch.int32)
    lens = torch.randint(0, 1 << 20, (n_seq + 3,), generator=g, dtype=torch.int32)
    hist.len.copy_(lens)
    flat = torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=DEV)
    mask, position, length = m.tree_stage(tr.offsets(counts).to(DEV), rows, parent=flat, hist=hist, slot=slot.to(DEV))
    want = tr.stage(parents, [int(lens[s]) for s in slot])
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(position.cpu(), want[1]) and torch.equal(length.cpu(), lens[slot.long()])
    mask, position, length = m.tree_stage(tr.offsets(counts).to(DEV), rows)  # chains over empty texts
    want = tr.stage([[i - 1 for i in range(n)] for n in counts], [0] * n_seq)
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(position.cpu(), want[1]) and not length.any()


# ---- verification


def verify_case(counts, kids, V, dtype, seed, guessed=False, masked=False, stride=0, sharp=1.0, chain=False, u0=None):
    """Logits with a few tokens that stand out, trees drafted from distributions near them, uniforms away from the borders, and the walks."""
    g = torch.Generator().manual_seed(seed)
    parents = [[i - 1 for i in range(n)] for n in counts] if chain else tr.random_trees(counts, kids, g)
    rows = sum(counts)
    x = torch.randn((rows, V), generator=g) * 2.0
    x.scatter_add_(1, torch.randint(V, (rows, 4), generator=g), sharp * (math.log(V) + 4.0 * torch.rand((rows, 4), generator=g)))
    x = x.to(dtype)
    inv_t = 1.0 / (0.7 + 0.5 * torch.rand(rows, generator=g))
    allow = None
    if masked:
        allow = torch.rand((rows, V), generator=g) < 0.3
        allow[torch.arange(rows), x.float().argmax(1)] = True
    ids, entries, first = torch.zeros(rows, dtype=torch.int32), [None] * rows, 0
    for tree in parents:
        for i in range(len(tree)):
            kidsof = [c for c, p in enumerate(tree) if p == i and c > i]
            z = x[first + i].double() * inv_t[first + i] + 0.5 * torch.randn(V, generator=g, dtype=torch.float64)
            if allow is not None and i % 3 != 2:  # (a draft head that knows the mask, and one that does not)
                z = torch.where(allow[first + i], z, torch.tensor(-1e9, dtype=torch.float64))
            n = min(V, int(torch.randint(1, 33, (1,), generator=g)))
            top = z.topk(n)
            q = torch.softmax(top.values, 0).float()
            order = torch.multinomial(q.double() + 1e-12, min(n, max(1, len(kidsof))), generator=g)
            for c, kid in enumerate(kidsof):
                ids[first + kid] = int(top.indices[order[c % len(order)]])
            if not guessed and not (guessed is None and i % 2):
                entries[first + i] = list(zip(top.indices.tolist(), q.tolist()))
        first += len(tree)
    u_accept = torch.rand(rows, generator=g, dtype=torch.float64)
    u_draw = torch.rand(len(counts), generator=g, dtype=torch.float64)
    if u0 is not None:
        u_draw[:] = u0
    walks, first = [], 0
    for s, tree in enumerate(parents):
        at = slice(first, first + len(tree))
        make = lambda ua, ud: tr.Verify(x[at], ids[at], tree, ua, ud, inv_t[at], None if allow is None else allow[at], entries[at])  # noqa: E731
        ua, ud = [float(v) for v in u_accept[at]], float(u_draw[s])
        if u0 is None:
            ua, ud, w = tr.uniforms_apart(make, ua, ud)
        else:
            w = make(ua, ud)
        u_accept[at], u_draw[s] = torch.tensor(ua, dtype=torch.float64), ud
        walks.append(w)
        first += len(tree)
    dx = torch.full((rows, V + stride), math.nan, dtype=dtype, device=DEV)[:, :V]
    dx.copy_(x)
    q = q_off = None
    if any(e is not None for e in entries):
        q, q_off = torch.zeros((rows, tr.Q_WORDS), dtype=torch.int32), torch.full((rows,), -1, dtype=torch.int32)
        for r, e in enumerate(entries):
            if e is not None:
                q_off[r], q[r, 0] = r * tr.Q_WORDS, len(e)
                q[r, 1:1 + len(e)] = torch.tensor([i for i, _ in e], dtype=torch.int32)
                q[r, 33:33 + len(e)] = torch.tensor([v for _, v in e], dtype=F32).view(torch.int32)
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    call = dict(logits=dx, ids=to(ids), seq_off=to(tr.offsets(counts)), u_accept=to(u_accept), u_draw=to(u_draw), parent=None if chain else to(torch.tensor([p for t in parents for p in t], dtype=torch.int32)),
                q=to(q), q_off=to(q_off), inv_t=to(inv_t), allow=None if allow is None else lr.pack_allow(allow).to(DEV))
    return call, walks, ids, parents


def check_walks(got, walks, depth, V):
    n_accepted, path, chosen, status, logprob = (t.cpu() for t in got)
    for s, w in enumerate(walks):
        # 1e-6: two comparisons' distance; 1e-9 of the sum: the draw's. Nearer ones may fall either way and do not occur (uniforms_apart)
        assert w.near > 1e-6 and w.draw_near > 1e-10, (s, w.near, w.draw_near)
        have = path[s].tolist()
        assert (int(n_accepted[s]), have[:len(w.path)], int(chosen[s]), int(status[s])) == (len(w.path), w.path[:depth], w.chosen, w.status), (s, w.path, have, int(chosen[s]), w.chosen)
        assert all(v == -1 for v in have[len(w.path):])
        lp = w.logprob + [0.0] * (depth + 1 - len(w.logprob))
        # a sum of V powers in 32 bits, each off by some 2^-22: ln S by as much; the float's own half step
        near(logprob[s], torch.tensor(lp[:depth + 1], dtype=torch.float64), 2.0 ** -21 + 2.0 ** -23 * max(abs(v) for v in lp if v > -math.inf), "logprob")


SHAPES = [([1], 1, 1, F32), ([2], 1, 2, F32), ([3, 1, 2], 1, 7, BF16), ([5], 4, 33, BF16), ([9, 4], 2, 1000, F32), ([16] * 5, 3, 4099, BF16), ([64, 1, 30], 2, 777, F32), ([25] * 40, 2, 8200, F32),
          ([6], 1, 151936, BF16), ([9, 12, 3], 3, 50257, F32), ([4] * 3, 2, 262144, BF16), ([2], 1, 1048575, F32), ([3], 1, 1048575, BF16), ([3] * 300, 2, 12345, BF16), ([2] * 600, 1, 513, F32)]


@pytest.mark.parametrize("counts,kids,V,dtype", SHAPES)
@pytest.mark.parametrize("kind", ["entries", "guesses", "both", "masked"])
def test_verify(counts, kids, V, dtype, kind):
    m = gc.pkg()
    if kind != "entries" and sum(counts) * V > 3_000_000:
        counts = counts[:2]
    call, walks, ids, _ = verify_case(counts, kids, V, dtype, sum(counts) + V, guessed={"guesses": True, "both": None}.get(kind, False), masked=kind == "masked", stride=3 if V % 2 else 0)
    depth = max(1, max(counts) - 1)
    got = m.verify_tree(depth=depth, **call)
    check_walks(got, walks, depth, V)
    again = m.verify_tree(depth=depth, spins=1, **call)  # workgroups that hardly wait: the same bits
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    assert sum(len(w.path) for w in walks) > 0 or sum(counts) < 100


@pytest.mark.parametrize("V", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_of_the_smallest_vocabularies(V, dtype):
    m = gc.pkg()
    for seed, masked in ((1, False), (2, True)):
        call, walks, ids, _ = verify_case([1, 4, 9, 2], 2, V, dtype, 10 * V + seed, guessed=None, masked=masked, stride=1)
        check_walks(m.verify_tree(depth=8, **call), walks, 8, V)


def test_verify_chains_and_few_columns():
    """No parents: chains. Fewer columns than accepted nodes: the first of them."""
    m = gc.pkg()
    call, walks, ids, _ = verify_case([8, 12, 20], 1, 3000, F32, 5, chain=True, sharp=1.6)
    assert max(len(w.path) for w in walks) > 3
    check_walks(m.verify_tree(depth=63, **call), walks, 63, 3000)
    check_walks(m.verify_tree(depth=64, **call), walks, 64, 3000)
    check_walks(m.verify_tree(depth=2, **call), walks, 2, 3000)


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -53, 1.0, 2.0, -1.0, math.nan])
def test_verify_draws_at_the_ends(u):
    """0 and below: the first token with any probability; 1 and beyond (or what is no number): the last."""
    m = gc.pkg()
    for V, dtype in ((9, F32), (5000, BF16), (40000, F32)):
        call, walks, _, _ = verify_case([1, 1], 1, V, dtype, 3 * V, masked=True, u0=0.5)
        call["u_draw"][:] = u
        allowed = [((call["allow"][s, torch.arange(V, device=DEV) // 32] >> (torch.arange(V, device=DEV) % 32).int()) & 1).nonzero()[:, 0] for s in range(2)]
        chosen = m.verify_tree(depth=1, **call)[2].cpu()
        if 1.0 - 2.0 ** -53 <= u < 1.0:
            assert all(int(chosen[s]) in allowed[s].tolist()[-20:] for s in range(2))  # (the last powers may not add up to as much)
        else:
            assert [int(c) for c in chosen] == [int(a[0] if u <= 0.0 else a[-1]) for a in allowed]


def test_verify_the_same_token_twice_and_ids_outside():
    """Siblings with one token, entries with an id twice, with ids outside the vocabulary, with no ids, with more than there can be; parents that are none."""
    m = gc.pkg()
    V = 300
    g = torch.Generator().manual_seed(1)
    x = torch.randn((4 * 6, V), generator=g)
    parent, ids = [-1, 0, 0, 0, 0, 9], [0, 5, 5, 7, 400, 3]
    q = torch.zeros((3, tr.Q_WORDS), dtype=torch.int32)
    lists = [[(5, 0.25), (5, 0.25), (7, 0.3), (-4, 0.1), (400, 0.1)], [], [(i, 1 / 32) for i in range(32)]]
    for r, e in enumerate(lists):
        q[r, 0] = len(e) if r < 2 else 1000
        for i, (id_, p) in enumerate(e):
            q[r, 1 + i], q[r, 33 + i] = id_, torch.tensor([p], dtype=F32).view(torch.int32)[0]
    entries = [[(i, float(torch.tensor(p, dtype=F32))) for i, p in e] for e in lists]
    q_off, every, walks, ua, ud = [], [], [], [], []
    for s in range(4):
        e = entries[s] if s < 3 else None
        q_off += [s * tr.Q_WORDS if s < 3 else -1] * 6
        rows = x[6 * s:6 * s + 6]
        make = lambda a, d: tr.Verify(rows, ids, parent, a, d, [1.0] * 6, None, [e] * 6)  # noqa: E731
        a, d, w = tr.uniforms_apart(make, [0.9, 0.9, 0.8, 0.95, 0.9, 0.5], 0.4 + 0.1 * s)
        ua, ud = ua + a, ud + [d]
        walks.append(w)
    to = lambda v, t: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    got = m.verify_tree(x.to(DEV), to(ids * 4, torch.int32), tr.offsets([6] * 4).to(DEV), to(ua, torch.float64), to(ud, torch.float64), parent=to(parent * 4, torch.int32), q=q.to(DEV),
                        q_off=to(q_off, torch.int32), depth=3)
    check_walks(got, walks, 3, V)


def test_verify_rows_without_anything_to_draw():
    """Masked rows, NaN, infinities, temperatures that are none, entries outside q, sequences without nodes: the host's, what was accepted before is reported, the history stays."""
    m = gc.pkg()
    V = 2000
    call, walks, ids, _ = verify_case([3] * 10, 1, V, F32, 11, guessed=True, chain=True, sharp=3.0)
    x, inv_t = call["logits"].clone(), call["inv_t"].clone()
    call["u_accept"][:] = 0.0
    words = (V + 31) // 32
    allow = torch.full((30, words), -1, dtype=torch.int32, device=DEV)
    x[0] = -math.inf
    x[3 * 1 + 1, 700] = math.nan
    x[3 * 2, 5] = math.inf
    inv_t[3 * 3], inv_t[3 * 4 + 1], inv_t[3 * 5] = 0.0, math.inf, -1.0
    allow[3 * 6 + 2] = 0
    inv_t[3 * 7] = math.nan
    hist = m.DeviceHistory(10, 16, DEV)
    hist.len[:] = torch.arange(10, device=DEV, dtype=torch.int32)
    hist.tokens[:] = 77
    call.update(logits=x, inv_t=inv_t, allow=allow)
    slot = torch.arange(10, device=DEV, dtype=torch.int32)
    q = torch.zeros(tr.Q_WORDS, dtype=torch.int32, device=DEV)
    q[0] = 1
    q_off = torch.full((30,), -1, dtype=torch.int32, device=DEV)
    q_off[3 * 8 + 1] = 1  # (its last word lies behind q)
    n_accepted, path, chosen, status, logprob = (t.cpu() for t in m.verify_tree(depth=2, hist=hist, slot=slot, **{**call, "q": q, "q_off": q_off}))
    assert status.tolist() == [1] * 9 + [0]
    assert n_accepted.tolist() == [0, 1, 0, 0, 1, 0, 2, 0, 1, 2] and chosen.tolist()[:9] == [-1] * 9 and 0 <= int(chosen[9]) < V
    assert path.tolist()[6] == [1, 2] and path.tolist()[8] == [1, -1]
    assert hist.len.cpu().tolist() == list(range(9)) + [12] and hist.n_gen.cpu().tolist() == [0] * 9 + [3]
    assert (hist.tokens[:9] == 77).all() and hist.tokens[9, 10:13].cpu().tolist() == [int(call["ids"][28]), int(call["ids"][29]), int(chosen[9])]
    off = torch.tensor([0, 0, 3, 3], dtype=torch.int32, device=DEV)
    got = m.verify_tree(call["logits"][27:30], call["ids"][27:30], off, call["u_accept"][27:30], call["u_draw"][:3], depth=2)
    assert got[3].cpu().tolist() == [1, 0, 1] and got[0].cpu().tolist() == [0, 2, 0] and got[2].cpu().tolist()[::2] == [-1, -1] and not got[4][0].any() and (got[1][2] == -1).all()


def test_verify_history_without_room():
    m = gc.pkg()
    call, _, _, _ = verify_case([3] * 4, 1, 500, F32, 2, guessed=True, chain=True)
    call["u_accept"][:] = 0.0  # (two accepted each: next, two and the chosen one have to fit)
    hist = m.DeviceHistory(4, 10, DEV)
    hist.len[:] = torch.tensor([6, 7, 5, 9], device=DEV, dtype=torch.int32)
    n_accepted, path, chosen, status, _ = (t.cpu() for t in m.verify_tree(depth=3, hist=hist, slot=None, **call))
    assert status.tolist() == [0, 5, 0, 5] and n_accepted.tolist() == [2, 0, 2, 0] and chosen.tolist()[1::2] == [-1, -1] and (path[1] == -1).all()
    assert hist.len.cpu().tolist() == [9, 7, 8, 9]


def test_verify_captured_and_replayed():
    """A captured call: new inputs, new streams, the eager call in between; every replay is the eager call's answer."""
    m = gc.pkg()
    cases = [verify_case([7, 16, 3], 2, 60000, BF16, 100 + i, guessed=None)[0] for i in range(3)]
    call = {k: None if v is None else v.clone() for k, v in cases[0].items()}
    m.lib().ws_probe()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.verify_tree(depth=15, **call)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.verify_tree(depth=15, **call)
    for c in cases + cases[::-1]:
        for k, v in c.items():
            if v is not None:
                call[k].copy_(v)
        want = m.verify_tree(depth=15, **c)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("begin", [0, 64, 4096])
def test_verify_replayed_where_others_use_the_workspace(begin):
    """A captured call's workspace belongs to others between its replays: some of it has the same in it each time, the rest what the last replay left. Other logits, other entries (some of them
    none) each time."""
    m = gc.pkg()
    counts = [7, 16, 3]
    cases = [verify_case(counts, 2, 60000, BF16, 200 + i, guessed=False)[0] for i in range(3)]
    cases[1]["q_off"][cases[1]["q_off"] >= 0] = cases[1]["q"].numel()  # (entries that lie outside: the sequences are the host's)
    call = {k: None if v is None else v.clone() for k, v in cases[0].items()}
    r = m._loss_rows(call["logits"], call["ids"], call["inv_t"], call["allow"])[0]
    small, logprob = torch.empty(3 * 3 + 3 * 15, dtype=torch.int32, device=DEV), torch.empty(3, 16, device=DEV)
    at = small.data_ptr()
    a = m.VerifyTree(3, *(0 if call.get(k) is None else call[k].data_ptr() for k in ("seq_off", "parent", "q")), call["q"].numel(),
                     *(call[k].data_ptr() for k in ("q_off", "u_accept", "u_draw")), 15, at, at + 36, at + 12, at + 24, logprob.data_ptr())
    need = m.lib().ws_verify_tree_workspace(r, a)
    work = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert need > 4160
    run = lambda: m.check(m.lib().ws_verify_tree(torch.cuda.current_stream().cuda_stream, r, a, work.data_ptr(), need), "ws_verify_tree")  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in (0, 1, 2, 1, 0, 2, 0, 0, 1, 1, 2):
        for k, v in cases[i].items():
            if v is not None:
                call[k].copy_(v)
        want = m.verify_tree(depth=15, **cases[i])
        for _ in range(2):
            work[begin:begin + 64] = 0
            small.fill_(-9)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(small[0:3], want[0]) and torch.equal(small[9:].view(3, 15), want[1]) and torch.equal(small[3:6], want[2]) and torch.equal(small[6:9], want[3])
            assert torch.equal(logprob, want[4])
            assert int(want[3].sum()) == (0 if i != 1 else 3)


@pytest.mark.parametrize("counts,V,dtype", [([7, 16, 3], 60000, BF16), ([1, 5], 151936, F32), ([2] * 3, 1048575, F32)])
def test_verify_leaves_no_words_for_its_replays(counts, V, dtype):
    """The replays of a captured call have one tag: no word of a launch, of a row's maximum or of its sum, may be whole where the next replay looks for it. The rows' words and the decisions are
    taken apart by the launch that left them, the draw's by the next one (here one whose sequences are empty, so that its draw leaves a maximum's word alone)."""
    m = gc.pkg()
    n_seq, rows = len(counts), sum(counts)
    call = verify_case(counts, 2, V, dtype, 300 + rows, guessed=True)[0]
    r = m._loss_rows(call["logits"], call["ids"], call["inv_t"], None)[0]
    small = torch.zeros(3 * n_seq + 15 * n_seq, dtype=torch.int32, device=DEV)
    at = small.data_ptr()
    a = m.VerifyTree(n_seq, call["seq_off"].data_ptr(), call["parent"].data_ptr(), None, 0, None, call["u_accept"].data_ptr(), call["u_draw"].data_ptr(), 15, at, at + 12 * n_seq, at + 4 * n_seq, at + 8 * n_seq)
    need = m.lib().ws_verify_tree_workspace(r, a)
    r.rows = 0
    draw = m.lib().ws_verify_tree_workspace(r, a)
    r.rows = rows
    parts, row_parts = draw // (32 * n_seq), (need - draw - 16 * rows) // (32 * rows)
    assert parts > 1 and row_parts > 1 and need == 32 * n_seq * parts + 16 * rows + 32 * rows * row_parts
    work = torch.full((need // 8,), -1, dtype=torch.int64, device=DEV)
    run = lambda: m.check(m.lib().ws_verify_tree(torch.cuda.current_stream().cuda_stream, r, a, work.data_ptr(), need), "ws_verify_tree")  # noqa: E731
    run()
    left = work.cpu()
    of_draw, decided, of_rows = left[:draw // 8].view(n_seq, 4, parts), left[draw // 8:draw // 8 + 2 * rows], left[draw // 8 + 2 * rows:].view(rows, 4, row_parts)
    assert not small[2 * n_seq:3 * n_seq].any() and (of_draw != -1).all()
    assert not decided.any()
    read = [sum(counts[:s]) + i for s in range(n_seq) for i in range(counts[s])]
    assert ((of_rows[read] == 0) | (of_rows[read] == -1)).all()  # (-1: rows of nodes without children)
    assert (of_rows[[sum(counts[:s]) for s in range(n_seq) if counts[s] > 1]] == 0).all()
    call["seq_off"].zero_()
    run()
    left = work.cpu()[:draw // 8].view(n_seq, 4, parts)
    assert (small[2 * n_seq:3 * n_seq] == 1).all()
    tag = left[:, 0] ^ left[:, 1]
    assert (tag == tag[0, 0]).all() and int(tag[0, 0]) != 0  # (the words that say only that one is there)
    assert not left[:, 2:].any()


# ---- attention


def attend_case(counts, lengths, heads, kv_heads, dim, page, dtype, seed, layout="tokens", spare=2, mask="tree", slots=False, extra=0):
    g = torch.Generator().manual_seed(seed)
    n_seq, rows = len(counts), sum(counts)
    need = [-(-(a + b) // page) for a, b in zip(lengths, counts)]
    pages, wide = sum(need) + spare, max(need + [1]) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((n_seq + (3 if slots else 0), wide), -1, dtype=torch.int32)
    slot = torch.randperm(n_seq + 3, generator=g)[:n_seq].to(torch.int32) if slots else None
    for s, n in enumerate(need):
        table[int(slot[s]) if slots else s, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    k, v = (torch.randn((pages, page, kv_heads, dim), generator=g).to(dtype) for _ in range(2))
    q = (torch.randn((rows + extra, heads, dim), generator=g) * 2.0).to(dtype)
    # stale memory: what no sequence holds is no number
    used = torch.zeros((pages, page), dtype=torch.bool)
    for s in range(n_seq):
        row = table[int(slot[s]) if slots else s]
        for p in range(lengths[s] + counts[s]):
            used[row[p // page], p % page] = True
    k[~used], v[~used] = math.nan, math.inf
    if mask == "tree":
        parents = tr.random_trees(counts, 3, g)
        masks = tr.stage(parents, [0] * n_seq)[0]
    elif mask == "any":
        masks = torch.randint(-(1 << 62), 1 << 62, (rows,), generator=g) * 2 + torch.randint(2, (rows,), generator=g)
        masks[::5] = 0
    else:
        masks = None
    if masks is not None and extra:
        masks = torch.cat([masks, torch.zeros(extra, dtype=torch.int64)])

    def device(t):
        if layout == "tokens":
            return t.to(DEV)
        if layout == "heads":  # a page's heads apart
            return t.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
        wide_t = torch.zeros((page, pages, kv_heads + 1, dim + 16), dtype=dtype, device=DEV)  # padded, pages inside of tokens
        wide_t[:, :, :kv_heads, :dim] = t.permute(1, 0, 2, 3).to(DEV)
        return wide_t[:, :, :kv_heads, :dim].permute(1, 0, 2, 3)
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    call = dict(q=q.to(DEV), k=device(k), v=device(v), table=to(table), length=torch.tensor(lengths, dtype=torch.int32, device=DEV), seq_off=to(tr.offsets(counts)), mask=to(masks), slot=to(slot))
    host = dict(q=q[:rows], k=k, v=v, table=table, lengths=lengths, counts=counts, masks=masks, slots=None if slot is None else slot.tolist())
    return call, host


def check_attention(call, host, scale=None, **more):
    m = gc.pkg()
    dim, rows = host["q"].shape[2], host["q"].shape[0]
    want, lse, tol, lse_tol = tr.attention(scale=dim ** -0.5 if scale is None else scale, **host)
    got, got_lse = m.tree_attention(want_lse=True, scale=scale, **call, **more)
    near(got[:rows], want, tol, "out")
    near(got_lse[:rows], lse, lse_tol, "lse")
    return got, got_lse


ATTEND = [  # nodes, lengths, heads, kv heads, dim, page, dtype
    ([1], [0], 1, 1, 64, 16, BF16), ([1], [1], 4, 2, 128, 16, F32), ([1, 1, 1], [31, 32, 33], 8, 2, 128, 1, BF16), ([1] * 9, [0, 1, 127, 128, 129, 255, 256, 300, 1000], 16, 4, 64, 8, BF16),
    ([1, 1], [5000, 4999], 32, 8, 128, 64, BF16), ([5], [100], 7, 1, 80, 4, BF16), ([64], [0], 2, 2, 128, 16, BF16), ([64, 3], [65, 700], 8, 1, 128, 32, BF16), ([9, 0, 1, 17], [77, 50, 300, 0], 14, 2, 64, 2, F32),
    ([64] * 3, [190, 0, 1025], 10, 2, 64, 256, BF16), ([33, 12], [640, 9], 6, 2, 256, 16, BF16), ([7, 64], [260, 130], 8, 2, 256, 128, F32), ([20, 64], [1000, 31], 8, 2, 128, 16, F32), ([2, 60], [40, 800], 12, 4, 96, 16, BF16),
    ([30] * 8, [64 * i + 1 for i in range(8)], 4, 4, 8, 16, BF16), ([64], [3000], 64, 4, 128, 16, BF16), ([1], [7], 300, 1, 40, 16, BF16), ([3] * 300, [i % 97 for i in range(300)], 2, 1, 64, 8, BF16)]


@pytest.mark.parametrize("case", ATTEND, ids=[f"{len(c[0])}x{max(c[0])}_{max(c[1])}_{c[2]}h{c[3]}_{c[4]}_p{c[5]}_{str(c[6])[6:]}" for c in ATTEND])
@pytest.mark.parametrize("mask", ["tree", "any", "chain"])
def test_attention(case, mask):
    counts, lengths, heads, kv_heads, dim, page, dtype = case
    layout = {"tree": "tokens", "any": "heads", "chain": "padded"}[mask]
    call, host = attend_case(counts, lengths, heads, kv_heads, dim, page, dtype, len(counts) + dim + heads, layout=layout, mask=mask, slots=mask == "any")
    a = check_attention(call, host)
    for nodes in (1, 64):  # other builds: the word on the nodes is a hint
        check_attention(call, host, max_nodes=nodes)
    b = check_attention(call, host)
    rows = sum(counts)
    assert all(torch.equal(x[:rows], y[:rows]) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype,dim,heads,n", [(BF16, 128, 4, 40), (BF16, 64, 2, 7), (BF16, 128, 2, 64), (BF16, 256, 8, 64), (F32, 64, 4, 64), (F32, 128, 8, 20), (BF16, 128, 16, 64)])
@pytest.mark.parametrize("before", [0, 25, 60, 100, 127, 1000])
def test_attention_nodes_that_workgroups_share(dtype, dim, heads, n, before):
    """Infinities in the V of nodes that several workgroups' positions hold: seen by those that see the node, whichever workgroup has it."""
    m = gc.pkg()
    call, host = attend_case([n], [before], heads, 2, dim, 16, dtype, before + dim + n)
    clean = m.tree_attention(**call)
    G = heads // 2
    for node in sorted({0, 1, 3, 31 - before % 32, 64 - before % 64, n // 2, n - 1}):
        if not 0 <= node < n:
            continue
        t = call["v"].clone()
        p = before + node
        t[host["table"][0, p // 16], p % 16, 1, 2] = math.inf
        got = m.tree_attention(**{**call, "v": t})
        sees = torch.tensor([bool(int(host["masks"][r]) >> node & 1) for r in range(n)])
        want = clean.clone()
        want[sees.to(DEV), G:, 2] = math.inf
        assert torch.equal(got, want), (node, int((got != want).sum()))


def test_attention_unseen_places_do_not_matter():
    """Infinities and NaN in the K and V of nodes that a row does not see leave it alone; those that see them get what the formula gives."""
    m = gc.pkg()
    for dtype, dim, heads, n in ((BF16, 128, 4, 40), (F32, 64, 4, 9), (BF16, 64, 2, 5), (BF16, 256, 8, 33), (F32, 128, 8, 20)):
        call, host = attend_case([n, 6], [150, 2], heads, 2, dim, 16, dtype, dim + n)
        clean = m.tree_attention(**call, want_lse=True)
        rows = n + 6
        sees = torch.tensor([[int(host["masks"][r]) >> j & 1 for j in range(n)] for r in range(n)], dtype=torch.bool)
        for node, value, side in ((3, math.inf, "v"), (4, -math.inf, "v"), (n - 1, math.nan, "v"), (2, math.nan, "k"), (1, math.inf, "k")):
            t = call[side].clone()
            p = 150 + node
            t[host["table"][0, p // 16], p % 16, 0, 1] = value
            got = m.tree_attention(**{**call, side: t}, want_lse=True)
            blind = torch.cat([~sees[:, node], torch.ones(6, dtype=torch.bool)])
            G = heads // 2
            for a, b in zip(got, clean):
                assert torch.equal(a[blind], b[blind]) and torch.equal(a[:, G:], b[:, G:]), (dtype, node, side)
            seeing = got[0][~blind][:, :G].float().cpu()
            if side == "v":
                rest = [d for d in range(dim) if d != 1]
                assert torch.equal(got[0][~blind][:, :G][..., rest], clean[0][~blind][:, :G][..., rest])
                assert (torch.isnan(seeing[..., 1]) if math.isnan(value) else seeing[..., 1] == value).all()
            else:
                assert torch.isnan(seeing).any(-1).logical_or((seeing != clean[0][~blind][:, :G].float().cpu()).any(-1)).all()
        # two infinities of either sign: no number for who sees both
        t = call["v"].clone()
        for node, value in ((0, math.inf), (1, -math.inf)):
            t[host["table"][0, (150 + node) // 16], (150 + node) % 16, 0, 1] = value
        got = m.tree_attention(**{**call, "v": t})[:n, 0, 1].float().cpu()
        assert torch.isnan(got[sees[:, 1]]).all() and (got[~sees[:, 1]] == math.inf).all()


def test_attention_pages_that_hold_nothing():
    """Entries outside the pages, positions past the table, slots that do not exist: not seen."""
    m = gc.pkg()
    for page, dtype, dim in ((1, BF16, 128), (16, BF16, 128), (16, F32, 64), (64, BF16, 64)):
        for n in (1, 30):
            call, host = attend_case([n, n, n], [200, 300, 90], 4, 2, dim, page, dtype, page + n)
            table = host["table"].clone()
            table[0, 1], table[0, 120 // page], table[1, -2] = -1, 1 << 30, -(1 << 31)
            table[2, :] = 100000
            host["table"], call["table"] = table, table.to(DEV)
            got, lse = check_attention(call, host)
            assert not got[2 * n:].any() and (lse[2 * n:] == -math.inf).all()
            call["slot"] = torch.tensor([1, 3, -1], dtype=torch.int32, device=DEV)
            host["slots"] = [1, 3, -1]
            check_attention(call, host)
            host["slots"], call["slot"] = None, None
            short = table[:, :90 // page].contiguous()  # the tables end before the texts do
            host["table"], call["table"] = short, short.to(DEV)
            check_attention(call, host)


def test_attention_rows_behind_the_last_and_strided():
    """Rows behind the last sequence are left as they were; q and out with rows and heads apart."""
    m = gc.pkg()
    call, host = attend_case([5, 3], [100, 400], 6, 2, 64, 16, BF16, 1, extra=4)
    q = torch.zeros((12, 9, 72), dtype=BF16, device=DEV)[:, :6, :64]
    q.copy_(call["q"])
    out = torch.full((12, 8, 80), 7.0, dtype=BF16, device=DEV)
    got = m.tree_attention(**{**call, "q": q}, out=out[:, :6, :64])
    want, _, tol, _ = tr.attention(scale=0.125, **host)
    near(got[:8], want, tol, "out")
    assert (out[8:] == 7.0).all() and (out[:, 6:] == 7.0).all() and (out[:, :, 64:] == 7.0).all()


def test_attention_scores_far_apart():
    """Scores that grow along the text by thousands, and a text whose first token outweighs all others."""
    for dtype in (BF16, F32):
        call, host = attend_case([17], [600], 4, 2, 64, 16, dtype, 3)
        for grow in (1.0, -1.0):
            by = (1.0 + torch.arange(617) * 0.05)[:, None, None] if grow > 0 else (1.0 + torch.arange(616, -1, -1) * 0.05)[:, None, None]
            used = host["table"][0, :39].long()
            flat = host["k"][used].reshape(-1, 2, 64).clone()
            flat[:617] = (flat[:617].float() * by).to(dtype)
            k = host["k"].clone()
            k[used] = flat.view(39, 16, 2, 64)
            check_attention({**call, "k": k.to(DEV)}, {**host, "k": k}, scale=0.5)


@pytest.mark.parametrize("dtype,dim,n,strides", [(BF16, 128, 1, ((1 << 31) + 64, 256, 128)), (BF16, 128, 40, ((1 << 31) + 64, 256, 128)), (F32, 64, 9, (128, 1 << 28, 64)), (BF16, 64, 20, (128, 1 << 28, 64))])
def test_attention_of_a_cache_beyond_32_bits(dtype, dim, n, strides):
    """Pages, or a page's tokens, further apart than 32 bits count."""
    call, host = attend_case([n, n], [30, 3], 8, 2, dim, 16, dtype, n + dim, spare=1)
    far = {}
    for side in ("k", "v"):
        shape = call[side].shape
        room = torch.empty(sum((size - 1) * by for size, by in zip(shape, strides)) + dim, dtype=dtype, device=DEV)
        far[side] = room.as_strided(shape, (*strides, 1))
        far[side].copy_(call[side])
        assert far[side].numel() * far[side].element_size() < 1 << 24 < 1 << 32 < room.numel() * room.element_size()
    check_attention({**call, **far}, host)


def test_attention_captured_and_replayed():
    m = gc.pkg()
    cases = [attend_case([12, 1, 33], [300 * i + 10, 5, 77], 8, 2, 128, 16, BF16, 50)[0] for i in range(1)]
    call, host = attend_case([12, 1, 33], [900, 5, 77], 8, 2, 128, 16, BF16, 51)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.tree_attention(**call)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.tree_attention(**call)
    for lengths in ([900, 5, 77], [3, 0, 0], [450, 4, 60], [900, 5, 77]):
        call["length"].copy_(torch.tensor(lengths, dtype=torch.int32))
        call["q"].mul_(-1.0)
        want = m.tree_attention(**call)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_attention_on_two_streams_at_once():
    m = gc.pkg()
    calls = [attend_case([9] * 4, [500 + 100 * i] * 4, 8, 2, 128, 16, BF16, 60 + i)[0] for i in range(2)]
    want = [m.tree_attention(**c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(10):
        for c, st in zip(calls, streams):
            with torch.cuda.stream(st):
                got.append(m.tree_attention(**c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (BF16, 256), (F32, 64), (BF16, 64), (F32, 128)])
def test_attention_infinities_of_some_of_a_workgroups_tiles(dtype, dim):
    """A workgroup works on several sequences' tiles, one behind the other: infinities in the V of some of the sequences' nodes are those sequences' alone, and none is lost."""
    m = gc.pkg()
    n = 2000
    call, host = attend_case([1] * n, [i % 61 for i in range(n)], 4, 2, dim, 16, dtype, dim)
    clean = m.tree_attention(**call)
    t, want = host["v"].clone(), clean.clone()
    for s in range(0, n, 3):
        p = host["lengths"][s]
        t[host["table"][s, p // 16], p % 16, s % 2, 5] = math.inf
        want[s, 2 * (s % 2):2 * (s % 2) + 2, 5] = math.inf
    call["v"] = t.to(DEV)
    for _ in range(3):
        got = m.tree_attention(**call)
        assert torch.equal(got, want), int((got != want).sum())


def test_attention_of_a_slot_that_does_not_exist_behind_infinities():
    """A workgroup that has met infinities in one sequence's nodes begins the text of the next, whose slot does not exist, and others end it: its rows see nothing, whatever lies behind the table."""
    m = gc.pkg()
    n, units = 2002, 9  # (2011 units of 128 positions, four a workgroup of 512: the last text begins in the third of one's, and three workgroups share it)
    lengths = [i % 61 for i in range(n)] + [128 * units - 1]
    call, host = attend_case([1] * (n + 1), lengths, 1, 1, 128, 16, BF16, 5)
    t = host["v"].clone()
    for s in range(n - 4, n + 1):
        t[host["table"][s, lengths[s] // 16], lengths[s] % 16, 0, 3] = math.inf
    call["v"] = t.to(DEV)
    for slot in (n, n + 1, -1):
        call["slot"] = torch.arange(n + 1, dtype=torch.int32, device=DEV)
        call["slot"][n] = slot
        table = torch.cat([host["table"][:n], host["table"][n:].repeat(2, 1)]).to(DEV)
        got, lse = m.tree_attention(**{**call, "table": table[:n]}, want_lse=True)
        assert not got[n].any() and float(lse[n, 0]) == -math.inf
        assert (got[n - 4:n, 0, 3] == math.inf).all() and torch.isfinite(got[:n - 4]).all() and torch.isfinite(lse[:n]).all()
    call["slot"] = None
    got = m.tree_attention(**call)
    assert (got[n - 4:, 0, 3] == math.inf).all() and torch.isfinite(got[n, 0, 4:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [8, 24, 40, 64, 72, 80, 96, 112, 128, 136, 200, 248, 256])
@pytest.mark.parametrize("heads,n", [(2, 1), (2, 24), (8, 40)])
def test_attention_keys_that_are_infinite(dtype, dim, heads, n):
    """A key with -inf where the rows' q is above 0 has the score -inf and weight 0, as if its position were not there: whatever the head's dimensions are filled up with."""
    m = gc.pkg()
    call, host = attend_case([n, 1], [150, 40], heads, 2, dim, 1, dtype, dim + n)
    q, k, table = host["q"].clone(), host["k"].clone(), host["table"].clone()
    gone = [(0, 3), (0, 77), (0, 149), (0, 150 + n // 2), (1, 0), (1, 39)]
    for i, (s, p) in enumerate(gone):
        e = (i * 5 + dim // 3) % dim if i % 2 else i
        q[..., e] = q[..., e].abs() + 0.25
        k[table[s, p], 0, :, e] = -math.inf
        table[s, p] = -1
    call["q"] = q.to(DEV)
    host.update(q=q, table=table)
    for nodes in (0, 1, 64):
        want = check_attention({**call, "table": table.to(DEV)}, host, max_nodes=nodes)
        got = m.tree_attention(want_lse=True, max_nodes=nodes, **{**call, "k": k.to(DEV)})
        for a, b in zip(got, want):
            assert torch.equal(a, b), (nodes, int((a != b).sum()), int(torch.isnan(a).sum()))


def test_verify_history_and_a_path_without_room():
    """With a history a walk that `path` cannot hold is the host's: nothing is appended that the cache could not be brought to. One that fits is appended."""
    m = gc.pkg()
    call, _, ids, _ = verify_case([6, 3, 4, 1], 1, 500, F32, 2, guessed=True, chain=True)
    call["u_accept"][:] = 0.0  # (all are accepted: 5, 2, 3 and none)
    for depth, n_want, status_want in ((5, [5, 2, 3, 0], [0, 0, 0, 0]), (4, [0, 2, 3, 0], [9, 0, 0, 0]), (2, [0, 2, 0, 0], [9, 0, 9, 0]), (1, [0, 0, 0, 0], [9, 9, 9, 0])):
        hist = m.DeviceHistory(4, 12, DEV)
        hist.len[:] = torch.tensor([5, 9, 7, 0], device=DEV, dtype=torch.int32)
        hist.tokens[:] = 77
        want = list(status_want)
        want[1] |= 5 if 9 + 2 + 2 > 12 else 0  # (5 + 5 + 2 tokens fit in 12, 9 + 2 + 2 do not)
        n = [0 if w else k for w, k in zip(want, n_want)]
        n_accepted, path, chosen, status, logprob = (t.cpu() for t in m.verify_tree(depth=depth, hist=hist, **call))
        assert status.tolist() == want and n_accepted.tolist() == n, (depth, status.tolist(), n_accepted.tolist())
        assert [int(c) < 0 for c in chosen] == [w != 0 for w in want]
        for s in range(4):
            assert path[s].tolist() == list(range(1, n[s] + 1)) + [-1] * (depth - n[s])
            before = [5, 9, 7, 0][s]
            assert int(hist.len[s]) == before + (0 if want[s] else n[s] + 1) and int(hist.n_gen[s]) == (0 if want[s] else n[s] + 1)
            first = sum([6, 3, 4, 1][:s])
            text = [77] * 12
            if not want[s]:
                text[before + 1:before + 2 + n[s]] = ids[first + 1:first + 1 + n[s]].tolist() + [int(chosen[s])]
            assert hist.tokens[s].cpu().tolist() == text
        n_accepted, path, chosen, status, _ = (t.cpu() for t in m.verify_tree(depth=depth, **call))  # without one: all are counted, the first named
        assert n_accepted.tolist() == [5, 2, 3, 0] and not status.any() and path[0].tolist() == list(range(1, depth + 1))


EXACT = [  # nodes, lengths, heads, kv heads, dim, page, dtype
    ([1], [8191], 8, 2, 128, 16, BF16), ([1, 1, 1], [4096, 5003, 129], 32, 8, 128, 16, BF16), ([1], [8001], 4, 1, 64, 64, BF16), ([1], [6000], 4, 2, 256, 16, BF16), ([24], [6001], 4, 2, 128, 32, BF16),
    ([64, 5], [8200, 3333], 8, 2, 128, 16, BF16), ([64, 64], [16000, 15001], 16, 4, 128, 16, BF16), ([40], [5001], 4, 1, 64, 16, BF16), ([33], [4097], 4, 2, 256, 16, BF16), ([20, 3], [5000, 4500], 8, 2, 80, 1, BF16),
    ([1], [8000], 8, 2, 64, 16, F32), ([1], [5001], 4, 2, 128, 16, F32), ([1], [4097], 4, 2, 256, 16, F32), ([40, 2], [6001, 40], 4, 1, 64, 16, F32), ([64], [4100], 4, 2, 128, 8, F32), ([9], [3001], 4, 2, 256, 16, F32)]


@pytest.mark.parametrize("case", EXACT, ids=[f"{len(c[0])}x{max(c[0])}_{max(c[1])}_{c[2]}h{c[3]}_{c[4]}_{str(c[6])[6:]}" for c in EXACT])
@pytest.mark.parametrize("mask", ["tree", "any"])
def test_attention_takes_every_position_once(case, mask):
    """q = 0, so that every weight is 1 and a row's sums are counts, which 32 bits hold: element d of V is 1 at the positions that are d modulo head_dim, so that one position more or less, of 126
    at most, shows in bf16 as well; and lse is the logarithm of how many are seen."""
    m = gc.pkg()
    counts, lengths, heads, kv_heads, dim, page, dtype = case
    call, host = attend_case(counts, lengths, heads, kv_heads, dim, page, dtype, 7 * dim + sum(counts), mask=mask)
    v = host["v"].clone()
    for s, (n, c) in enumerate(zip(lengths, counts)):
        p = torch.arange(n + c)
        pg = host["table"][s, p // page].long()
        v[pg, p % page] = 0.0
        for h in range(kv_heads):
            v[pg, p % page, h, (p + 3 * h) % dim] = 1.0
    call["v"], call["q"] = v.to(DEV), torch.zeros_like(call["q"])
    got, lse = (t.cpu().double() for t in m.tree_attention(want_lse=True, **call))
    G = heads // kv_heads
    for r, (s, see) in enumerate(tr.visible(lengths, counts, host["masks"])):
        at = see.nonzero()[:, 0]
        n = at.numel()
        for h in range(kv_heads):
            have = torch.bincount((at + 3 * h) % dim, minlength=dim).double()
            # 1 / n, its product, and the result: half a step each (2^-24, 2^-24, the type's); a count that is off by one is off by 1 / count
            tol = have / n * (2.0 ** -23 + tr.HALF[dtype]) * 1.01
            assert 1.0 / float(have.max()) > 2.0 * 1.01 * (2.0 ** -23 + tr.HALF[dtype])  # (so that it shows, rounded either way)
            mine = got[r, h * G:(h + 1) * G]
            assert ((mine - have / n).abs() <= tol).all(), (r, h)
        # the logarithm to base two by one instruction (a step), its factor and product (half a step each) of a number of 14 at most
        assert ((lse[r] - math.log(n)).abs() <= 2.0 ** -22 * max(1.0, math.log(n))).all() and 1.0 / n > 2.0 ** -20 * math.log(n), r


def test_attention_replayed_with_other_tables_masks_and_offsets():
    """A captured call: other tables, masks, offsets, lengths and rows than it was captured with, the eager call's answer each time."""
    m = gc.pkg()
    cases = [attend_case(c, n, 8, 2, 128, 16, BF16, 70 + i, mask=k)[0] for i, (c, n, k) in enumerate([
        ([12, 1, 33], [900, 5, 77], "tree"), ([1, 44, 1], [20, 600, 300], "any"), ([20, 20, 6], [0, 1, 850], "tree"), ([46, 0, 0], [910, 3, 3], "any")])]
    pages, wide = max(c["k"].shape[0] for c in cases), max(c["table"].shape[1] for c in cases)
    call = dict(q=torch.zeros_like(cases[0]["q"]), k=torch.zeros((pages, 16, 2, 128), dtype=BF16, device=DEV), v=torch.zeros((pages, 16, 2, 128), dtype=BF16, device=DEV), table=torch.full((3, wide), -1, dtype=torch.int32, device=DEV),
                length=torch.zeros(3, dtype=torch.int32, device=DEV), seq_off=torch.zeros(4, dtype=torch.int32, device=DEV), mask=torch.zeros(46, dtype=torch.int64, device=DEV))

    def put(c):
        call["table"].fill_(-1)
        for k, v in c.items():
            if v is not None:
                call[k][tuple(slice(0, n) for n in v.shape)].copy_(v)
    put(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.tree_attention(want_lse=True, **call)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.tree_attention(want_lse=True, **call)
    for i in (1, 0, 2, 3, 3, 1, 2, 0):
        put(cases[i])
        want = m.tree_attention(want_lse=True, **cases[i])  # (its own table and pages, as wide as they are)
        for _ in range(3):
            for t in got:
                t.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
