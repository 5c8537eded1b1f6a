"""GPU: the pages of a paged cache (ws_cache_reserve, _fork, _release, _keep) against lists on the host (tree_ref.Pages), and a cycle with trees of drafts from its stage to its cache."""
import math
import random

import pytest
import torch

import gpu_cases as gc
import tree_ref as tr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def numbered(c, seed=0):
    """The cache's memory filled with numbers of its own places."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in (c.k, c.v):
        t.copy_(torch.randn(t.shape, generator=g, device=DEV))


def same(c, p):
    assert c.table.cpu().tolist() == p.table and c.held.cpu().tolist() == p.held and c.refs.cpu().tolist() == p.refs
    n = int(c.n_free[0])
    assert c.free[:n].cpu().tolist() == p.free
    # every page is held as often as its count says, or free
    seen = [0] * len(p.refs)
    for row in p.table:
        for e in row:
            if e >= 0:
                seen[e] += 1
    assert seen == p.refs and sorted(p.free) == [i for i, r in enumerate(p.refs) if r == 0]


def copied(before, c, p):
    """The copies since the last look, done on the host."""
    want = [t.clone() for t in before]
    for a, b, n in p.copies:
        for w, t in zip(want, before):
            w[:, b, :n] = t[:, a, :n]
    p.copies = []
    for w, t in zip(want, (c.k, c.v)):
        assert torch.equal(w, t)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("page,pages,slots,wide", [(1, 40, 6, 20), (4, 24, 5, 9), (16, 200, 40, 8), (256, 7, 4, 3)])
def test_pages_through_many_calls(page, pages, slots, wide, seed):
    """Random calls, good and bad ones: every table, count and free page as the lists have it, every copy where it should be and nothing else touched."""
    m = gc.pkg()
    r = random.Random(1000 * seed + page)
    c = m.PagedCache.empty(2, pages, page, 2, 16, slots, wide, dtype=BF16 if seed % 2 else F32)
    numbered(c, seed)
    p = tr.Pages(slots, wide, pages, page)
    full = bad = shared = 0
    for _ in range(200):
        what, n = r.choice(["reserve", "reserve", "fork", "fork", "release"]), r.randint(1, max(1, slots // 2))
        name = lambda: r.randint(-1, slots) if r.random() < 0.08 else r.randrange(slots)  # noqa: E731
        tokens = lambda: r.choice([0, 1, page, page + 1, r.randint(0, page * wide), -1 if r.random() < 0.1 else page, page * (wide + 1) if r.random() < 0.1 else 2 * page])  # noqa: E731
        before = (c.k.clone(), c.v.clone())
        if what == "reserve":
            s, t = [name() for _ in range(n)], [tokens() for _ in range(n)]
            got, want = c.reserve(i32(s), i32(t)), p.reserve(s, t)
        elif what == "release":
            s, t = [name() for _ in range(n)], [r.choice([0, 0, 1, page, 3 * page, -1 if r.random() < 0.1 else 0]) for _ in range(n)]
            got, want = c.release(i32(s), i32(t)), p.release(s, t)
        else:
            held = [i for i in range(slots) if p.held[i]]
            empty = [i for i in range(slots) if not p.held[i]]
            a = [r.choice(held) if held and r.random() < 0.9 else name() for _ in range(n)]
            b = [r.choice(empty) if empty and r.random() < 0.9 else name() for _ in range(n)]
            t = [r.randint(0, p.held[x] * page) if 0 <= x < slots and r.random() < 0.9 else tokens() for x in a]
            got, want = c.fork(i32(a), i32(b), i32(t)), p.fork(a, b, t)
        assert got.cpu().tolist() == want, what
        full, bad, shared = full + want.count(1), bad + want.count(2), max(shared, max(p.refs))
        same(c, p)
        copied(before, c, p)
    assert full and bad and shared > 1


def test_many_slots_and_long_texts():
    """1024 slots in a call; entries of more than one round of the workgroup's threads; pages shared by slots of one call go back once."""
    m = gc.pkg()
    c, p = m.PagedCache.empty(1, 20000, 2, 1, 8, 1100, 3000), tr.Pages(1100, 3000, 20000, 2)
    first = list(range(1023, -1, -1))
    need = [(7 * i) % 31 for i in first]
    assert c.reserve(i32(first), i32(need)).cpu().tolist() == p.reserve(first, need) == [0] * 1024
    same(c, p)
    assert c.reserve(i32([1024]), i32([6000])).cpu().tolist() == p.reserve([1024], [6000]) == [0]
    assert c.fork(i32([1024] * 5), i32(range(1025, 1030)), i32([6000, 5999, 4001, 0, 1])).cpu().tolist() == p.fork([1024] * 5, list(range(1025, 1030)), [6000, 5999, 4001, 0, 1]) == [0] * 5
    same(c, p)
    gone = [1024, 1025, 1027, 1026, 3, 1029]
    assert c.release(i32(gone), i32([100, 0, 0, 7, 0, 0])).cpu().tolist() == p.release(gone, [100, 0, 0, 7, 0, 0]) == [0] * 6
    same(c, p)
    assert c.release(i32(first), i32([0] * 1024)).cpu().tolist() == p.release(first, [0] * 1024)
    same(c, p)
    assert c.reserve(i32([]), i32([])).numel() == 0 and c.fork(i32([]), i32([]), i32([])).numel() == 0
    with pytest.raises(m.WsError):
        c.reserve(i32([0] * 1025), i32([0] * 1025))


@pytest.mark.parametrize("dtype,page,kv_heads,dim,layers,layout", [(BF16, 16, 8, 128, 3, "plain"), (F32, 1, 2, 64, 2, "plain"), (BF16, 4, 3, 80, 2, "heads"), (BF16, 64, 1, 8, 5, "padded"), (F32, 2, 4, 256, 1, "heads")])
def test_keep(dtype, page, kv_heads, dim, layers, layout):
    m = gc.pkg()
    g = torch.Generator().manual_seed(page + dim)
    n_seq, lengths = 9, [0, 1, 15, 16, 17, 100, 63, 5, 90]
    need = [-(-(n + 64) // page) for n in lengths]
    pages, wide = sum(need) + 2, max(need) + 1
    shape = (layers, pages, page, kv_heads, dim)
    k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    order, table = torch.randperm(pages, generator=g).tolist(), torch.full((n_seq + 2, wide), -1, dtype=torch.int32)
    slot = torch.randperm(n_seq + 2, generator=g)[:n_seq].to(torch.int32)
    for s, n in enumerate(need):
        table[slot[s], :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    paths = [[], [1], [3], [1, 2, 3], [2, 3, 5, 9, 20, 33, 40, 41, 50, 63], list(range(1, 64)), [5, 7, 7, 9], [64, 70], [4, 0, 6]]
    depth = 63
    path = torch.full((n_seq, depth), -1, dtype=torch.int32)
    counts = [len(p) for p in paths]
    counts[1] = 40  # more than the path holds: the -1 behind it ends it
    for s, p in enumerate(paths):
        path[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    table[slot[8], (lengths[8] + 4) // page] = -1 if page == 1 else table[slot[8], (lengths[8] + 4) // page]

    def device(t):
        if layout == "heads":
            return t.permute(1, 0, 3, 2, 4).contiguous().to(DEV).permute(1, 0, 3, 2, 4)
        if layout == "padded":
            wide_t = torch.zeros((layers, pages, page + 1, kv_heads, dim + 8), dtype=dtype, device=DEV)
            wide_t[:, :, :page, :, :dim] = t.to(DEV)
            return wide_t[:, :, :page, :, :dim]
        return t.to(DEV)
    dk, dv = device(k), device(v)
    c = m.PagedCache(dk, dv, table.to(DEV), i32([0] * (n_seq + 2)), i32([0] * pages), i32([0] * pages), i32([0]))
    c.keep(path.to(DEV), i32(counts), i32(lengths), slot=slot.to(DEV))
    for t in (k, v):
        for s, p in enumerate(paths):
            last = 0
            for i, node in enumerate(p):
                if not last < node < 64:
                    break
                last = node
                a, b = lengths[s] + node, lengths[s] + 1 + i
                pa, pb = int(table[slot[s], a // page]), int(table[slot[s], b // page])
                if pa >= 0 and pb >= 0:
                    t[:, pb, b % page] = t[:, pa, a % page].clone()
    assert torch.equal(dk.cpu(), k) and torch.equal(dv.cpu(), v)
    c.keep(path[:, :1].contiguous().to(DEV), i32([0] * n_seq), i32(lengths), slot=i32([-1, 100000] + [0] * 7))  # nothing to move, slots that do not exist
    assert torch.equal(dk.cpu(), k)


@pytest.mark.parametrize("strides", [((1 << 27) + 512, (1 << 29) + 1024, 64, 32), (1 << 13, 1 << 14, 1 << 29, 32)])
def test_caches_beyond_32_bits(strides):
    """Layers, pages or tokens further apart than 32 bits count: a fork's copy, an accepted path."""
    m = gc.pkg()
    layers, pages, page, kv_heads, dim = shape = (2, 5, 4, 2, 32)
    sides = []
    for _ in range(2):
        room = torch.empty(sum((size - 1) * by for size, by in zip(shape, (*strides, 1))) + 1, dtype=F32, device=DEV)
        sides.append(room.as_strided(shape, (*strides, 1)))
        assert room.numel() * 4 > 1 << 32
    e = m.PagedCache.empty(*shape, 2, 4, dtype=F32, device=DEV)
    c = m.PagedCache(*sides, e.table, e.held, e.refs, e.free, e.n_free)
    numbered(c)
    want = [t.contiguous() for t in sides]
    assert c.reserve(i32([0]), i32([11])).tolist() == [0] and c.table[0].tolist() == [0, 1, 2, -1]
    assert c.fork(i32([0]), i32([1]), i32([10])).tolist() == [0] and c.table[1].tolist() == [0, 1, 3, -1]
    c.keep(i32([[2, 3]]), i32([2]), i32([6]))  # slot 0: token 8 to 7, 9 to 8
    for t, w in zip(sides, want):
        w[:, 3, :2] = w[:, 2, :2].clone()
        w[:, 1, 3], w[:, 2, 0] = w[:, 2, 0].clone(), w[:, 2, 1].clone()
        assert torch.equal(t, w)


def test_captured_and_replayed():
    """Fork, room for drafts and release in a graph, replayed with eager calls in between: the lists go through the same calls."""
    m = gc.pkg()
    c, p = m.PagedCache.empty(3, 60, 16, 2, 64, 10, 6), tr.Pages(10, 6, 60, 16)
    numbered(c)
    assert c.reserve(i32([0, 1]), i32([37, 64])).cpu().tolist() == p.reserve([0, 1], [37, 64])
    m.lib().ws_probe()
    src, dst, length, need, none = i32([0, 0, 1]), i32([4, 5, 6]), i32([37, 20, 50]), i32([60, 30, 51]), i32([0, 0, 0])

    def branch():
        return c.fork(src, dst, length), c.reserve(dst, need), c.table[4:7].clone(), c.release(dst, none)

    def listed():
        n = length.cpu().tolist()
        return [p.fork([0, 0, 1], [4, 5, 6], n), p.reserve([4, 5, 6], [60, 30, 51]), [list(r) for r in p.table[4:7]], p.release([4, 5, 6], [0, 0, 0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        branch()
    torch.cuda.current_stream().wait_stream(side)
    listed()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = branch()
    for i in range(4):
        length[0] = 16 + 5 * i
        assert [t.cpu().tolist() for t in branch()] == listed()
        for _ in range(2):
            before, p.copies = (c.k.clone(), c.v.clone()), []
            graph.replay()
            torch.cuda.synchronize()
            assert [t.cpu().tolist() for t in got] == listed()
            same(c, p)
            copied(before, c, p)


# ---- a cycle: stage, attention, logits, verification, history, cache


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cycles_with_trees(dtype):
    """Three cycles of a one-layer model over a paged cache. What the model knows of a token is its embedding; a row's attention over what it sees makes its logits. After each cycle the cache holds
    the text's tokens in order, so that the last row's logits are those of the text alone, without any tree."""
    m = gc.pkg()
    g = torch.Generator().manual_seed(4)
    V, H, K, D, page, n_seq = 1000, 8, 2, 64, 16, 5
    embed = torch.randn((V, K * D), generator=g).to(dtype).to(DEV)
    wq, wo = (torch.randn((K * D, H * D), generator=g) / 8).to(dtype).to(DEV), (torch.randn((H * D, V), generator=g) / 4).to(dtype).to(DEV)
    c = m.PagedCache.empty(1, 120, page, K, D, n_seq + 1, 12, dtype=dtype)
    hist = m.DeviceHistory(n_seq + 1, 160, DEV)
    slot = i32([5, 2, 0, 4, 1])
    start = [3, 16, 1, 40, 31]
    text = torch.randint(V, (n_seq + 1, 160), generator=g, dtype=torch.int32)
    hist.tokens.copy_(text)
    for s, n in zip(slot.tolist(), start):
        hist.len[s] = n
    assert not c.reserve(slot, i32(start)).any()

    def write(slots, positions, tokens):  # keys and values: the embedding, negated for the values
        pages = c.table[slots.long(), (positions // page).long()].long()
        e = embed[tokens.long()].view(-1, K, D)
        c.k[0, pages, (positions % page).long()], c.v[0, pages, (positions % page).long()] = e, -e

    for s, n in zip(slot.tolist(), start):
        write(torch.full((n,), s, device=DEV), torch.arange(n, device=DEV), hist.tokens[s, :n])
    u = torch.Generator().manual_seed(9)
    gained = 0
    for cycle in range(3):
        counts = [[7, 1, 12, 20, 33], [4, 9, 1, 64, 2], [16] * 5][cycle]
        rows, parents = sum(counts), tr.random_trees(counts, 2, g)
        off, parent = tr.offsets(counts).to(DEV), i32([p for t in parents for p in t])
        mask, position, length = m.tree_stage(off, rows, parent=parent, hist=hist, slot=slot)
        assert not c.reserve(slot, (length + i32(counts))).any()
        of = torch.repeat_interleave(torch.arange(n_seq, device=DEV), i32(counts).long())
        node = torch.arange(rows, device=DEV) - off[of].long()
        ids = torch.randint(V, (rows,), generator=g, dtype=torch.int32).to(DEV)
        ids[off[:-1].long()] = hist.tokens[slot.long(), hist.len[slot.long()].long()]
        # drafts that are likely: level by level the model's own favourites, as a draft model that has read it would name them
        for _ in range(4):
            write(slot[of], length[of] + node, ids)
            q = (embed[ids.long()] @ wq).view(rows, H, D)
            out = c.attention(0, q, length, off, mask=mask, slot=slot, max_nodes=max(counts))
            logits = (out.reshape(rows, H * D) @ wo).contiguous()
            best = logits.float().topk(2, 1).indices
            up = off[of].long() + parent.clamp(min=0).long()
            mine = torch.where(node % 2 == 0, best[up, 0], best[up, 1]).to(torch.int32)
            ids = torch.where(node == 0, ids, mine)
        u_accept = torch.rand(rows, generator=u, dtype=torch.float64).to(DEV) * 0.5
        before = hist.len.clone()
        n_accepted, path, chosen, status, logprob = m.verify_tree(logits, ids, off, u_accept, torch.rand(n_seq, generator=u, dtype=torch.float64).to(DEV), parent=parent, hist=hist, slot=slot)
        c.keep(path, n_accepted, length, slot=slot)
        c.release(slot, (length + 1 + n_accepted))
        assert not status.any() and torch.equal(hist.len[slot.long()], before[slot.long()] + 1 + n_accepted)
        gained += int(n_accepted.sum())
        # the log-probabilities are those that token_logprobs gives the same rows
        for s in range(n_seq):
            a, k_ = int(off[s]), int(n_accepted[s])
            walk = [0] + path[s, :k_].tolist()
            at = torch.tensor([a + i for i in walk], device=DEV)
            kept = torch.cat([ids[at[1:]], chosen[s:s + 1]])
            lp = m.token_logprobs(logits[at].contiguous(), kept)[0]
            assert torch.allclose(logprob[s, :k_ + 1], lp, atol=2e-6, rtol=1e-6)
        # the text so far, read as a chain of its own in a fresh pool of keys: the last accepted row again
        for s in range(n_seq):
            sl, n = int(slot[s]), int(hist.len[slot[s].long()])
            e = embed[hist.tokens[sl, :n].long()].view(n, K, D)
            pages = c.table[sl, :-(-n // page)].long()
            assert torch.equal(c.k[0, pages].reshape(-1, K, D)[:n], e) and torch.equal(c.v[0, pages].reshape(-1, K, D)[:n], -e), (cycle, s)
            assert int(c.held[sl]) == -(-n // page)
    assert gained > 5
    # forks go on by themselves: the pages that are shared stay as they are
    a, b = slot[:1], i32([3])
    n = int(hist.len[a.long()])
    assert not c.fork(a, b, hist.len[a.long()]).any() and not c.reserve(b, i32([n + 1])).any()
    kept = [c.k[0, c.table[int(a), :-(-n // page)].long()].clone()]
    write(b, i32([n]), i32([1]))
    assert torch.equal(c.k[0, c.table[int(a), :-(-n // page)].long()].reshape(-1, K, D)[:n], kept[0].reshape(-1, K, D)[:n])
    q = (embed[hist.tokens[a.long(), n].long()] @ wq).view(1, H, D)
    write(a, i32([n]), hist.tokens[a.long(), n]) if int(c.held[a.long()]) * page > n else None
    one = c.attention(0, q, i32([n - 1]), i32([0, 1]), slot=a)
    two = c.attention(0, q, i32([n - 1]), i32([0, 1]), slot=b)
    assert torch.equal(one, two) and not math.isnan(float(one.float().sum()))


def test_autograd_sees_what_is_written():
    """A backward pass that has kept a cache's K or V refuses to go on once a call has written there; the tables and counts that the calls write have another version, too."""
    m = gc.pkg()
    one, two, none = i32([0]), i32([20]), i32([0])
    calls = {"reserve": lambda c: c.reserve(i32([1]), two), "release": lambda c: c.release(one, none), "fork": lambda c: c.fork(one, i32([1]), i32([5])), "keep": lambda c: c.keep(i32([[3, -1]]), i32([1]), i32([5]))}
    for name, call in calls.items():
        c = m.PagedCache.empty(1, 8, 16, 1, 16, 2, 3, dtype=F32)
        assert c.reserve(one, two).cpu().tolist() == [0]
        w = torch.ones((), device=DEV, requires_grad=True)
        kept = [(w * t).sum() for t in (c.k, c.v)]
        lists = [c.table, c.held, c.refs, c.free, c.n_free]
        before = [t._version for t in lists]
        call(c)
        assert all((t._version > b) == (name != "keep") for t, b in zip(lists, before)), name
        for y in kept:
            if name in ("fork", "keep"):
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.backward()
            else:
                y.backward()
    with torch.inference_mode():  # (no versions are counted there)
        c = m.PagedCache.empty(1, 8, 16, 1, 16, 2, 3, dtype=F32)
        assert c.reserve(one, two).cpu().tolist() == c.fork(one, i32([1]), i32([5])).cpu().tolist() == c.release(one, none).cpu().tolist() == [0]
        c.keep(i32([[3, -1], [2, -1]]), i32([1, 1]), i32([5, 0]))
