"""The operators of a decoding cycle whose drafted tokens form a tree, over the real range of their calls.

  verify  drafted tokens against the target's probabilities, from given uniforms: the walk down the tree, the token drawn behind it and the log-probabilities of what is kept
  attend  attention of a tree's rows over a paged cache (one row a sequence: plain decoding)
  keep    the accepted path's keys and values moved to where the sequence's text goes on
  fork    a sequence's cache forked into others, room made for their drafts, and given back

`own` says which side `run` computes: plain torch operations, or the package's calls."""
import math

import torch

own = False

DEVICE = "cuda:0"
Q_WORDS, Q_MAX = 72, 32  # a draft distribution: count, up to 32 ids from word 1 on, their probabilities from word 33 on
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a lone request with a chain of four drafts from a draft head's own distributions
        dict(name="verify_1x5x151936_bf16", kind="verify", seqs=1, nodes=5, kids=1, vocab=151936, dtype="bf16", guessed=False, masked=False),
        # a server's batch, trees of a draft model's likeliest tokens
        dict(name="verify_64x16x151936_bf16_guessed", kind="verify", seqs=64, nodes=16, kids=3, vocab=151936, dtype="bf16", guessed=True, masked=False),
        # many sequences under grammars, fp32 logits, an odd vocabulary, siblings drawn without replacement
        dict(name="verify_256x25x50257_f32_masked", kind="verify", seqs=256, nodes=25, kids=2, vocab=50257, dtype="f32", guessed=False, masked=True),
        # a single token of a single sequence
        dict(name="attend_1x1_4096_bf16", kind="attend", seqs=1, nodes=1, longest=4096, ragged=False, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a server's batch of single tokens, ragged
        dict(name="attend_64x1_4096_bf16", kind="attend", seqs=64, nodes=1, longest=4096, ragged=True, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # trees over ragged sequences
        dict(name="attend_16x48_8192_bf16", kind="attend", seqs=16, nodes=48, longest=8192, ragged=True, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # two very long sequences, few key heads
        dict(name="attend_2x64_131072_bf16", kind="attend", seqs=2, nodes=64, longest=131072, ragged=False, heads=32, kv_heads=4, dim=128, page=128, dtype="bf16"),
        # a small fp32 model, odd counts
        dict(name="attend_5x9_1001_f32", kind="attend", seqs=5, nodes=9, longest=1001, ragged=True, heads=14, kv_heads=2, dim=64, page=32, dtype="f32"),
        # a lone request's accepted path, all layers
        dict(name="keep_1x16_28_bf16", kind="keep", seqs=1, nodes=16, longest=1000, layers=28, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a server's batch
        dict(name="keep_64x32_48_bf16", kind="keep", seqs=64, nodes=32, longest=300, layers=48, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a prompt answered four times
        dict(name="fork_1x4_28_bf16", kind="fork", seqs=1, copies=4, nodes=8, longest=1500, layers=28, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # beams of a batch over large pages
        dict(name="fork_16x3_32_bf16", kind="fork", seqs=16, copies=3, nodes=33, longest=700, layers=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number between the two, spread over its logarithm."""
    hi = max(lo, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "attend", "attend", "attend", "keep", "fork"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "verify":
        vocab = _between(rng, 500, 262144)
        if rng.random() < 0.5:
            vocab = rng.choice([32000, 50257, 65536, 128256, 151936, 151937, 262144])
        nodes = _between(rng, 1, 64)
        seqs = _between(rng, 1, min(512, max(1, 300_000_000 // (vocab * nodes))))
        return dict(kind=kind, seqs=seqs, nodes=nodes, kids=rng.choice([1, 2, 3, 4]), vocab=vocab, dtype=dtype, guessed=rng.random() < 0.5, masked=rng.random() < 0.3)
    kv_heads, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([1, 8, 16, 16, 32, 64, 256])
    if kind == "attend":
        nodes = rng.choice([1, 1, _between(rng, 1, 64), _between(rng, 1, 64)])
        longest = _between(rng, 1, 65536)
        group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        most = min(100_000_000 // (longest * kv_heads * dim), 1_500_000_000 // ((longest + nodes) * nodes * kv_heads * group))
        return dict(kind=kind, seqs=_between(rng, 1, min(256, max(1, most))), nodes=nodes, longest=longest, ragged=rng.random() < 0.6, heads=group * kv_heads,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    layers, longest, seqs = _between(rng, 1, 64), _between(rng, 1, 2000), _between(rng, 1, 64)
    copies = rng.choice([1, 2, 3, 4, 8])
    nodes = _between(rng, 1, 64)
    while layers * seqs * (longest + 65 * (copies if kind == "fork" else 1) + 2 * page) * kv_heads * dim > 1_000_000_000:
        layers, seqs, longest = max(1, layers // 2), max(1, seqs // 2), max(1, longest // 2)
    case = dict(kind=kind, seqs=seqs, nodes=nodes, longest=longest, layers=layers, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "fork":
        case["copies"] = copies
    return case


# ---- inputs


def _spread(n, lo, hi):
    """n whole numbers over a range, the same total for every seed."""
    return [round(lo + (hi - lo) * (i + 0.5) / n) for i in range(n)]


def _shuffled(values, g):
    return [values[i] for i in torch.randperm(len(values), generator=g).tolist()]


def _node_counts(case):
    """Nodes of each sequence, its root among them."""
    most = case["nodes"]
    return _spread(case["seqs"], most if case["seqs"] == 1 else max(1, (most + 1) // 2), most)


def _lengths(case):
    longest = case["longest"]
    return _spread(case["seqs"], max(1, longest // 16), longest) if case.get("ragged", True) and case["seqs"] > 1 else [longest] * case["seqs"]


def _deepest(case):
    """Levels below the root that a tree may have."""
    return max(1, case["nodes"] - 1 if case["kids"] == 1 else min(case["nodes"] - 1, 8))


def _trees(counts, kids, deepest, g):
    """Parents of every sequence's nodes: each hangs below an earlier one with room for a child, of the last few rather than the first."""
    parents = []
    for n in counts:
        mine, room, depth = [-1], [kids] * n, [0] * n
        pick = torch.rand(n, generator=g).tolist()
        for i in range(1, n):
            free = [j for j in range(i) if room[j] and depth[j] < deepest]
            free = [j for j in free if j >= i - 2 * kids] or free
            p = free[min(len(free) - 1, int(pick[i] * len(free)))]
            room[p] -= 1
            depth[i] = depth[p] + 1
            mine.append(p)
        parents.append(mine)
    return parents


def _offsets(counts):
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
    return off.to(DEVICE)


CHUNK = 1 << 26  # logits made at a time


def _prepare_verify(case, host, g):
    V, counts = case["vocab"], _shuffled(_node_counts(case), host)
    parents = _trees(counts, case["kids"], _deepest(case), host)
    rows = sum(counts)
    s = dict(seq_off=_offsets(counts), parent=torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=DEVICE), most=max(counts),
             depth=_deepest(case))
    first, at = [0], []
    for n in counts:
        first.append(first[-1] + n)
    for t, f in zip(parents, first):  # each node's row of drafts, and which of them it is
        seen = {}
        for j, p in enumerate(t):
            at.append((f + max(p, 0), seen.get(p, 0)))
            seen[p] = seen.get(p, 0) + 1
    words = (V + 31) // 32
    s["inv_t"] = 1.0 / (0.7 + 0.4 * torch.rand(rows, generator=g, device=DEVICE))
    s["logits"] = torch.empty((rows, V), dtype=DTYPES[case["dtype"]], device=DEVICE)
    s["allow"] = torch.empty((rows, words), dtype=torch.int32, device=DEVICE) if case["masked"] else None
    k = min(Q_MAX, V)
    s["q"] = None if case["guessed"] else torch.zeros((rows, Q_WORDS), dtype=torch.int32, device=DEVICE)
    drafts = torch.empty((rows, k), dtype=torch.int32, device=DEVICE)
    step = max(1, CHUNK // V)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        # a broad bulk and a few tokens that stand out, as a language model's
        x = torch.randn((b - a, V), generator=g, device=DEVICE) * 2.0
        stand = 10.0 + 14.0 * torch.rand((b - a, 1), generator=g, device=DEVICE) - torch.tensor([0.0, 1.0, 2.0, 4.0], device=DEVICE)
        x.scatter_add_(1, torch.randint(V, (b - a, 4), generator=g, device=DEVICE), stand)
        s["logits"][a:b] = x
        z = s["logits"][a:b].float()
        if case["masked"]:  # a random eighth of the tokens and the four that stand out
            bits = [torch.randint(-(1 << 31), 1 << 31, (b - a, words), generator=g, device=DEVICE, dtype=torch.int64) for _ in range(3)]
            ones = (torch.ones((), dtype=torch.int64, device=DEVICE) << torch.arange(32, device=DEVICE))
            top = torch.zeros((b - a, words * 32), dtype=torch.bool, device=DEVICE).scatter_(1, z.topk(min(4, V), 1).indices, True)
            s["allow"][a:b] = ((bits[0] & bits[1] & bits[2]) | (top.view(b - a, words, 32) * ones).sum(2)).to(torch.int32)
            z = z.masked_fill(~_bits(s["allow"][a:b], V), -math.inf)
        # the draft model's view of the row: its likeliest tokens, somewhat off
        z = z * s["inv_t"][a:b, None]
        z = (z + 0.4 * torch.randn(z.shape, generator=g, device=DEVICE)).clamp(min=-1e4)
        vals, ids = z.topk(k, 1)
        p = (vals - vals[:, :1]).exp()
        p = p / p.sum(1, keepdim=True)
        if case["guessed"]:
            drafts[a:b] = ids
            continue
        race = torch.empty_like(p).exponential_(generator=g) / p
        drafts[a:b] = ids.gather(1, race.argsort(1)).to(torch.int32)
        order = ids.argsort(1)
        s["q"][a:b, 0] = k
        s["q"][a:b, 1:1 + k] = ids.gather(1, order).to(torch.int32)
        s["q"][a:b, 33:33 + k] = p.gather(1, order).view(torch.int32)
    at = torch.tensor(at, device=DEVICE)
    s["ids"] = drafts[at[:, 0], at[:, 1].clamp(max=k - 1)].contiguous()
    s["q_off"] = None if case["guessed"] else torch.arange(rows, dtype=torch.int32, device=DEVICE) * Q_WORDS
    s["u_accept"] = torch.rand(rows, generator=g, device=DEVICE, dtype=torch.float64)
    s["u_draw"] = torch.rand(case["seqs"], generator=g, device=DEVICE, dtype=torch.float64)
    return s


def _prepare_attend(case, host, g):
    counts, lengths = _shuffled(_node_counts(case), host), _shuffled(_lengths(case), host)
    page, seqs, dtype = case["page"], case["seqs"], DTYPES[case["dtype"]]
    need = [-(-(n + c) // page) for n, c in zip(lengths, counts)]
    wide, pages = max(need), sum(need) + 3
    where = torch.randperm(pages, generator=host)[:sum(need)].tolist()  # a pool that has been in use for a while
    table = torch.full((seqs, wide), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(where[:n], dtype=torch.int32)
        where = where[n:]
    shape = (pages, page, case["kv_heads"], case["dim"])
    s = dict(k=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype), v=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype), table=table.to(DEVICE),
             length=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), seq_off=_offsets(counts), most=max(counts), longest=max(lengths))
    # a row's scores lie some two either side of zero, as a trained model's do
    s["q"] = torch.randn((sum(counts), case["heads"], case["dim"]), generator=g, device=DEVICE, dtype=dtype) * 2.0
    seen = []
    for t in _trees(counts, 3, 64, host):
        mine = []
        for i, p in enumerate(t):
            mine.append((mine[p] if i else 0) | (1 << i))
        seen += [m - (1 << 64) if m >> 63 else m for m in mine]
    s["mask"] = torch.tensor(seen, dtype=torch.int64, device=DEVICE)
    return s


def _pool(case, slots, need, spare, host, g):
    """A cache whose first slots hold pages for `need` tokens each, and `spare` pages beside them; with what an allocator knows of it."""
    page, dtype = case["page"], DTYPES[case["dtype"]]
    held = [-(-n // page) for n in need] + [0] * (slots - len(need))
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=host).tolist()
    wide = -(-(max(need) + 128) // page) + 1
    table = torch.full((slots, wide), -1, dtype=torch.int32)
    for i, n in enumerate(held):
        table[i, :n] = torch.tensor(order[:n], dtype=torch.int32)
        order = order[n:]
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    free = torch.full((pages,), -1, dtype=torch.int32)
    free[:len(order)] = torch.tensor(order, dtype=torch.int32)
    shape = (case["layers"], pages, page, case["kv_heads"], case["dim"])
    return dict(k=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype), v=torch.randn(shape, generator=g, device=DEVICE, dtype=dtype), table=table.to(DEVICE),
                held=torch.tensor(held, dtype=torch.int32, device=DEVICE), refs=refs.to(DEVICE), free=free.to(DEVICE),
                n_free=torch.tensor([len(order)], dtype=torch.int32, device=DEVICE))


def _accepted(case):
    """Accepted nodes of each sequence: about three in ten of what a path could be, none among them."""
    most = min(case["nodes"] - 1, 8)
    return _spread(case["seqs"], 0 if case["seqs"] > 1 else most, most)


def _prepare_keep(case, host, g):
    lengths, counts = _shuffled(_lengths(case), host), _shuffled(_accepted(case), host)
    pool = _pool(case, case["seqs"], [n + case["nodes"] for n in lengths], 2, host, g)
    most = max(1, max(counts))
    path = torch.full((case["seqs"], most), -1, dtype=torch.int32)
    for i, n in enumerate(counts):
        path[i, :n] = (torch.randperm(case["nodes"] - 1, generator=host)[:n].sort().values + 1).to(torch.int32)
    return dict(pool=pool, path=path.to(DEVICE), n_accepted=torch.tensor(counts, dtype=torch.int32, device=DEVICE),
                length=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), most=most)


def _prepare_fork(case, host, g):
    seqs, copies, page = case["seqs"], case["copies"], case["page"]
    lengths = _shuffled(_lengths(case), host)
    pool = _pool(case, seqs * (1 + copies), lengths, seqs * copies * (2 + -(-case["nodes"] // page)), host, g)
    src = [i for i in range(seqs) for _ in range(copies)]
    to = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return dict(pool=pool, src=to(src), dst=to([seqs + i for i in range(seqs * copies)]), length=to([lengths[i] for i in src]),
                need=to([lengths[i] + case["nodes"] for i in src]), none=to([0] * (seqs * copies)))


def prepare(case, seed):
    host = torch.Generator().manual_seed(1000003 * int(seed) + 17)
    g = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 29)
    s = dict(verify=_prepare_verify, attend=_prepare_attend, keep=_prepare_keep, fork=_prepare_fork)[case["kind"]](case, host, g)
    s["case"], s["kind"] = case, case["kind"]
    return s


def _bits(words, V):
    """A bitmap's rows as truth values."""
    return (((words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1) != 0).reshape(words.shape[0], -1)[:, :V]


# ---- the plain forms


def _plain_verify(s):
    """In float64: uniforms are compared with sums over the whole vocabulary, and the answers are whole numbers."""
    logits, ids, kids, most, depth = s["logits"], s["ids"].long(), s["case"]["kids"], s["most"], s["depth"]
    V, off = logits.shape[1], s["seq_off"].long()
    first, count = off[:-1], off[1:] - off[:-1]
    S = first.numel()
    node = torch.arange(most, device=DEVICE)
    rows = (first[:, None] + node).clamp(max=logits.shape[0] - 1)
    there = (node < count[:, None]) & (node > 0)
    parent = torch.where(there, s["parent"].long()[rows], -1)
    cur, walking = torch.zeros(S, dtype=torch.long, device=DEVICE), torch.ones(S, dtype=torch.bool, device=DEVICE)
    path, accepted = torch.full((S, depth), -1, dtype=torch.int32, device=DEVICE), torch.zeros(S, dtype=torch.int32, device=DEVICE)
    last, last_log = (torch.zeros((S, V), dtype=torch.float64, device=DEVICE) for _ in range(2))
    logprob = torch.zeros((S, depth + 1), dtype=torch.float64, device=DEVICE)
    step = torch.arange(depth + 1, device=DEVICE)
    for _ in range(depth + 1):
        at = first + cur
        x = logits[at].double()
        if s["allow"] is not None:
            x = x.masked_fill(~_bits(s["allow"][at], V), -math.inf)
        z = (x - x.amax(1, keepdim=True)) * s["inv_t"][at].double()[:, None]
        P = z.exp()
        total = P.sum(1, keepdim=True)
        logP, P = z - total.log(), P / total
        if s["q"] is not None:
            entry = s["q"][at]
            listed_here = torch.arange(Q_MAX, device=DEVICE) < entry[:, :1]
            Q = torch.zeros_like(P).scatter_add_(1, torch.where(listed_here, entry[:, 1:33], 0).long(), torch.where(listed_here, entry[:, 33:65].view(torch.float32), 0.0).double())
        below = parent == cur[:, None]
        number = below.cumsum(1)
        moved, to = torch.zeros_like(walking), cur
        for c in range(kids):
            child = below & (number == c + 1)
            has, which = child.any(1) & walking & ~moved, child.int().argmax(1)
            row = first + which
            token = ids[row][:, None]
            if s["q"] is None:
                Q = torch.zeros_like(P).scatter_(1, token, 1.0)
            taken = has & (s["u_accept"][row] * Q.gather(1, token)[:, 0] < P.gather(1, token)[:, 0])
            rejected = (has & ~taken)[:, None]
            rest = (P - Q).clamp(min=0.0)
            total = rest.sum(1, keepdim=True)
            P = torch.where(rejected & (total > 0), rest / total, P)
            less = Q.scatter(1, token, 0.0)
            left = less.sum(1, keepdim=True)
            Q = torch.where(rejected, torch.where(left > 0, less / left, less), Q)
            moved, to = moved | taken, torch.where(taken, which, to)
        ends = (walking & ~moved)[:, None]
        last, last_log = torch.where(ends, P, last), torch.where(ends, logP, last_log)
        here = (step == accepted[:, None]) & moved[:, None]
        path = torch.where(here[:, :depth], to[:, None].to(torch.int32), path)
        logprob = torch.where(here, logP.gather(1, ids[first + to][:, None]), logprob)
        accepted = accepted + moved
        cur, walking = to, moved
    cum = last.cumsum(1)
    end = (last > 0).long().mul(torch.arange(V, device=DEVICE)).amax(1)
    chosen = torch.minimum((cum <= s["u_draw"][:, None] * cum[:, -1:]).sum(1), end)
    logprob = torch.where(step == accepted[:, None], last_log.gather(1, chosen[:, None]), logprob).float()
    return accepted, path, chosen.to(torch.int32), torch.zeros(S, dtype=torch.int32, device=DEVICE), logprob


def _places(table, page, at):
    """Pages and places in them of a table's rows' positions."""
    return table.gather(1, (at // page).clamp(max=table.shape[1] - 1)).long(), at % page


def _plain_attend(s):
    case = s["case"]
    page, H, K, D, most = case["page"], case["heads"], case["kv_heads"], case["dim"], s["most"]
    off, length = s["seq_off"].long(), s["length"].long()
    first, count, S = off[:-1], off[1:] - off[:-1], case["seqs"]
    node = torch.arange(most, device=DEVICE)
    rows, there = (first[:, None] + node).clamp(max=s["q"].shape[0] - 1), node < count[:, None]
    at = torch.arange(s["longest"] + most, device=DEVICE)
    pages, place = _places(s["table"], page, at[None].expand(S, -1))
    inside = at < (length + count)[:, None]
    pages = torch.where(inside, pages, 0)
    k = torch.where(inside[:, :, None, None], s["k"][pages, place].float(), 0.0).permute(0, 2, 3, 1).contiguous()  # [S, K, D, L]
    v = torch.where(inside[:, :, None, None], s["v"][pages, place].float(), 0.0).permute(0, 2, 1, 3).contiguous()
    q = s["q"][rows].float().view(S, most, K, H // K, D).permute(0, 2, 1, 3, 4).reshape(S, K, most * (H // K), D).contiguous()
    own_at = at - length[:, None]
    bit = (s["mask"][rows][:, :, None] >> own_at.clamp(0, 63)[:, None]) & 1
    seen = ((own_at < 0)[:, None] | ((bit != 0) & (own_at < 64)[:, None])) & inside[:, None] & there[:, :, None]
    scores = torch.matmul(q, k) * D ** -0.5
    scores = scores.view(S, K, most, H // K, -1).masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(S, K, most * (H // K), -1), v).view(S, K, most, H // K, D) / total.clamp(min=1e-37)
    return out.permute(0, 2, 1, 3, 4).reshape(S, most, H, D)[there].to(s["q"].dtype)


def _plain_keep(s):
    pool, page = s["pool"], s["case"]["page"]
    i = torch.arange(s["most"], device=DEVICE)
    moved = i < s["n_accepted"][:, None]
    length = s["length"].long()[:, None]
    src = _places(pool["table"], page, length + torch.where(moved, s["path"], 0).long())
    dst = _places(pool["table"], page, length + 1 + i)
    at, to = (src[0][moved], src[1][moved]), (dst[0][moved], dst[1][moved])
    for t in (pool["k"], pool["v"]):
        t[:, to[0], to[1]] = t[:, at[0], at[1]]
    return pool["k"], pool["v"]


def _plain_take(pool, wanted):
    """Pages off the top of the free ones, for each in turn: a matrix of them, who got theirs, how many were taken."""
    upto = wanted.cumsum(0)
    served = upto <= pool["n_free"]
    wide = torch.arange(pool["table"].shape[1], device=DEVICE)
    number = (upto - wanted)[:, None] + wide
    mine = (wide < wanted[:, None]) & served[:, None]
    got = pool["free"].long()[torch.where(mine, pool["n_free"].long() - 1 - number, 0)]
    pool["n_free"] -= (wanted * served).sum().to(torch.int32)
    return got, mine, served


def _plain_fork(s):
    pool, page = s["pool"], s["case"]["page"]
    table, held, refs, free, n_free = (pool[k] for k in ("table", "held", "refs", "free", "n_free"))
    src, dst, length = s["src"].long(), s["dst"].long(), s["length"].long()
    wide = torch.arange(table.shape[1], device=DEVICE)
    # whole pages are shared, the last one is copied as far as it is filled
    whole, part = length // page, length % page
    got, mine, served = _plain_take(pool, (part > 0).long())
    status = torch.where(served, 0, 1).to(torch.int32)
    shared = (wide < whole[:, None]) & served[:, None]
    refs.index_add_(0, table[src][shared].long(), torch.ones_like(table[src][shared]))
    refs[got[mine]] = 1
    copied = (wide == whole[:, None]) & (part > 0)[:, None] & served[:, None]
    new = torch.where(shared, table[src], torch.where(copied, got[:, :1], -1).to(torch.int32))
    table[dst] = new
    held[dst] = (new >= 0).sum(1).to(torch.int32)
    of = table[src].gather(1, whole.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    inside = (torch.arange(page, device=DEVICE) < part[:, None]) & served[:, None]
    one, place = torch.nonzero(inside, as_tuple=True)
    for t in (pool["k"], pool["v"]):
        t[:, got[one, 0], place] = t[:, of[one], place]
    # room for the drafts
    want = (-(-s["need"].long() // page) - held[dst]).clamp(min=0)
    got, mine, served = _plain_take(pool, want)
    refs[got[mine]] = 1
    number = wide - held[dst][:, None]
    put = (number >= 0) & (number < want[:, None]) & served[:, None]
    table[dst] = torch.where(put, got.gather(1, number.clamp(0)).to(torch.int32), table[dst])
    held[dst] += (want * served).to(torch.int32)
    room = torch.where(served, 0, 1).to(torch.int32)
    forked = table[dst]
    # and all of it given back: a page that nobody holds any more goes on top of the free ones, the first given back uppermost
    entries = forked[forked >= 0].long()
    refs.index_add_(0, entries, -torch.ones_like(entries, dtype=torch.int32))
    order = torch.arange(entries.numel(), device=DEVICE)
    lowest = torch.full((refs.numel(),), entries.numel(), dtype=torch.long, device=DEVICE).scatter_reduce_(0, entries, order, "amin")
    gone = entries[(refs[entries] == 0) & (lowest[entries] == order)]
    n = gone.numel()
    free[n_free.long() + torch.arange(n, device=DEVICE)] = gone.flip(0).to(torch.int32)
    n_free += n
    table[dst] = -1
    held[dst] = 0
    return status, room, forked, pool["k"], pool["v"], table, held, refs, free, n_free


PLAIN = dict(verify=_plain_verify, attend=_plain_attend, keep=_plain_keep, fork=_plain_fork)


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return PLAIN[kind](s)
    from __graft_entry__ import load_package
    m = load_package()
    if kind == "verify":
        return m.verify_tree(s["logits"], s["ids"], s["seq_off"], s["u_accept"], s["u_draw"], parent=s["parent"], q=s["q"], q_off=s["q_off"], inv_t=s["inv_t"],
                             allow=s["allow"], depth=s["depth"])
    if kind == "attend":
        return m.tree_attention(s["q"], s["k"], s["v"], s["table"], s["length"], s["seq_off"], mask=s["mask"], max_nodes=s["most"])
    if "cache" not in s:  # the handle that a program keeps beside its memory
        s["cache"] = m.PagedCache(**s["pool"])
    cache, pool = s["cache"], s["pool"]
    if kind == "keep":
        cache.keep(s["path"], s["n_accepted"], s["length"])
        return pool["k"], pool["v"]
    status = cache.fork(s["src"], s["dst"], s["length"])
    room = cache.reserve(s["dst"], s["need"])
    forked = pool["table"][s["dst"].long()]
    cache.release(s["dst"], s["none"])
    return status, room, forked, pool["k"], pool["v"], pool["table"], pool["held"], pool["refs"], pool["free"], pool["n_free"]


def work(case):
    kind, seqs = case["kind"], case["seqs"]
    e = 4 if case["dtype"] == "f32" else 2
    if kind == "verify":
        # the rows that a walk meets, its accepted nodes' and the one it ends at: the inputs are made so that a node's drafts are accepted some six times in ten, those drawn
        # from draft distributions eight
        V, walked, rate = case["vocab"], 0, 0.6 if case["guessed"] else 0.8
        for n in _node_counts(case):
            levels = math.log(1 + n * (1 + 0.5 * (case["kids"] - 1)), 1.8) if case["kids"] > 1 else n - 1
            walked += min(n, sum(rate ** i for i in range(int(levels) + 1)))
        row = V * e + ((V + 31) // 32 * 4 if case["masked"] else 0)
        return {"bytes": int(walked * row) + 40 * sum(_node_counts(case)), "flops": int(walked * V * 5) + seqs * V * 20}
    if kind == "attend":
        K, D, H = case["kv_heads"], case["dim"], case["heads"]
        # lengths and node counts are shuffled apart: their means
        counts, lengths = _node_counts(case), _lengths(case)
        rows, held = sum(counts), sum(lengths) + sum(counts)
        each = rows / seqs
        return {"bytes": 2 * held * K * D * e + 2 * rows * H * D * e + 4 * -(-held // case["page"]) + 8 * rows, "flops": int(4 * each * H * D * held)}
    token = 2 * case["layers"] * case["kv_heads"] * case["dim"] * e
    if kind == "keep":
        moved = sum(_accepted(case))
        return {"bytes": 2 * moved * token + 16 * seqs, "flops": 0}
    copied = sum(n % case["page"] for n in _lengths(case)) * case["copies"]
    entries = sum(-(-n // case["page"]) for n in _lengths(case)) * case["copies"]
    return {"bytes": 2 * copied * token + 40 * entries, "flops": 0}


# ---- the definition in float64


def _exact_verify(s):
    off, parent, ids, u_accept, u_draw = (s[k].tolist() for k in ("seq_off", "parent", "ids", "u_accept", "u_draw"))
    V = s["logits"].shape[1]
    out = torch.zeros((len(u_draw), s["depth"] + 1), dtype=torch.float64)
    for i, (a, b) in enumerate(zip(off[:-1], off[1:])):
        node, level = 0, 0
        while True:
            z = s["logits"][a + node].double() * s["inv_t"][a + node].double()
            if s["allow"] is not None:
                z = torch.where(_bits(s["allow"][a + node][None], V)[0], z, -math.inf)
            logp = torch.log_softmax(z, 0)
            p, to = logp.exp(), None
            q = None
            if s["q"] is not None:
                n = int(s["q"][a + node, 0])
                q = torch.zeros(V, dtype=torch.float64, device=DEVICE)
                q[s["q"][a + node, 1:1 + n].long()] = s["q"][a + node, 33:33 + n].view(torch.float32).double()
            for c in range(node + 1, b - a):
                if parent[a + c] != node:
                    continue
                y = ids[a + c]
                if u_accept[a + c] * (1.0 if q is None else float(q[y])) < float(p[y]):
                    to = c
                    break
                if q is None:
                    p[y] = 0.0
                else:
                    p = torch.relu(p - q)
                    q[y] = 0.0
                    q /= q.sum()
                p /= p.sum()
            if to is None:
                cum = p.cumsum(0)
                out[i, level] = logp[min(int((cum <= u_draw[i] * cum[-1]).sum()), V - 1)]
                break
            out[i, level] = logp[ids[a + to]]
            node, level = to, level + 1
    return out


def exact(case, seed):
    """Whole numbers and moved values have no other form. Attention a sequence and a head at a time, log-probabilities along each sequence's walk."""
    if case["kind"] in ("keep", "fork"):
        return None
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return None, None, None, None, _exact_verify(s)
    page, G, D = case["page"], case["heads"] // case["kv_heads"], case["dim"]
    off, lengths, mask = s["seq_off"].tolist(), s["length"].tolist(), s["mask"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for i in range(case["seqs"]):
        n, L = off[i + 1] - off[i], lengths[i]
        used = s["table"][i, :-(-(L + n) // page)].long()
        k = s["k"][used].reshape(-1, *s["k"].shape[2:])[:L + n].double()
        v = s["v"][used].reshape(-1, *s["v"].shape[2:])[:L + n].double()
        see = torch.ones((n, L + n), dtype=torch.bool)
        for r in range(n):
            for j in range(n):
                see[r, L + j] = bool(mask[off[i] + r] >> j & 1)
        see = see.to(DEVICE)
        for h in range(case["heads"]):
            z = s["q"][off[i]:off[i + 1], h].double() @ k[:, h // G].t().contiguous() / math.sqrt(D)
            out[off[i]:off[i + 1], h] = torch.softmax(z.masked_fill(~see, -math.inf), 1) @ v[:, h // G].contiguous()
    return out
