"""Plain implementations in 64 bits, on the host, of the calls over a cycle with a tree of drafts (ws_tree_stage, ws_verify_tree, ws_tree_attention, ws_cache_*), written from the
header's formulas, and what the kernels may be off by."""
import math

import torch

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
TREE_MAX, Q_WORDS = 64, 72
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}  # half a step of a result, relative to it
HOST, HISTORY_FULL = 1, 4


# ---- trees


def random_trees(counts, kids, g):
    """Parents within each sequence, -1 at the root; each node below an earlier one that has room."""
    out = []
    for n in counts:
        mine, room = [], [kids] * n
        for i in range(n):
            free = [j for j in range(i) if room[j]]
            p = free[int(torch.randint(len(free), (1,), generator=g))] if free else -1
            if p >= 0:
                room[p] -= 1
            mine.append(p)
        out.append(mine)
    return out


def offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts, dtype=torch.int64).cumsum(0)), dtype=torch.int32) if len(counts) else torch.zeros(1, dtype=torch.int32)


def stage(parents, lens):
    masks, positions = [], []
    for tree, n in zip(parents, lens):
        above = []
        for i, p in enumerate(tree):
            reached = i == 0 or (0 <= p < i and above[p] is not None)
            above.append(None if not reached else (0 if i == 0 else above[p]) | 1 << i)
        for i, a in enumerate(above):
            m = a if a is not None else 1 << i
            masks.append(m - (1 << 64) if m >> 63 else m)
            positions.append(n + (bin(a).count("1") - 1 if a is not None else 0))
    return torch.tensor(masks, dtype=torch.int64), torch.tensor(positions, dtype=torch.int32)


# ---- verification


def row_probabilities(x, inv_t, allow):
    """p of a row in 64 bits; None where it has none."""
    x = x.double()
    if allow is not None:
        x = torch.where(allow, x, torch.tensor(-math.inf, dtype=F64))
    t = float(inv_t)
    if not (t > 0.0 and t < math.inf) or torch.isnan(x).any() or (x == math.inf).any() or (x == -math.inf).all():
        return None
    w = torch.exp((x - x.max()) * t)
    return w / w.sum()


class Verify:
    """The walk of one sequence: what comes out, and how near each of its comparisons was (relative, and of the draw in shares of the sum)."""

    def __init__(self, rows, ids, parent, u_accept, u_draw, inv_t, allow=None, entries=None):
        self.path, self.logprob, self.status, self.chosen, self.near, self.draw_near = [], [], 0, -1, math.inf, math.inf
        self.tests, self.interval = [], None
        node, n = 0, len(rows)
        if n == 0:
            self.status = HOST
            return
        while True:
            p = row_probabilities(rows[node], inv_t[node], None if allow is None else allow[node])
            if p is None:
                self.status = HOST
                return
            P, V = p.clone(), p.numel()
            Q, entry = None, None if entries is None else entries[node]
            if entry is not None:
                Q = {}
                for i, q in entry:
                    Q[i] = Q.get(i, 0.0) + float(q)
            to = None
            for c in range(node + 1, n):
                if parent[c] != node:
                    continue
                y = int(ids[c])
                q = 1.0 if Q is None else Q.get(y, 0.0)
                mine = float(P[y]) if 0 <= y < V else 0.0
                self.tests.append((c, q, mine))
                self.near = min(self.near, abs(u_accept[c] * q - mine) / max(mine, 1e-300) if mine > 0 or q > 0 else math.inf)
                if u_accept[c] * q < mine:
                    to = c
                    break
                rest = P.clone()
                if Q is None:
                    if 0 <= y < V:
                        rest[y] = 0.0
                else:
                    for i, v in Q.items():
                        if 0 <= i < V:
                            rest[i] = max(float(rest[i]) - v, 0.0)
                    left = sum(v for i, v in Q.items() if i != y)
                    Q = {i: (0.0 if i == y else v) / (left if left > 0 else 1.0) for i, v in Q.items()}
                Z = float(rest.sum())
                if Z > 0:
                    P = rest / Z
            if to is None:
                cum = P.cumsum(0)
                target = u_draw * float(cum[-1])
                above = (cum > target).nonzero()
                pick = int(above[0]) if above.numel() else int(P.nonzero()[-1])
                lo = float(cum[pick - 1]) if pick else 0.0
                self.interval = (lo / float(cum[-1]), float(cum[pick]) / float(cum[-1]))
                self.draw_near = min(abs(target - lo) if pick else math.inf, abs(float(cum[pick]) - target)) / float(cum[-1])
                self.chosen = pick
                self.logprob.append(math.log(float(p[pick])) if p[pick] > 0 else -math.inf)
                return
            self.path.append(to)
            self.logprob.append(math.log(float(p[int(ids[to])])))
            node = to


def uniforms_apart(make, u_accept, u_draw):
    """Uniforms of a sequence moved away from where the comparisons they meet turn: those of tests by a thousandth of the border, the draw's into the middle of its token's share. make(u_accept,
    u_draw) is the walk. Done on the host, before anything is compared."""
    for _ in range(200):
        w = make(u_accept, u_draw)
        moved = False
        for c, q, p in w.tests:
            border = p / q if q > 0 else math.inf
            if border < math.inf and abs(u_accept[c] - border) < 1e-3 * border:
                u_accept[c] = border * (0.99 if u_accept[c] < border else 1.01)
                moved = True
        if w.interval is not None:
            mid = 0.5 * (w.interval[0] + w.interval[1])
            if abs(u_draw - mid) > 0.25 * (w.interval[1] - w.interval[0]):
                u_draw, moved = mid, True
        if not moved:
            return u_accept, u_draw, w
    return u_accept, u_draw, w


# ---- attention


def visible(lengths, counts, masks):
    """For every row: its sequence, and a truth value a position."""
    out, r = [], 0
    for s, n in enumerate(counts):
        for i in range(n):
            m = int(masks[r]) & (1 << 64) - 1 if masks is not None else (2 << i) - 1
            out.append((s, torch.tensor([True] * lengths[s] + [bool(m >> j & 1) for j in range(n)], dtype=torch.bool)))
            r += 1
    return out


def attention(q, k, v, table, lengths, counts, masks, slots, scale, bad_from=None):
    """(out, lse, tolerance of out, of lse) in 64 bits, a row and a head at a time. k, v: [pages, page_tokens, kv_heads, dim]."""
    rows, H, D = q.shape
    page, K = k.shape[1], k.shape[2]
    half, dtype = HALF[q.dtype], q.dtype
    out, lse = torch.zeros((rows, H, D), dtype=F64), torch.full((rows, H), -math.inf, dtype=F64)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for r, (s, see) in enumerate(visible(lengths, counts, masks)):
        slot = slots[s] if slots is not None else s
        pos = torch.arange(see.numel())
        if not 0 <= slot < table.shape[0]:
            continue
        col = pos // page
        inside = col < table.shape[1]
        pg = torch.where(inside, table[slot][col.clamp(max=table.shape[1] - 1)].long(), torch.tensor(-1))
        see = see & (pg >= 0) & (pg < k.shape[0])
        at = see.nonzero()[:, 0]
        if not at.numel():
            continue
        kk, vv = k[pg[at], at % page].double(), v[pg[at], at % page].double()  # [T, K, D]
        qq = q[r].double().view(K, H // K, D)
        z = torch.einsum("kgd,tkd->kgt", qq, kk) * scale
        size = torch.einsum("kgd,tkd->kgt", qq.abs(), kk.abs()) * scale
        p = torch.softmax(z, -1)
        T = at.numel()
        # a score: products of D terms added in 32 bits (a step a term), scaled to base two (two steps), and the power itself (two): relative to the power, |score| steps
        d = (size * (D + 2) * 2.0 ** -23 + (z.abs() + z.abs().amax(-1, keepdim=True)) * 2.0 ** -23 + 2.0 ** -22)
        # sums of up to T terms in 32 bits, of which no more than 33 * 4 are added one to the other before sums of sums: T / 32 + 64 steps
        steps = (T / 32 + 64) * 2.0 ** -23
        pv = torch.einsum("kgt,tkd->kgd", p * (half * (dtype is BF16) + 2 * d + steps), vv.abs())
        mean = (p * d).sum(-1, keepdim=True) + steps
        o = torch.einsum("kgt,tkd->kgd", p, vv)
        out[r] = o.reshape(H, D)
        tol[r] = (pv + o.abs() * (mean + half) + 1e-37).reshape(H, D)
        lse[r] = torch.logsumexp(z, -1).reshape(H)
        lse_tol[r] = (mean[..., 0] + d.amax(-1) + lse[r].view(K, H // K).abs() * 2.0 ** -22 + 2.0 ** -22).reshape(H)
    return out, lse, tol, lse_tol


# ---- the cache's pages


class Pages:
    """The allocator's state as lists, and what the calls do to it."""

    def __init__(self, slots, slot_pages, pages, page_tokens):
        self.table = [[-1] * slot_pages for _ in range(slots)]
        self.held, self.refs, self.free = [0] * slots, [0] * pages, list(range(pages - 1, -1, -1))
        self.slot_pages, self.page = slot_pages, page_tokens
        self.copies = []  # (from page, to page, tokens)

    def _need(self, tokens):
        return -(-tokens // self.page)

    def _serve(self, wanted):
        """Who gets pages: in order, none behind the first for whom they do not suffice."""
        got, used = [], 0
        full = False
        for w in wanted:
            full = full or (w > 0 and used + w > len(self.free))
            ok = w == 0 or not full
            got.append(ok)
            used += w if ok else 0
        return got

    def reserve(self, slots, tokens):
        status, wanted = [], []
        for i, (s, t) in enumerate(zip(slots, tokens)):
            if not 0 <= s < len(self.held) or t < 0 or s in slots[:i]:
                status.append(2)
                wanted.append(0)
            elif self._need(t) > self.slot_pages:
                status.append(1)
                wanted.append(0)
            else:
                status.append(0)
                wanted.append(max(0, self._need(t) - self.held[s]))
        for i, ok in enumerate(self._serve(wanted)):
            if not ok:
                status[i] = 1
                continue
            for _ in range(wanted[i]):
                p = self.free.pop()
                self.table[slots[i]][self.held[slots[i]]] = p
                self.refs[p] = 1
                self.held[slots[i]] += 1
        return status

    def fork(self, src, dst, lengths):
        status, wanted, held = [], [], list(self.held)
        for i, (a, b, t) in enumerate(zip(src, dst, lengths)):
            ok = 0 <= a < len(held) and 0 <= b < len(held) and a != b and t >= 0 and b not in dst[:i]
            ok = ok and held[b] == 0 and held[a] >= self._need(t)
            status.append(0 if ok else 2)
            wanted.append(1 if ok and t % self.page else 0)
        for i, ok in enumerate(self._serve(wanted)):
            if status[i]:
                continue
            if not ok:
                status[i] = 1
                continue
            whole = lengths[i] // self.page
            for j in range(whole):
                p = self.table[src[i]][j]
                self.table[dst[i]][j] = p
                self.refs[p] += 1
            if wanted[i]:
                p = self.free.pop()
                self.table[dst[i]][whole] = p
                self.refs[p] = 1
                self.copies.append((self.table[src[i]][whole], p, lengths[i] % self.page))
            self.held[dst[i]] = whole + wanted[i]
        return status

    def release(self, slots, tokens):
        status, gone = [], []
        for i, (s, t) in enumerate(zip(slots, tokens)):
            if not 0 <= s < len(self.held) or t < 0 or s in slots[:i]:
                status.append(2)
                continue
            status.append(0)
            keep = min(self._need(t), self.held[s])
            for j in range(keep, self.held[s]):
                p = self.table[s][j]
                self.table[s][j] = -1
                self.refs[p] -= 1
                if p not in gone:
                    gone.append(p)
            self.held[s] = keep
        self.free += [p for p in reversed(gone) if self.refs[p] == 0]
        return status
