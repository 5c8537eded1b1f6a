"""Log-probabilities, losses over them and their gradients in 64 bits, from their formulas: what the GPU tests of ws_token_logprobs,
ws_policy_loss, ws_policy_loss_rows and ws_preference_loss compare with. Test infrastructure."""
import math

import torch

EPS = 2.0 ** -24  # half a step of float32


def pack_allow(allow):
    """[rows, V] truth values -> int32 bitmap [rows, (V + 31) / 32]."""
    rows, V = allow.shape
    full = torch.zeros((rows, (V + 31) // 32 * 32), dtype=torch.int64)
    full[:, :V] = allow.to(torch.int64)
    words = (full.reshape(rows, -1, 32) << torch.arange(32)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def score(logits, ids, inv_t=None, allow=None):
    """logits [rows, V] (any float type), ids, inv_t, allow [rows, V] truth values, on the CPU. A dict of float64 tensors: lp, H, m, S, p, a (the
    exponents), per row or logit."""
    x = logits.double()
    rows, V = x.shape
    t = torch.ones(rows, dtype=torch.float64) if inv_t is None else inv_t.double()
    t = torch.where((t > 0) & torch.isfinite(t), t, torch.full_like(t, math.nan))
    if allow is not None:
        x = torch.where(allow, x, torch.full_like(x, -math.inf))
    m = x.amax(1) if V else None
    none = m == -math.inf
    d = (x - m[:, None]) * t[:, None]
    d = torch.where(none[:, None], torch.full_like(d, -math.inf), d)
    e = d.exp()
    S = e.sum(1)
    a = torch.where(d == -math.inf, torch.zeros_like(d), d)
    lnS = S.log()
    H = torch.where(none, torch.zeros_like(S), lnS - (e * a).sum(1) / S)
    has = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1).long()
    lp = d.gather(1, at[:, None])[:, 0] - lnS
    lp = torch.where(none, torch.full_like(lp, -math.inf), lp)
    lp = torch.where(has, lp, torch.zeros_like(lp))
    return dict(lp=lp, H=H, m=torch.where(none, torch.full_like(m, -math.inf), m), S=S, p=torch.where(none[:, None], torch.zeros_like(e), e / S[:, None]),
                a=a, t=t, has=has, at=at, none=none, x=x)


def grad(r, g, h):
    """d_logits in float64 for derivatives g, h (float64 [rows]) by lp and H, and the size of what is added up in each of its entries."""
    g = torch.where(r["has"], g, torch.zeros_like(g))
    lnp = torch.where(r["p"] > 0, r["p"].clamp(min=1e-300).log(), torch.zeros_like(r["p"]))
    inner = r["p"] * (g[:, None] + h[:, None] * (lnp + r["H"][:, None]))
    size = r["p"] * (g.abs()[:, None] + h.abs()[:, None] * (lnp.abs() + r["H"].abs()[:, None]))
    out = -inner
    own = torch.zeros_like(out)
    keep = r["has"] & (r["x"].gather(1, r["at"][:, None])[:, 0] > -math.inf) & ~r["none"]
    own.scatter_(1, r["at"][:, None], torch.where(keep, g, torch.zeros_like(g))[:, None])
    t = r["t"][:, None]
    still = ((g == 0) & (h == 0)) | r["none"]
    out = torch.where(still[:, None], torch.zeros_like(out), (out + own) * t)
    return out, (size + own.abs()) * t


def policy(lp, old, adv, ref=None, w=None, H=None, clip_low=0.2, clip_high=0.2, dual_clip=0.0, kl_coef=0.0, entropy_coef=0.0):
    """(sums [5], g, h, what each sum adds up in size) in float64."""
    n = lp.numel()
    lp, old, A = lp.double(), old.double(), adv.double()
    w = torch.full((n,), 1.0 / max(n, 1), dtype=torch.float64) if w is None else w.double()
    zero = torch.zeros(n, dtype=torch.float64)
    r = (lp - old).exp()
    free, held = r * A, r.clamp(1 - clip_low, 1 + clip_high) * A
    clipped = held < free
    gain = torch.where(clipped, held, free)
    if dual_clip:
        low = (A < 0) & (gain < dual_clip * A)
        gain, clipped = torch.where(low, dual_clip * A, gain), clipped | low
    kl, back = zero, zero
    if ref is not None:
        b = ref.double() - lp
        back = torch.expm1(b)
        kl = back - b
    Hd = zero if H is None else H.double()
    terms = [-gain + (kl_coef * kl if kl_coef else 0) - (entropy_coef * Hd if entropy_coef else 0), -gain, kl, Hd, clipped.double()]
    live = w != 0
    terms = [torch.where(live, w * v, zero) for v in terms]
    g = torch.where(live, w * (torch.where(clipped, zero, -free) - (kl_coef * back if kl_coef else 0)), zero)
    return torch.stack([v.sum() for v in terms]), g, torch.where(live, -entropy_coef * w, zero), torch.stack([v.abs().sum() for v in terms])


def preference(lp, off, ref=None, w=None, beta=0.1, label_smoothing=0.0):
    n, P = lp.numel(), (len(off) - 1) // 2
    d = lp.double() - (0 if ref is None else ref.double())
    s = torch.stack([d[a:b].sum() for a, b in zip(off[:-1], off[1:])]).reshape(P, 2)
    h = beta * (s[:, 0] - s[:, 1])
    soft = lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    each = (1 - label_smoothing) * soft(-h) + label_smoothing * soft(h)
    w = torch.full((P,), 1.0 / P, dtype=torch.float64) if w is None else w.double()
    c = w * beta * (label_smoothing - 1.0 / (1.0 + torch.exp(h)))
    c = torch.where(w != 0, c, torch.zeros_like(c))
    g = torch.zeros(n, dtype=torch.float64)
    for p in range(P):
        g[off[2 * p]:off[2 * p + 1]] = c[p]
        g[off[2 * p + 1]:off[2 * p + 2]] = -c[p]
    return torch.where(w != 0, w * each, torch.zeros_like(each)).sum(), each, beta * s, g


# ---- how far the kernels may be off
# A term 2^a of a row's sum: the difference x - m and the product with the split factor round once each, by EPS |a| at most (in base two; ln 2 in the
# result), the power by one step (2 EPS). A thread adds V / 256 terms and fewer, the wave and the rest in 64 bits; parts are rounded once more.
def sum_tol(r, V):
    """Relative error of S, per row."""
    weighted = (r["p"] * r["a"].abs()).sum(1)
    return EPS * (2.0 * weighted + 2.0 + V / 256.0 + 40.0)


def lp_tol(r, V):
    return sum_tol(r, V) + EPS * torch.where(torch.isfinite(r["lp"]), r["lp"], torch.zeros_like(r["lp"])).abs()


def H_tol(r, V):
    """ln S and the mean exponent, which has S's relative error twice, and one rounding a product."""
    mean = (r["p"] * r["a"].abs()).sum(1)
    square = (r["p"] * r["a"] ** 2).sum(1)
    return sum_tol(r, V) * (1.0 + 2.0 * mean) + EPS * (2.0 * square + r["H"].abs() + 4.0 * mean)


def grad_tol(r, size, want, V, dtype, extra=0.0, h=None):
    """Each entry: p as above (its own exponent, S), six roundings of factors and sums (extra: relative error of g and h), and the rounding to the
    logits' type. h, the derivative by the entropy: ln p = d - ln S comes from the S of the stats, a float32. S (1 + e) with |e| <= EPS has ln S + ln(1 + e),
    so ln p is off by up to EPS / (1 - EPS) whatever its size - where one token has nearly all of the row, ln p is 5e-4 and that is more than any rounding
    relative to it - and the entry by t |h| p times that."""
    step = torch.finfo(dtype).eps / 2
    rel = EPS * (2.0 * r["a"].abs() + 12.0) + sum_tol(r, V)[:, None] + extra
    tol = size * rel + want.abs() * step + 2.0 ** -126
    return tol if h is None else tol + (r["t"] * h.double().abs())[:, None] * r["p"] * (EPS / (1.0 - EPS))
