"""The operators that score and train a model on the tokens it answered with, over the real range of their calls.

  score       log-probability of one token a row of logits, with the row's maximum and sum and, where asked for, its entropy
  grad        the gradient of such log-probabilities and entropies with respect to the logits
  policy      the clipped policy loss with a KL term and an entropy bonus, from logits to its gradient in them
  tokens      the same loss over log-probabilities that the caller has
  preference  the loss of paired log ratios, from logits to its gradient in them
  pairs       the same loss over log-probabilities that the caller has

`own` says which side `run` computes: plain torch operations, or the package's calls."""
import math

import torch

own = False

DEVICE = "cuda:0"
SUMS = 5  # loss, surrogate, KL, entropy, clipped share


def listed():
    return [
        # the log-probability that a decode step reports beside its token
        dict(name="score_1x151936_f32", kind="score", rows=1, vocab=151936, dtype="f32", entropy=False, masked=False, skip=0.0),
        # tokens drawn under a grammar's mask, an odd vocabulary
        dict(name="score_200x50257_f32_masked", kind="score", rows=200, vocab=50257, dtype="f32", entropy=True, masked=True, skip=0.0),
        # a prompt scored
        dict(name="score_2048x151936_bf16", kind="score", rows=2048, vocab=151936, dtype="bf16", entropy=False, masked=False, skip=0.0),
        # a small micro-batch with an entropy term, an odd vocabulary
        dict(name="grad_300x50257_f32", kind="grad", rows=300, vocab=50257, dtype="f32", entropy=True, masked=False, skip=0.0),
        # supervised tokens: a quarter of the rows are the prompt's, without a target
        dict(name="grad_1024x151936_bf16", kind="grad", rows=1024, vocab=151936, dtype="bf16", entropy=False, masked=False, skip=0.25),
        # a handful of tokens, as an online learner takes them
        dict(name="policy_16x151936_bf16", kind="policy", rows=16, vocab=151936, dtype="bf16", entropy=True, masked=False, skip=0.0, kl=True),
        # fp32 logits, tokens drawn under a mask
        dict(name="policy_256x50257_f32_masked", kind="policy", rows=256, vocab=50257, dtype="f32", entropy=True, masked=True, skip=0.0, kl=True),
        # a micro-batch of rollouts, prompts among them
        dict(name="policy_2048x151936_bf16", kind="policy", rows=2048, vocab=151936, dtype="bf16", entropy=True, masked=False, skip=0.2, kl=True),
        # the largest: a long vocabulary, no KL term and no entropy
        dict(name="policy_4096x262144_bf16", kind="policy", rows=4096, vocab=262144, dtype="bf16", entropy=False, masked=False, skip=0.0, kl=False),
        # a batch of rollouts whose log-probabilities come from elsewhere (logits split over devices)
        dict(name="tokens_65536", kind="tokens", rows=65536, vocab=0, dtype="f32", entropy=True, masked=False, skip=0.2, kl=True),
        # four pairs of answers of up to 257 tokens
        dict(name="preference_4x257x151936_bf16", kind="preference", pairs=4, longest=257, vocab=151936, dtype="bf16"),
        # a batch of pairs scored before
        dict(name="pairs_64x2048", kind="pairs", pairs=64, longest=2048, vocab=0, dtype="f32"),
    ]


def _between(rng, lo, hi):
    """A whole number between the two, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "grad", "grad", "policy", "policy", "policy", "tokens", "preference", "pairs"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "tokens":
        return dict(kind=kind, rows=_between(rng, 1, 262144), vocab=0, dtype="f32", entropy=rng.random() < 0.5, masked=False,
                    skip=round(rng.uniform(0.0, 0.5), 3), kl=rng.random() < 0.5)
    if kind == "pairs":
        return dict(kind=kind, pairs=_between(rng, 1, 256), longest=_between(rng, 1, 4096), vocab=0, dtype="f32")
    vocab = _between(rng, 1000, 262144)
    if rng.random() < 0.5:
        vocab = rng.choice([32000, 32768, 50257, 65536, 128256, 151936, 151937, 262144])
    if kind == "preference":
        pairs = _between(rng, 1, 16)
        most = min(1024, max(1, 400_000_000 // (vocab * pairs)))
        return dict(kind=kind, pairs=pairs, longest=_between(rng, 1, most), vocab=vocab, dtype=dtype)
    rows = _between(rng, 1, min(8192, max(1, 400_000_000 // vocab)))
    case = dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, entropy=rng.random() < 0.5, masked=rng.random() < 0.3,
                skip=rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.5), 3)]))
    if kind == "policy":
        case["kl"] = rng.random() < 0.5
    return case


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _lengths(case, g):
    """Lengths of a batch's answers, ragged: 2 * pairs of them, from one token up; the same total for every seed."""
    n = 2 * case["pairs"]
    share = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    lengths = (1 + (case["longest"] - 1) * share).round().to(torch.int64)
    return lengths[torch.randperm(n, generator=g)]


def _rows(case):
    if "rows" in case:
        return case["rows"]
    return int(_lengths(case, torch.Generator().manual_seed(0)).sum())


def _skipped(case):
    return int(case.get("skip", 0.0) * _rows(case))


CHUNK = 1 << 26  # logits made at a time


def prepare(case, seed):
    host = torch.Generator().manual_seed(1000003 * int(seed) + 17)
    g = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 29)
    rows, V, kind = _rows(case), case["vocab"], case["kind"]
    s = dict(case=case, kind=kind)

    def normal(n, sigma):
        return torch.randn(n, generator=g, device=DEVICE) * sigma

    counts = torch.ones(rows, dtype=torch.bool)
    counts[torch.randperm(rows, generator=host)[:_skipped(case)]] = False
    counts = counts.to(DEVICE)

    if V:
        # logits of a language model: a broad bulk and in each row one token that stands out by up to 14; the row's token is drawn from them
        s["inv_t"] = 1.0 / (0.7 + 0.6 * torch.rand(rows, generator=g, device=DEVICE))
        s["logits"] = torch.empty((rows, V), dtype=_dtype(case), device=DEVICE)
        s["allow"] = None
        words = (V + 31) // 32
        if case.get("masked"):
            s["allow"] = torch.empty((rows, words), dtype=torch.int32, device=DEVICE)
        ids = torch.empty(rows, dtype=torch.int32, device=DEVICE)
        scored = torch.empty(rows, device=DEVICE)
        step = max(1, CHUNK // V)
        for a in range(0, rows, step):
            b = min(rows, a + step)
            x = torch.randn((b - a, V), generator=g, device=DEVICE) * 2.0
            x.scatter_add_(1, torch.randint(V, (b - a, 1), generator=g, device=DEVICE), 14.0 * torch.rand((b - a, 1), generator=g, device=DEVICE))
            s["logits"][a:b] = x
            z = s["logits"][a:b].float() * s["inv_t"][a:b, None]
            if case.get("masked"):  # a random eighth of the tokens: three bits drawn together
                bits = [torch.randint(-(1 << 31), 1 << 31, (b - a, words), generator=g, device=DEVICE, dtype=torch.int64) for _ in range(3)]
                s["allow"][a:b] = (bits[0] & bits[1] & bits[2]).to(torch.int32)
                z = z.masked_fill(~_bits(s["allow"][a:b], V), -math.inf)
            race = torch.empty_like(z).exponential_(generator=g)
            pick = (z - race.log()).argmax(1)
            ids[a:b] = pick
            scored[a:b] = z.gather(1, pick[:, None])[:, 0] - torch.logsumexp(z, 1)
            del x, z, race
        s["ids"] = torch.where(counts, ids, torch.full_like(ids, -1))
    else:
        scored = -torch.empty(rows, device=DEVICE).exponential_(generator=g)
    if kind == "grad":
        s["stats"], s["entropy"] = _stats(s, case["entropy"])
        s["d_logprob"] = torch.where(counts, normal(rows, 1.0 / max(1, rows)), torch.zeros(rows, device=DEVICE))
        s["d_entropy"] = torch.where(counts, torch.full((rows,), -0.01 / max(1, rows), device=DEVICE), torch.zeros(rows, device=DEVICE)) if case["entropy"] else None
    if kind in ("policy", "tokens"):
        s["old"] = scored + normal(rows, 0.2)
        s["ref"] = scored + normal(rows, 0.3) if case["kl"] else None
        s["advantage"] = normal(rows, 1.0)
        s["weight"] = counts.float() / max(1, rows - _skipped(case))
        s["args"] = dict(clip_low=0.2, clip_high=0.28, dual_clip=3.0, kl_coef=0.04 if case["kl"] else 0.0, entropy_coef=0.01 if case["entropy"] else 0.0)
        if kind == "tokens":
            s["logprob"] = scored
            s["entropy"] = (torch.rand(rows, generator=g, device=DEVICE) * 6.0) if case["entropy"] else None
    if kind in ("preference", "pairs"):
        lengths = _lengths(case, host)
        off = torch.zeros(lengths.numel() + 1, dtype=torch.int64)
        off[1:] = lengths.cumsum(0)
        s["seq_off"] = off.to(torch.int32).to(DEVICE)
        s["ref"] = scored + normal(rows, 0.3)
        s["args"] = dict(beta=0.1, label_smoothing=0.05)
        if kind == "pairs":
            s["logprob"] = scored
    return s


def _bits(words, V):
    """A bitmap's rows as truth values."""
    return (((words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1) != 0).reshape(words.shape[0], -1)[:, :V]


def _stats(s, want_entropy):
    """What the forward pass of a training step keeps for its backward pass: {maximum, sum} and entropy of every row."""
    rows, V = s["logits"].shape
    stats, entropy, step = torch.empty((rows, 2), device=DEVICE), torch.empty(rows, device=DEVICE), max(1, CHUNK // V)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        _, stats[a:b], entropy[a:b] = _plain_score(s["logits"][a:b], s["ids"][a:b], s["inv_t"][a:b], None if s["allow"] is None else s["allow"][a:b], True)[:3]
    return stats, entropy if want_entropy else None


# ---- the plain form: elementary operations on float32, sums of a row and of a batch in float64


def _plain_score(logits, ids, inv_t, allow, want_entropy):
    x = logits.float()
    V = x.shape[1]
    if allow is not None:
        x = x.masked_fill(~_bits(allow, V), -math.inf)
    top = x.amax(1)
    d = (x - top[:, None]) * inv_t[:, None]
    e = d.exp()
    total = e.sum(1, dtype=torch.float64)
    has = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1).long()[:, None]
    logprob64 = torch.where(has, d.gather(1, at)[:, 0].double() - total.log(), torch.zeros_like(total))
    entropy64 = None
    if want_entropy:
        part = (e * d.masked_fill(d == -math.inf, 0.0)).sum(1, dtype=torch.float64)
        entropy64 = total.log() - part / total
    stats = torch.stack([top, total.float()], 1)
    return logprob64.float(), stats, None if entropy64 is None else entropy64.float(), logprob64, entropy64, d, e, total


def _plain_grad(d, e, total, ids, inv_t, d_logprob, entropy, d_entropy, dtype):
    V = e.shape[1]
    p = e * (1.0 / total)[:, None].float()
    c = d_logprob[:, None]
    if d_entropy is not None:
        c = c + d_entropy[:, None] * (d.masked_fill(d == -math.inf, 0.0) - total.log().float()[:, None] + entropy[:, None])
    out = -p * c
    has = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1).long()[:, None]
    out.scatter_add_(1, at, torch.where(has & torch.isfinite(d.gather(1, at)[:, 0]), d_logprob, torch.zeros_like(d_logprob))[:, None])
    return (out * inv_t[:, None]).to(dtype)


def _plain_policy(logprob, old, ref, advantage, weight, entropy, clip_low, clip_high, dual_clip, kl_coef, entropy_coef):
    """In float64: a ratio next to the clip decides whether its token has a gradient."""
    delta = logprob.double() - old.double()
    A, w = advantage.double(), weight.double()
    ratio = delta.exp()
    free, held = ratio * A, ratio.clamp(1.0 - clip_low, 1.0 + clip_high) * A
    gain = torch.minimum(free, held)
    clipped = held < free
    if dual_clip:
        floor = dual_clip * A
        low = (A < 0) & (gain < floor)
        gain, clipped = torch.where(low, floor, gain), clipped | low
    zero = torch.zeros_like(gain)
    g = torch.where(clipped, zero, -free)
    kl = zero
    if ref is not None:
        back = ref.double() - logprob.double()
        kl = torch.expm1(back) - back
        g = g - kl_coef * torch.expm1(back)
    H = zero if entropy is None else entropy.double()
    each = -gain + kl_coef * kl - entropy_coef * H
    counts = w != 0
    total = lambda v: torch.where(counts, w * v, zero).sum()  # noqa: E731
    sums = torch.stack([total(each), total(-gain), total(kl), total(H), total(clipped.double())]).float()
    d_logprob = torch.where(counts, w * g, zero)
    return sums, d_logprob.float(), (-entropy_coef * w).float() if entropy is not None else None


def _plain_preference(logprob, ref, seq_off, beta, label_smoothing):
    off = seq_off.long()
    rows = logprob.shape[0]
    of = torch.searchsorted(off, torch.arange(rows, device=logprob.device), right=True) - 1  # each row's answer
    sums = torch.zeros(off.numel() - 1, dtype=torch.float64, device=logprob.device).index_add_(0, of, logprob.double() - ref.double())
    h = beta * (sums[0::2] - sums[1::2])
    P = h.numel()
    softplus = lambda v: v.clamp(min=0.0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    loss = (1.0 - label_smoothing) * softplus(-h) + label_smoothing * softplus(h)
    c = beta / P * (label_smoothing - 1.0 / (1.0 + h.exp()))
    slope = torch.stack([c, -c], 1).reshape(-1)
    reward = (beta * sums).reshape(P, 2)
    return (loss.sum() / P).float().reshape(1), loss.float(), reward.float(), slope[of].float()


def _plain(s):
    kind, case = s["kind"], s["case"]
    if kind == "tokens":
        return _plain_policy(s["logprob"], s["old"], s["ref"], s["advantage"], s["weight"], s["entropy"], **s["args"])
    if kind == "pairs":
        return _plain_preference(s["logprob"], s["ref"], s["seq_off"], **s["args"])
    logits, ids, inv_t = s["logits"], s["ids"], s["inv_t"]
    if kind == "score":
        return _plain_score(logits, ids, inv_t, s["allow"], case["entropy"])[:3]
    if kind == "grad":
        x = logits.float()
        if s["allow"] is not None:
            x = x.masked_fill(~_bits(s["allow"], x.shape[1]), -math.inf)
        d = (x - s["stats"][:, :1]) * inv_t[:, None]
        return _plain_grad(d, d.exp(), s["stats"][:, 1].double(), ids, inv_t, s["d_logprob"], s["entropy"], s["d_entropy"], logits.dtype)
    if kind == "preference":
        logprob, _, _, _, _, d, e, total = _plain_score(logits, ids, inv_t, None, False)
        loss, each, reward, d_logprob = _plain_preference(logprob, s["ref"], s["seq_off"], **s["args"])
        return loss, each, reward, logprob, _plain_grad(d, e, total, ids, inv_t, d_logprob, None, None, logits.dtype)
    want = case["entropy"]
    logprob, _, entropy, logprob64, entropy64, d, e, total = _plain_score(logits, ids, inv_t, s["allow"], want)
    sums, d_logprob, d_entropy = _plain_policy(logprob64, s["old"], s["ref"], s["advantage"], s["weight"], entropy64, **s["args"])
    out = _plain_grad(d, e, total, ids, inv_t, d_logprob, entropy, d_entropy, logits.dtype)
    counts = (s["weight"] != 0) & (ids >= 0)
    none = torch.zeros_like(logprob)
    return sums, torch.where(counts, logprob, none), torch.where(counts, entropy, none) if want else None, out


def run(state):
    if not own:
        return _plain(state)
    from __graft_entry__ import load_package
    m = load_package()
    s, kind, case = state, state["kind"], state["case"]
    if kind == "score":
        return m.token_logprobs(s["logits"], s["ids"], inv_t=s["inv_t"], allow=s["allow"], want_entropy=case["entropy"])
    if kind == "grad":
        return m.token_logprobs_grad(s["logits"], s["ids"], s["stats"], d_logprob=s["d_logprob"], entropy=s["entropy"], d_entropy=s["d_entropy"],
                                     inv_t=s["inv_t"], allow=s["allow"])
    if kind == "policy":
        return m.policy_loss_rows(s["logits"], s["ids"], s["old"], s["advantage"], ref_logprob=s["ref"], weight=s["weight"], inv_t=s["inv_t"],
                                  allow=s["allow"], want_entropy=case["entropy"], **s["args"])
    if kind == "tokens":
        return m.policy_loss(s["logprob"], s["old"], s["advantage"], ref_logprob=s["ref"], entropy=s["entropy"], weight=s["weight"], **s["args"])
    if kind == "pairs":
        return m.preference_loss(s["logprob"], s["seq_off"], ref_logprob=s["ref"], **s["args"])
    logprob, stats, _ = m.token_logprobs(s["logits"], s["ids"], inv_t=s["inv_t"])
    loss, each, reward, d_logprob = m.preference_loss(logprob, s["seq_off"], ref_logprob=s["ref"], **s["args"])
    return loss, each, reward, logprob, m.token_logprobs_grad(s["logits"], s["ids"], stats, d_logprob=d_logprob, inv_t=s["inv_t"])


def work(case):
    rows, V, kind = _rows(case), case["vocab"], case["kind"]
    live = rows - _skipped(case)
    e = 4 if case["dtype"] == "f32" else 2
    # rows that count for nothing are not read; every row of a gradient is written. Operations a logit: difference, scale, exponential,
    # sum (and maximum) forwards, two more for the entropy; scale and product backwards
    if kind == "tokens":
        arrays = 4 + (1 if case["kl"] else 0) + (1 if case["entropy"] else 0) + 1 + (1 if case["entropy"] else 0)
        return {"bytes": 4 * rows * arrays + 4 * SUMS, "flops": 30 * rows}
    if kind == "pairs":
        return {"bytes": 4 * rows * 3 + 4 * (2 * case["pairs"] + 1) + 4 * (3 * case["pairs"] + 1), "flops": 4 * rows}
    mask = live * ((V + 31) // 32) * 4 if case.get("masked") else 0
    read, written = live * V * e + mask, rows * V * e
    extra = 2 if case.get("entropy") else 0
    if kind == "score":
        return {"bytes": read + rows * (4 + 4 + 12 + (4 if extra else 0)), "flops": live * V * (5 + extra)}
    if kind == "grad":
        return {"bytes": read + written + rows * (20 + (8 if extra else 0)), "flops": live * V * (5 + extra)}
    per_row = 32 if kind == "policy" else 20
    return {"bytes": read + written + rows * per_row, "flops": live * V * (8 + 2 * extra)}


# ---- the definition in float64, its gradients by differentiation


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "tokens":
        lp = s["logprob"].double().requires_grad_()
        H = None if s["entropy"] is None else s["entropy"].double().requires_grad_()
        sums = _exact_policy(lp, H, s, slice(None))
        grads = torch.autograd.grad(sums[0], [lp] + ([H] if H is not None else []))
        return sums.detach(), grads[0], grads[1] if H is not None else None
    if kind == "pairs":
        lp = s["logprob"].double().requires_grad_()
        loss, each, reward = _exact_preference(lp, s)
        return loss.detach().reshape(1), each.detach(), reward.detach(), torch.autograd.grad(loss, lp)[0]
    rows, V = s["logits"].shape
    if rows * V > 1_200_000_000:
        return None
    step, outs = max(1, (1 << 25) // V), []
    slope = None
    if kind == "preference":
        lp = torch.cat([_exact_score(s, slice(a, min(rows, a + step)))[0] for a in range(0, rows, step)]).requires_grad_()
        loss, each, reward = _exact_preference(lp, s)
        slope = torch.autograd.grad(loss, lp)[0]
    for a in range(0, rows, step):
        at = slice(a, min(rows, a + step))
        if kind == "score":
            logprob, top, total, H, _ = _exact_score(s, at)
            outs.append((logprob, torch.stack([top, total], 1), H))
            continue
        x = s["logits"][at].double().requires_grad_()
        logprob, _, _, H, counts = _exact_score(s, at, x)
        if kind == "grad":
            aim = (logprob * s["d_logprob"][at].double()).sum()
            if s["d_entropy"] is not None:
                aim = aim + (H * s["d_entropy"][at].double()).sum()
            outs.append((torch.autograd.grad(aim, x)[0].float(),))
        elif kind == "preference":
            outs.append((torch.autograd.grad((logprob * slope[at]).sum(), x)[0].float(),))
        else:
            sums = _exact_policy(logprob, H if case["entropy"] else None, s, at)
            live = counts & (s["weight"][at] != 0)
            d = torch.autograd.grad(sums[0], x)[0].float()
            outs.append((sums.detach(), torch.where(live, logprob.detach(), 0.0), torch.where(live, H.detach(), 0.0), d))
        del x
    if kind == "score":
        logprob, stats, H = (torch.cat(v) for v in zip(*outs))
        return logprob, stats, H if case["entropy"] else None
    if kind == "grad":
        return torch.cat([o[0] for o in outs])
    if kind == "preference":
        return loss.detach().reshape(1), each.detach(), reward.detach(), lp.detach(), torch.cat([o[0] for o in outs])
    sums = torch.stack([o[0] for o in outs]).sum(0)
    logprob, H, d = (torch.cat([o[k] for o in outs]) for k in (1, 2, 3))
    return sums, logprob, H if case["entropy"] else None, d


def _exact_score(s, at, x=None):
    x = s["logits"][at].double() if x is None else x
    z = x * s["inv_t"][at].double()[:, None]
    if s["allow"] is not None:
        z = torch.where(_bits(s["allow"][at], x.shape[1]), z, -math.inf)
    lse = torch.logsumexp(z, 1)
    ids = s["ids"][at].long()
    counts = (ids >= 0) & (ids < x.shape[1])
    rows = torch.arange(ids.numel(), device=ids.device)
    picked = z[rows, torch.where(counts, ids, 0)]
    logprob = torch.where(counts, picked, lse) - lse
    logp = z - lse[:, None]
    p = logp.exp()
    H = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    top = z.detach().amax(1) / s["inv_t"][at].double()
    return logprob, top, (lse.detach() - z.detach().amax(1)).exp(), H, counts


def _exact_policy(lp, H, s, at):
    o = s["args"]
    w, A = s["weight"][at].double(), s["advantage"][at].double()
    r = torch.exp(lp - s["old"][at].double())
    inside = torch.clamp(r, 1.0 - o["clip_low"], 1.0 + o["clip_high"])
    gain = torch.where(A >= 0, torch.clamp(r, max=1.0 + o["clip_high"]), torch.clamp(r, 1.0 - o["clip_low"], o["dual_clip"])) * A
    held = ((A > 0) & (r > inside)) | ((A < 0) & ((r < inside) | (r > o["dual_clip"])))
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        q = torch.exp(s["ref"][at].double() - lp)
        kl = q - torch.log(q) - 1.0
    ent = torch.zeros_like(lp) if H is None else H
    return torch.stack([(w * (-gain + o["kl_coef"] * kl - o["entropy_coef"] * ent)).sum(), (w * -gain).sum(), (w * kl).sum(), (w * ent).sum(), (w * held.double()).sum()])


def _exact_preference(lp, s):
    o, off = s["args"], s["seq_off"].tolist()
    gap = lp - s["ref"].double()
    reward = o["beta"] * torch.stack([gap[a:b].sum() for a, b in zip(off[:-1], off[1:])]).reshape(-1, 2)
    h = reward[:, 0] - reward[:, 1]
    each = -(1.0 - o["label_smoothing"]) * torch.nn.functional.logsigmoid(h) - o["label_smoothing"] * torch.nn.functional.logsigmoid(-h)
    return each.mean(), each, reward
