"""GPU: the operators over log-probabilities where their formulas meet infinities, empty rows and the ends of their types, and what their calls leave behind.
Expected values come from the formulas in 64 bits, with the limits that the header states written out; tolerances as in loss_ref.py, where they are derived."""
import ctypes as C
import math

import pytest
import torch

import gpu_cases as gc
import loss_ref as lr
from test_gpu_loss import BF16, DEV, F32, SPECIAL, make, near

pytestmark = pytest.mark.gpu
INF = math.inf
f32 = lambda *v: torch.tensor(v, dtype=F32)  # noqa: E731


def preference_by_limits(lp, ref, off, w, beta, smoothing):
    """The loss of each pair with a term of factor 0 left out and tokens that neither model can give skipped: (loss, pair losses, rewards, derivatives)."""
    P = (len(off) - 1) // 2
    total, each, reward, d = 0.0, [], [], [0.0] * len(lp)
    for p in range(P):
        s, live = [], []
        for a, b in ((off[2 * p], off[2 * p + 1]), (off[2 * p + 1], off[2 * p + 2])):
            rows = [i for i in range(a, b) if not (lp[i] == -INF and ref[i] == -INF)]
            s.append(math.fsum(lp[i] - ref[i] for i in rows) if all(math.isfinite(lp[i]) and math.isfinite(ref[i]) for i in rows) else sum(lp[i] - ref[i] for i in rows))
            live.append(rows)
        h = beta * (s[0] - s[1])
        soft = lambda v: INF if v == INF else (0.0 if v == -INF else max(v, 0.0) + math.log1p(math.exp(-abs(v))))  # noqa: E731
        loss = 0.0 if smoothing == 1.0 else (1.0 - smoothing) * soft(-h)
        loss += 0.0 if smoothing == 0.0 else smoothing * soft(h)
        sigma = 0.0 if h == INF else (1.0 if h == -INF else 1.0 / (1.0 + math.exp(h)))
        each.append(loss)
        reward.append([beta * s[0], beta * s[1]])
        if w[p] != 0.0:
            total += w[p] * loss
            for k, sign in ((0, 1.0), (1, -1.0)):
                for i in live[k]:
                    d[i] = sign * w[p] * beta * (smoothing - sigma)
    return [torch.tensor(v, dtype=torch.float64) for v in ([total], each, reward, d)]


@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
@pytest.mark.parametrize("where", ["chosen", "rejected", "both weigh nothing", "neither model", "reference"])
@pytest.mark.parametrize("lengths", [[3, 2, 4, 5, 1, 1], [700, 513, 30, 1030, 2, 9]])
def test_preference_of_tokens_that_a_mask_leaves_out(lengths, where, smoothing):
    """A token of log-probability -inf in one pair of three: that pair's loss goes to its limit, the others' and all gradients stay. Sums in 64 bits, outputs rounded once: 1e-10 as in
    test_gpu_loss.py."""
    m = gc.pkg()
    g = torch.Generator().manual_seed(7)
    off = [0]
    for n in lengths:
        off.append(off[-1] + n)
    n = off[-1] + 2
    lp, ref = -5.0 * torch.rand(n, generator=g), -5.0 * torch.rand(n, generator=g)
    w = f32(0.5, 0.25, 1.0)
    last = off[4] - 1 if where == "rejected" else off[3] - 1  # of the middle pair's second or first answer
    if where == "neither model":
        lp[last] = ref[last] = lp[off[4] - 1] = ref[off[4] - 1] = -INF
    elif where == "reference":
        ref[last] = -INF
    else:
        lp[last] = -INF
    if where == "both weigh nothing":
        lp[off[4] - 1] = -INF
        w[1] = 0.0
    beta = 0.1
    got = m.preference_loss(lp.to(DEV), torch.tensor(off, dtype=torch.int32, device=DEV), ref_logprob=ref.to(DEV), weight=w.to(DEV), beta=beta, label_smoothing=smoothing)
    want = preference_by_limits(lp.double().tolist(), ref.double().tolist(), off, w.double().tolist(), beta, smoothing) if where != "both weigh nothing" else None
    if want is None:  # (the difference of the two has no value: the pair's loss is NaN, and counts for nothing)
        assert math.isnan(got[1][1].item()) and not got[3][off[2]:off[4]].any() and got[2][1].tolist() == [-INF, -INF]
        lp[off[2]:off[4]] = 0.0
        want = preference_by_limits(lp.double().tolist(), ref.double().tolist(), off, w.double().tolist(), beta, smoothing)
        got = [got[0], got[1].clone(), got[2].clone(), got[3]]
        got[1][1], got[2][1] = want[1][1], want[2][1]
    tol = lambda v: torch.nan_to_num((lr.EPS * 1.001 + 1e-10) * v.abs(), posinf=0.0) + 1e-10  # noqa: E731
    for a, b, what in zip(got[:3], want[:3], ("loss", "pair_loss", "reward")):
        near(a, b, tol(b), what)
    near(got[3], want[3], (lr.EPS * 1.001 + 1e-10) * want[3].abs() + 2.0 ** -149, "d_logprob")
    if where == "rejected" and smoothing == 0.0:
        assert got[1][1].item() == 0.0 and math.isfinite(got[0].item())
    if where == "chosen" and smoothing == 1.0:
        assert got[1][1].item() == 0.0 and math.isfinite(got[0].item())
    if where == "neither model":
        assert bool(torch.isfinite(got[0]).all()) and got[3][last].item() == 0.0 and got[3][off[2]].item() != 0.0


def test_preference_without_a_reference_and_a_token_that_a_mask_leaves_out():
    m = gc.pkg()
    lp = f32(-1.0, -2.0, -INF, -1.5, -0.5)
    loss, each, reward, d = m.preference_loss(lp.to(DEV), torch.tensor([0, 2, 3, 4, 5], dtype=torch.int32, device=DEV), beta=0.5)
    other = math.log1p(math.exp(0.5))  # (h = -0.5 of the second pair: -1.5 against -0.5, halved)
    assert each[0].item() == 0.0 and abs(each[1].item() - other) <= 2 * lr.EPS * other and abs(loss.item() - other / 2) <= 2 * lr.EPS * other
    assert reward[0].tolist() == [-1.5, -INF] and d[:3].tolist() == [0.0, 0.0, 0.0] and d[3].item() < 0.0 < d[4].item()


# (logprob, old, advantage, ref): tokens where a difference of infinities or 0 * inf stands in the formulas
AT_THE_ENDS = [(-INF, -2.0, 1.0, -1.0), (-INF, -2.0, -1.0, -1.0), (-INF, -2.0, 1.0, -INF), (-INF, -2.0, -1.0, -INF), (-1.0, -2.0, 1.0, -INF), (-INF, -2.0, 0.0, -1.0), (-1.25, -1.0, 0.5, -0.75),
               (-1.0, -1.25, 0.5, -1.0), (-1.0, -900.0, 0.0, -1.0), (-1.0, -INF, 0.0, -1.0), (-1.0, -INF, 1.0, -1.0), (-1.0, -INF, -1.0, -1.0), (-1.0, -900.0, -2.0, -1.5),
               (-900.0, -1.0, 0.0, -900.0), (-INF, -INF, 1.0, -1.0), (-INF, -INF, -1.0, -INF), (-INF, -INF, 0.0, -2.0)]


def policy_by_limits(lp, old, A, ref, w, H, clip_low, clip_high, dual_clip, kl_coef, entropy_coef):
    """One token: ([loss, surrogate, kl, entropy, clipped], derivative by the log-probability, by the entropy)."""
    lp = -INF if lp < -3.4028236e38 else lp  # (a float's)
    if w == 0.0 or (lp == -INF and old == -INF):
        return [0.0] * 5, 0.0, 0.0
    ratio = 0.0 if lp == -INF else (INF if lp - old > 709.0 else math.exp(lp - old))
    times = lambda a, b: 0.0 if b == 0.0 else a * b  # noqa: E731
    free, held = times(ratio, A), times(min(max(ratio, 1.0 - clip_low), 1.0 + clip_high), A)
    gain, clipped = (held, True) if held < free else (free, False)
    if dual_clip and A < 0.0 and gain < dual_clip * A:
        gain, clipped = dual_clip * A, True
    kl, back = 0.0, 0.0
    if ref is not None and not (lp == -INF and ref == -INF):
        b = ref - lp
        kl, back = (INF, INF) if b > 709.0 else ((INF, -1.0) if b == -INF else (math.expm1(b) - b, math.expm1(b)))
    loss = -gain + (kl_coef * kl if kl_coef else 0.0) - entropy_coef * H
    return [w * loss, -w * gain, w * kl, w * H, w * clipped], w * ((0.0 if clipped else -free) - (kl_coef * back if kl_coef else 0.0)), -entropy_coef * w


@pytest.mark.parametrize("dual_clip", [0.0, 3.0])
@pytest.mark.parametrize("kl_coef", [0.0, 0.05])
@pytest.mark.parametrize("with_ref", [False, True])
def test_policy_loss_at_the_ends(with_ref, kl_coef, dual_clip):
    """Each token by itself, then all that stay finite together. 64 bits, rounded once: half a step."""
    m = gc.pkg()
    if kl_coef and not with_ref:
        pytest.skip("a KL term needs a reference")
    o = dict(clip_low=0.2, clip_high=0.28, dual_clip=dual_clip, kl_coef=kl_coef, entropy_coef=0.01)
    finite = []
    for lp, old, A, ref in AT_THE_ENDS:
        want = policy_by_limits(lp, old, A, ref if with_ref else None, 1.0, 2.0, **o)
        d = dict(ref_logprob=f32(ref).to(DEV) if with_ref else None, entropy=f32(2.0).to(DEV), **o)
        sums, g, h = m.policy_loss(f32(lp).to(DEV), f32(old).to(DEV), f32(A).to(DEV), **d)
        sums_w = torch.tensor(want[0], dtype=torch.float64)
        near(sums, sums_w, torch.nan_to_num(sums_w.abs(), posinf=0.0) * lr.EPS * 1.001 + 1e-12, ("sums", lp, old, A, ref))
        near(g, torch.tensor([want[1]], dtype=torch.float64), (0.0 if math.isinf(want[1]) else abs(want[1])) * lr.EPS * 1.001, ("d_logprob", lp, old, A, ref))
        near(h, torch.tensor([want[2]], dtype=torch.float64), abs(want[2]) * lr.EPS * 1.001, ("d_entropy", lp, old, A, ref))
        if all(math.isfinite(v) for v in want[0]):
            finite.append((lp, old, A, ref, want))
    assert len(finite) >= 4
    n = len(finite)
    col = lambda k: torch.tensor([f[k] for f in finite], dtype=F32, device=DEV)  # noqa: E731
    sums, g, h = m.policy_loss(col(0), col(1), col(2), ref_logprob=col(3) if with_ref else None, entropy=torch.full((n,), 2.0, device=DEV), weight=torch.ones(n, device=DEV), **o)
    want = torch.tensor([f[4][0] for f in finite], dtype=torch.float64)
    near(sums, want.sum(0), want.abs().sum(0) * lr.EPS * 1.001, "sums together")


def special_case(dtype, V, seed=5):
    """The rows of test_special_rows, for the policy step: (case, score in 64 bits, names)."""
    rows = len(SPECIAL)
    c = make(rows, V, dtype, seed, masked=True)
    x, ids, inv_t, allow = c["x"], c["ids"], c["inv_t"], c["allow"]
    at = {n: i for i, n in enumerate(SPECIAL)}
    allow[:, 0] = True
    ids[ids == 1] = 0
    allow[:, 1] = False
    allow[at["none_allowed"]] = False
    x[at["all_minus_inf"]] = -INF
    x[at["lowest"]] = torch.finfo(dtype).min
    x[at["some_lowest"], ::2] = torch.finfo(dtype).min
    ids[at["id_masked"]] = 1
    ids[at["no_id"]] = -1
    ids[at["id_past_the_row"]] = V
    x[at["nan_masked"], 1] = math.nan
    x[at["inf_masked"], 1] = INF
    x[at["nan"], 0] = math.nan
    x[at["inf"], 0] = INF
    inv_t[at["cold"]] = 1000.0
    inv_t[at["hot"]] = 1e-3
    for n, v in (("t_zero", 0.0), ("t_nan", math.nan), ("t_inf", INF), ("t_negative", -1.0)):
        inv_t[at[n]] = v
    x[at["huge"], 0] = x[at["huge"], 2] = 1e9
    allow[at["huge"], 2] = True
    allow[at["one_allowed"]] = False
    allow[at["one_allowed"], 0] = True
    ids[at["one_allowed"]] = 0
    x[at["id_minus_inf"], ids[at["id_minus_inf"]].long()] = -INF
    ids[at["lowest"]] = ids[at["huge"]] = 0
    if V < 6:  # the lowest number against another: -5e38, which is no float
        ids[at["some_lowest"]] = 0
        inv_t[at["some_lowest"]] = 1.5
        allow[at["some_lowest"], 3] = True
    else:
        ids[at["some_lowest"]] = int(allow[at["some_lowest"], 3::2].nonzero()[0]) * 2 + 3
    r = lr.score(x, ids, inv_t, allow)
    r["lp"] = torch.where(torch.isneginf(r["lp"].float()), torch.full_like(r["lp"], -INF), r["lp"])
    return c, r, at


BAD = ("nan", "inf", "t_zero", "t_nan", "t_inf", "t_negative")  # rows that are NaN


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,spins", [(5, 0), (1000, 0), (40001, 0), (40001, 1)])
@pytest.mark.parametrize("old_kind", ["all -inf", "finite"])
@pytest.mark.parametrize("with_ref", [False, True])
def test_policy_loss_rows_of_special_rows(dtype, V, spins, old_kind, with_ref):
    """The policy step over them, from one part a row and from several, waiting or not: the sums of all rows that are not NaN, and every row's outputs. `finite`: the dead tokens' old
    log-probability is -2, they have the ratio 0 (and an infinite KL term where there is a reference: a call of their own)."""
    m = gc.pkg()
    c, r, at = special_case(dtype, V)
    g = c["g"]
    dead = torch.isneginf(r["lp"]).nonzero()[:, 0].tolist()
    assert set(dead) >= {at[n] for n in ("none_allowed", "all_minus_inf", "id_masked", "id_minus_inf")}
    live = [i for n, i in at.items() if n not in BAD]
    noise = lambda: 0.1 * torch.randn(len(SPECIAL), generator=g)  # noqa: E731
    old = torch.nan_to_num((r["lp"] + noise()).float(), nan=-3.0, neginf=-INF)
    ref = torch.nan_to_num((r["lp"] + noise()).float(), nan=-3.0, neginf=-INF)
    adv = torch.randn(len(SPECIAL), generator=g)
    w = torch.rand(len(SPECIAL), generator=g) + 0.5
    if old_kind == "finite":
        old[dead] = -2.0
    o = dict(clip_low=0.2, clip_high=0.28, dual_clip=3.0, kl_coef=0.05 if with_ref else 0.0, entropy_coef=0.01)
    ratio = (r["lp"] - old.double()).exp()
    assert all(bool(((ratio - b).abs()[live].nan_to_num(1.0) > 1e-4).all()) for b in (0.8, 1.28, 3.0))
    for rows in (live, list(range(len(SPECIAL)))):
        pick = lambda t: t[rows].to(DEV).contiguous()  # noqa: E731
        x = pick(c["x"].to(dtype))
        out = m.policy_loss_rows(x, pick(c["ids"]), pick(old), pick(adv), ref_logprob=pick(ref) if with_ref else None, weight=pick(w), inv_t=pick(c["inv_t"]),
                                 allow=lr.pack_allow(c["allow"][rows]).to(DEV), want_entropy=True, spins=spins, **o)
        own = m.policy_loss_rows(x, pick(c["ids"]), pick(old), pick(adv), ref_logprob=pick(ref) if with_ref else None, weight=pick(w), inv_t=pick(c["inv_t"]),
                                 allow=lr.pack_allow(c["allow"][rows]).to(DEV), want_entropy=True, spins=spins, out=x, **o)
        for a, b in zip(out, own):  # (the new gradient and the logits both begin on a boundary)
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.float().nan_to_num(7.0), b.float().nan_to_num(7.0))
        want, dg, dh = zip(*[policy_by_limits(float(r["lp"][i]), float(old[i]), float(adv[i]), float(ref[i]) if with_ref else None, float(w[i]) if bool(r["has"][i]) else 0.0, float(r["H"][i]), **o)
                             if SPECIAL[i] not in BAD else ([math.nan, math.nan, math.nan if with_ref else 0.0, math.nan, 0.0], 0.0, 0.0) for i in rows])
        want = torch.tensor(want, dtype=torch.float64)
        sums = want.sum(0)
        off, Hoff = lr.lp_tol(r, V)[rows].nan_to_num(0.0), lr.H_tol(r, V)[rows].nan_to_num(0.0)
        size = (ratio * adv.double().abs())[rows].nan_to_num(0.0, posinf=0.0).clamp(max=10.0) + 2.0  # (ratios and KL terms are below e^0.5 here)
        near(out[0], sums, (w[rows].double() * (size * off + Hoff)).sum() + lr.EPS * sums.abs().nan_to_num(0.0, posinf=0.0) + 1e-12 * want.abs().sum().nan_to_num(0.0, posinf=0.0), ("sums", len(rows)))
        has = r["has"][rows]
        near(out[1], torch.where(has, r["lp"][rows], torch.zeros_like(r["lp"][rows])), off, "logprob")
        near(out[2], torch.where(has, r["H"][rows], torch.zeros_like(r["H"][rows])), Hoff, "entropy")
        dg, dh = torch.tensor(dg, dtype=torch.float64), torch.tensor(dh, dtype=torch.float64)
        part = {k: v[rows] for k, v in r.items()}
        d, gsize = lr.grad(part, dg, dh)
        tol = lr.grad_tol(part, gsize, d, V, dtype, h=dh) + part["t"][:, None] * (w[rows].double() * size * (1.01 * off + 4 * lr.EPS))[:, None] * (part["p"] + 1.0 * (torch.arange(V)[None] == part["at"][:, None])) \
            + dh.abs()[:, None] * part["p"] * part["t"][:, None] * Hoff[:, None]
        k = [i for i, row in enumerate(rows) if SPECIAL[row] not in BAD]
        near(out[3][k], d[k], tol[k], "gradient")
        for i, row in enumerate(rows):
            if SPECIAL[row] in BAD:
                assert math.isnan(out[1][i].item()) and bool(torch.isnan(out[3][i].float()).all()), SPECIAL[row]
            if SPECIAL[row] in ("none_allowed", "all_minus_inf", "no_id", "id_past_the_row") or (row in dead and old_kind == "all -inf"):
                assert not out[3][i].any(), SPECIAL[row]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [9, 40001])
def test_infinite_derivatives_leave_masked_places_at_zero(dtype, V):
    """g or h infinite, or so large that t g / S passes the largest float: what is not allowed has the derivative 0 all the same, and nothing is NaN."""
    m = gc.pkg()
    c = make(4, V, dtype, 11, masked=True)
    c["x"][:, 0] = INF  # (in a masked place)
    c["allow"][:, 0] = False
    c["ids"][c["ids"] == 0] = 1
    c["allow"][:, 1] = True
    inv_t = torch.full((4,), 4.0)
    x, ids, allow, inv = c["x"].to(DEV), c["ids"].to(DEV), lr.pack_allow(c["allow"]).to(DEV), inv_t.to(DEV)
    lp, stats, H = m.token_logprobs(x, ids, inv_t=inv, allow=allow, want_entropy=True)
    g = f32(-INF, INF, 3e38, -3e38).to(DEV)
    masked = ~c["allow"]
    for d_entropy in (None, torch.zeros(4, device=DEV)):
        d = m.token_logprobs_grad(x, ids, stats, d_logprob=g, entropy=H, d_entropy=d_entropy, inv_t=inv, allow=allow).cpu().float()
        assert not torch.isnan(d).any() and not d[masked].any()
        own = torch.zeros_like(masked).scatter(1, c["ids"].long()[:, None], True)
        sign = torch.sign(g.cpu())[:, None].expand_as(d)
        assert bool((d * sign <= 0.0)[~own].all()) and bool((d * sign)[own].gt(0.0).all())
    for h in (f32(INF, -INF, 3e38, -3e38), f32(-3e38, INF, 1.0, INF)):
        for by_lp in (None, g):
            d = m.token_logprobs_grad(x, ids, stats, d_logprob=by_lp, entropy=H, d_entropy=h.to(DEV), inv_t=inv, allow=allow).cpu().float()
            assert not torch.isnan(d).any() and not d[masked].any() and bool((d.abs().amax(1) > 0.0).all())
    # a KL term that is infinite: the row's token is masked out, the reference could give it
    ids[0] = 0
    old, ref = torch.full((4,), -2.0, device=DEV), f32(-1.0, 0.0, 0.0, 0.0).to(DEV)
    ref[1:] = lp[1:]
    sums, lp, _, d = m.policy_loss_rows(x, ids, old, torch.ones(4, device=DEV), ref_logprob=ref, inv_t=inv, allow=allow, kl_coef=0.1)
    assert lp[0].item() == -INF and sums[0].item() == INF and sums[2].item() == INF and math.isfinite(sums[1].item())
    d = d.cpu().float()
    assert not torch.isnan(d).any() and not d[masked].any() and bool((d[0][c["allow"][0]] >= 0.0).all()) and bool((d[0] > 1e30).any())


def test_results_do_not_keep_their_workspace():
    """A result's memory is its own entries', and behind them a workspace of 4 KiB at most: a larger one, of megabytes with many rows, goes when the call is made."""
    m = gc.pkg()
    c = make(600, 65537, BF16, 3)
    v = torch.zeros(600, device=DEV)
    off = torch.arange(0, 601, dtype=torch.int32, device=DEV)
    r = m.LossRows(c["dx"].data_ptr(), m.DTYPE_BF16, 600, 65537, 65537)
    assert m.lib().ws_policy_loss_rows_workspace(C.byref(r)) > 100000 and m.lib().ws_token_logprobs_workspace(C.byref(r)) > 10000
    lp, stats, H = m.token_logprobs(c["dx"], c["dids"], want_entropy=True)
    many = torch.zeros(300000, device=DEV)
    results = [lp, stats, H, *m.policy_loss_rows(c["dx"], c["dids"], v, v, want_entropy=True), *m.preference_loss(lp, off), *m.policy_loss(many, many, many)]
    one = m.token_logprobs(c["dx"][:1], c["dids"][:1])
    for t in [*results, *one]:
        if t is not None:
            own = t.numel() * t.element_size()
            assert own <= t.untyped_storage().nbytes() <= own + 4096 + 8 and t.storage_offset() == 0, t.shape


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_between_the_logits_rows(dtype):
    """Logits and gradient in the two halves of one matrix's rows, in either order: they do not overlap. And one row, whose stride is nobody's."""
    m = gc.pkg()
    rows, V = 5, 1003
    for at, to in ((0, V + 3), (V + 3, 0), (0, V)):
        c = make(rows, V, dtype, 17)
        both = torch.full((rows, 2 * V + 6), 5.0, dtype=dtype, device=DEV)
        x, d = both[:, at:at + V], both[:, to:to + V]
        x.copy_(c["x"])
        g = torch.randn(rows, generator=c["g"]).to(DEV)
        lp, stats, _ = m.token_logprobs(x, c["dids"])
        want = m.token_logprobs_grad(x.clone(), c["dids"], stats, d_logprob=g)
        got = m.token_logprobs_grad(x, c["dids"], stats, d_logprob=g, out=d)
        assert got.data_ptr() == d.data_ptr() and torch.equal(got, want) and torch.equal(x.cpu(), c["x"])
        rest = torch.ones(2 * V + 6, dtype=torch.bool)
        rest[at:at + V] = rest[to:to + V] = False
        assert bool((both.cpu()[:, rest] == 5.0).all())
        one = m.policy_loss_rows(x, c["dids"], lp, g, out=d)
        r = lr.score(c["x"], c["ids"])
        want, size = lr.grad(r, -g.cpu().double() / rows, torch.zeros(rows, dtype=torch.float64))
        near(one[3], want, lr.grad_tol(r, size, want, V, dtype, extra=2 * float(lr.lp_tol(r, V).max())), "policy gradient")
    x = c["x"][:1].to(DEV)
    d = m.LossRows(x.data_ptr(), m.DTYPE_F32 if dtype is F32 else m.DTYPE_BF16, 1, V, V, c["dids"].data_ptr())
    want = m.token_logprobs_grad(x, c["dids"][:1], stats[:1], d_logprob=g[:1])
    m.check(m.lib().ws_token_logprobs_grad(torch.cuda.current_stream().cuda_stream, C.byref(d), stats.data_ptr(), g.data_ptr(), None, None, x.data_ptr(), V + 9), "ws_token_logprobs_grad")
    assert torch.equal(x, want)


def test_pairs_and_looks_past_32_bits_are_refused():
    m = gc.pkg()
    x, ids, v = torch.zeros((2, 9), device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV)
    for spins in (-1, 65537, 1 << 32, (1 << 32) + 1):
        with pytest.raises(m.WsError):
            m.policy_loss_rows(x, ids, v, v, spins=spins)
    with pytest.raises(m.WsError, match="at most"):
        m.preference_loss(v, torch.empty((1 << 33) + 1, dtype=torch.int8, device="meta"))


def test_a_gradient_written_over_a_tensor_is_seen_by_autograd():
    """`out` is overwritten: what autograd keeps of it is no longer what it was, and a backward pass that needs it has to say so. The gradient itself is carried on with logits.backward."""
    m = gc.pkg()
    c = make(4, 300, F32, 29)
    v = torch.zeros(4, device=DEV)
    lp, stats, _ = m.token_logprobs(c["dx"], c["dids"])
    calls = (lambda x, out: m.token_logprobs_grad(x, c["dids"], stats, d_logprob=v + 1.0, out=out), lambda x, out: m.policy_loss_rows(x, c["dids"], lp, v + 1.0, out=out)[3])
    for call in calls:
        hidden = c["dx"].clone().requires_grad_()
        logits = 30.0 * torch.tanh(hidden / 30.0)
        d = call(logits, None)
        assert not d.requires_grad
        (want,) = torch.autograd.grad(logits, hidden, d)
        assert bool(want.any())
        logits = 30.0 * torch.tanh(hidden / 30.0)  # (keeps the tangent, which is another tensor: over these logits it can be written)
        d = call(logits, logits)
        (got,) = torch.autograd.grad(logits, hidden, d.clone())
        assert torch.equal(got, want)
        logits = torch.tanh(hidden)  # (keeps these)
        version = logits._version
        d = call(logits, logits)
        assert logits._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(logits, hidden, d.clone())
        with torch.inference_mode():
            x = c["dx"].clone()
            call(x, x)


@pytest.mark.parametrize("rows,V", [(3, 50257), (300, 50257), (5, 777), (2, 151936)])
def test_entropy_gradient_of_nearly_even_rows(rows, V):
    """Where a row is nearly even ln p + H is small beside ln p and H: H - ln S is taken before either is rounded. An entry is h t p (d - mean d) with exponents d of a thousandth: the difference
    x - m, the product with the split factor and the power round by EPS |d| and one step, the mean's sums by sum_tol's steps; one more rounding each of factors and result."""
    m = gc.pkg()
    g = torch.Generator().manual_seed(V)
    ids, none, h = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows, device=DEV), -1.0
    for sigma in (0.0, 1e-3):
        x = 3.0 + sigma * torch.randn((rows, V), generator=g)
        r = lr.score(x, ids.cpu())
        _, _, _, d = m.policy_loss_rows(x.to(DEV), ids, none, none, weight=none + 1.0, entropy_coef=1.0)
        want, _ = lr.grad(r, torch.zeros(rows, dtype=torch.float64), torch.full((rows,), h, dtype=torch.float64))
        mean = (r["p"] * r["a"].abs()).sum(1, keepdim=True)
        near(d, want, r["p"] * (r["a"].abs() + mean) * lr.EPS * (2.0 * 42.0) + 2.0 ** -126, ("gradient", sigma))
        if sigma == 0.0:
            assert not d.any()


@pytest.mark.parametrize("V", [5, 1000, 40001])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_everything_of_a_row_that_is_nan(dtype, V):
    """Its maximum in `stats` too; a row without a token keeps its logprob of 0."""
    m = gc.pkg()
    c, r, at = special_case(dtype, V)
    c["ids"][at["t_nan"]] = -1
    lp, stats, H = m.token_logprobs(c["x"].to(DEV), c["ids"].to(DEV), inv_t=c["inv_t"].to(DEV), allow=lr.pack_allow(c["allow"]).to(DEV), want_entropy=True)
    for n in BAD:
        assert bool(torch.isnan(stats[at[n]]).all()) and math.isnan(H[at[n]].item()), n
        assert lp[at[n]].item() == 0.0 if n == "t_nan" else math.isnan(lp[at[n]].item()), n
    ok = [i for n, i in at.items() if n not in BAD]
    assert torch.equal(stats[ok, 0].cpu().double(), r["m"][ok])


@pytest.mark.parametrize("rows,V", [(1, 1048575), (2, 1048573), (3, 786409), (2, 262144), (40, 151937), (700, 20485), (3, 4099), (9, 33), (2100, 261)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
def test_even_rows_count_every_logit_once(rows, V, dtype, masked):
    """Every power is 1 and every partial sum a whole number: S is the number of allowed tokens, to the bit, and a logit lost or taken twice shows whatever the row's length. ln S in 64 bits, rounded
    once. The gradient's entries are all the same: -g / S, two roundings of factors and, of bf16, the result's."""
    m = gc.pkg()
    g = torch.Generator().manual_seed(rows + V)
    stride, shift = 3, 1
    mem = torch.full((rows * (V + stride) + shift,), 50.0, dtype=dtype, device=DEV)
    x = mem[shift:].view(rows, V + stride)[:, :V]
    x.fill_(-1.5)
    ids = torch.randint(V, (rows,), generator=g, dtype=torch.int32)
    allow = torch.rand((rows, V), generator=g) < 0.4 if masked else torch.ones((rows, V), dtype=torch.bool)
    allow[torch.arange(rows), ids.long()] = True
    S = allow.sum(1).double()
    words = lr.pack_allow(allow).to(DEV) if masked else None
    dids, inv_t = ids.to(DEV), torch.full((rows,), 0.7, device=DEV)
    adv = torch.ones(rows, device=DEV)
    for entropy in (False, True):
        lp, stats, H = m.token_logprobs(x, dids, inv_t=inv_t, allow=words, want_entropy=entropy)
        assert torch.equal(stats[:, 1].cpu().double(), S) and bool((stats[:, 0] == -1.5).all())
        tol = lr.EPS * 1.001 * S.log() + 1e-12
        near(lp, -S.log(), tol, "logprob")
        if entropy:
            near(H, S.log(), tol, "entropy")
        for spins in (0, 1):
            _, lp, H, d = m.policy_loss_rows(x, dids, (-S.log()).float().to(DEV), adv, weight=adv, inv_t=inv_t, allow=words, want_entropy=entropy, spins=spins)
            near(lp, -S.log(), tol, "logprob of the step")
            if entropy:
                near(H, S.log(), tol, "entropy of the step")
            # (the ratio is e^(rounding of the old log-probability): 1 within EPS ln S)
            want = torch.where(allow, (0.7 / S)[:, None], torch.zeros(1, dtype=torch.float64))
            want[torch.arange(rows), ids.long()] -= 0.7
            rel = lr.EPS * (S.log()[:, None] + 6.0) + torch.finfo(dtype).eps / 2
            near(d, want, 1.001 * rel * (want.abs() + (0.7 / S)[:, None] * allow) + 2.0 ** -126, "gradient")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [5, 1000, 40001])
def test_the_three_calls_of_a_policy_step_on_special_rows(dtype, V):
    """Scores, loss and gradient one after the other, rows without a token weighing 0 in the loss: what the policy step does at once (ws_policy_loss sees a log-probability of 0 there, and would count it)."""
    m = gc.pkg()
    c, r, at = special_case(dtype, V)
    rows = [i for n, i in at.items() if n not in BAD]
    pick = lambda t: t[rows].to(DEV).contiguous()  # noqa: E731
    x, ids, inv_t, allow = pick(c["x"]), pick(c["ids"]), pick(c["inv_t"]), lr.pack_allow(c["allow"][rows]).to(DEV)
    old = torch.nan_to_num((r["lp"] + 0.1).float(), neginf=-INF)[rows].to(DEV)
    adv, w = torch.linspace(-1, 1, len(rows), device=DEV), torch.ones(len(rows), device=DEV)
    o = dict(kl_coef=0.05, entropy_coef=0.01)
    want = m.policy_loss_rows(x, ids, old, adv, ref_logprob=old, weight=w, inv_t=inv_t, allow=allow, **o)
    lp, stats, H = m.token_logprobs(x, ids, inv_t=inv_t, allow=allow, want_entropy=True)
    has = (ids >= 0) & (ids < V)
    sums, g, h = m.policy_loss(lp, old, adv, ref_logprob=old, entropy=H, weight=torch.where(has, w, 0.0 * w), **o)
    d = m.token_logprobs_grad(x, ids, stats, d_logprob=g, entropy=H, d_entropy=h, inv_t=inv_t, allow=allow)
    # log-probabilities and entropies are rounded between the calls: EPS of their size, and of ratios as much; both sides are off by lp_tol and H_tol
    off = (2 * lr.lp_tol(r, V) + 2 * lr.H_tol(r, V))[rows].nan_to_num(0.0)
    near(sums, want[0].cpu(), 3.0 * off.sum() + 4 * lr.EPS * float(want[0].abs().sum()), "sums")
    assert torch.equal(torch.isneginf(lp), torch.isneginf(want[1])) and not torch.isnan(d).any() and bool(torch.isfinite(sums).all())
    near(torch.where(has, lp, 0.0 * lp).nan_to_num(neginf=-1e30), want[1].cpu().nan_to_num(neginf=-1e30), off, "logprob")
    near(d, want[3].cpu().float(), (3.0 * off + 40 * lr.EPS)[:, None] * r["t"][rows][:, None] + 2.0 * torch.finfo(dtype).eps * want[3].cpu().double().abs(), "gradient")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
def test_very_small_inverse_temperatures(dtype, masked):
    """1 / temperature down to the smallest float, with logits as large as it takes to matter (differences that a float holds): the second float of the factor may not be larger than it is. Below
    2^-126 floats lie 2^-149 apart: a factor c is off by 2^-149 / c then, and exponents by that much of their size."""
    m = gc.pkg()
    rows, V = 6, 3001
    c = make(rows, V, dtype, 83, masked)
    inv_t = f32(1e-30, 1e-34, 1e-36, 1e-37, 1.2e-38, 3e-40)
    x = (torch.rand((rows, V), generator=c["g"]) * 4.0 / inv_t.double()[:, None].clamp(min=2.5e-38)).to(dtype)
    if masked:
        x[:, 7] = -INF
    r = lr.score(x, c["ids"], inv_t, c["allow"])
    assert float((r["a"].abs().amax(1)).min()) > 0.01
    dx, ids, inv, allow = x.to(DEV), c["dids"], inv_t.to(DEV), c["dallow"]
    lp, stats, H = m.token_logprobs(dx, ids, inv_t=inv, allow=allow, want_entropy=True)
    extra = (2.0 ** -149 / inv_t.double()) * (r["p"] * r["a"].abs()).sum(1) * 2.0
    near(stats[:, 1], r["S"], r["S"] * (lr.sum_tol(r, V) + extra), "sum")
    near(lp, r["lp"], lr.lp_tol(r, V) + extra, "logprob")
    near(H, r["H"], lr.H_tol(r, V) + 4.0 * extra, "entropy")
    # (times t the gradient would leave the floats: g makes up for it)
    g = (1.0 / inv_t.double()).clamp(max=1e37).float()
    for d in (m.token_logprobs_grad(dx, ids, stats, d_logprob=g.to(DEV), inv_t=inv, allow=allow), ):
        want, size = lr.grad(r, g.double(), torch.zeros(rows, dtype=torch.float64))
        near(d, want, lr.grad_tol(r, size, want, V, dtype) + size * (2.0 ** -148 / inv_t.double())[:, None] * (1.0 + r["a"].abs()), "gradient")


def share_tol(r):
    """lr.sum_tol for rows that workgroups share: a share is 15 vectors of 8 logits a thread at most (scores with entropy: 1.5 x 2560 vectors over 256 threads; the policy step: 12), and one of the
    row's ends, 121 terms however long the row."""
    return lr.EPS * (2.0 * (r["p"] * r["a"].abs()).sum(1) + 2.0 + 121.0 + 40.0)


@pytest.mark.parametrize("rows,V", [(2, 1048575), (3, 786409), (9, 262144), (70, 151937)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_rows_within_what_a_share_rounds(rows, V, dtype):
    m = gc.pkg()
    c = make(rows, V, dtype, 97 + rows, False, 3, 1, sigma=0.5)
    r = lr.score(c["x"], c["ids"], c["inv_t"])
    tol = share_tol(r)
    mean, square = (r["p"] * r["a"].abs()).sum(1), (r["p"] * r["a"] ** 2).sum(1)
    Htol = tol * (1.0 + 2.0 * mean) + lr.EPS * (2.0 * square + r["H"].abs() + 4.0 * mean)
    old, adv = torch.full((rows,), -12.0, device=DEV), torch.zeros(rows, device=DEV)
    for entropy in (False, True):
        lp, stats, H = m.token_logprobs(c["dx"], c["dids"], inv_t=c["dinv"], want_entropy=entropy)
        near(stats[:, 1], r["S"], r["S"] * tol, "sum")
        _, lp2, H2, _ = m.policy_loss_rows(c["dx"], c["dids"], old, adv, inv_t=c["dinv"], want_entropy=entropy, entropy_coef=0.01 if entropy else 0.0)
        for what, got in (("scores", lp), ("step", lp2)):
            near(got, r["lp"], tol + lr.EPS * r["lp"].abs(), what)
        for what, got in (("scores", H), ("step", H2)):
            if entropy:
                near(got, r["H"], Htol, what)
