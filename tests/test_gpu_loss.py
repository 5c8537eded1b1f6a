"""GPU: log-probabilities of given tokens, the policy and preference losses and their gradients (ws_token_logprobs, ws_token_logprobs_grad,
ws_policy_loss, ws_policy_loss_rows, ws_preference_loss) against their formulas in 64 bits (loss_ref.py, where the tolerances are derived)."""
import math

import pytest
import torch

import gpu_cases as gc
import loss_ref as lr

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def make(rows, V, dtype, seed, masked=False, stride=0, shift=0, sigma=2.0):
    """Host tensors of a case and the device's: logits in a matrix whose rows are V + stride apart and which begins `shift` elements into its memory."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, V), generator=g) * sigma)
    x.scatter_add_(1, torch.randint(V, (rows, 1), generator=g), 14.0 * torch.rand((rows, 1), generator=g))
    x = x.to(dtype)
    ids = torch.randint(V, (rows,), generator=g, dtype=torch.int32)
    inv_t = 1.0 / (0.5 + torch.rand(rows, generator=g))
    allow = None
    if masked:
        allow = torch.rand((rows, V), generator=g) < 0.3
        allow[torch.arange(rows), ids.long()] = True
    mem = torch.full((rows * (V + stride) + shift + 64,), math.nan, dtype=dtype, device=DEV)
    dx = mem[shift:shift + rows * (V + stride)].view(rows, V + stride)[:, :V]
    dx.copy_(x)
    return dict(x=x, ids=ids, inv_t=inv_t, allow=allow, dx=dx, dids=ids.to(DEV), dinv=inv_t.to(DEV), dallow=lr.pack_allow(allow).to(DEV) if masked else None,
                rows=rows, V=V, dtype=dtype, g=g)


def near(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    # (what a float32 cannot hold is an infinity in it: a token at the lowest number, at t > 1, has a log-probability of -3.98e38 where -3.40e38 is the last)
    want = torch.where(want.abs() > torch.finfo(F32).max, torch.sign(want) * math.inf, want)
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    same = (torch.isnan(got) & torch.isnan(want)) | (got == want)
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        i = bad.nonzero()[0].tolist()
        raise AssertionError((what, i, float(got[tuple(i)]), float(want[tuple(i)]), float(tol[tuple(i)]), int(bad.sum()), bad.numel()))


SHAPES = [(1, 1), (3, 2), (2, 7), (5, 31), (4, 33), (6, 129), (9, 1000), (3, 4099), (300, 777), (2, 20481), (3, 50257), (260, 8200), (1, 151936), (2, 262144), (2, 65543), (2, 1048575), (70001, 9)]  # (more rows than a grid has in its second dimension)


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
def test_logprobs(rows, V, dtype, masked):
    m = gc.pkg()
    for stride, shift in ((0, 0), (3, 1)):
        c = make(rows, V, dtype, 7 * rows + V, masked, stride, shift)
        r = lr.score(c["x"], c["ids"], c["inv_t"], c["allow"])
        for want_entropy in (False, True):
            lp, stats, H = m.token_logprobs(c["dx"], c["dids"], inv_t=c["dinv"], allow=c["dallow"], want_entropy=want_entropy)
            near(lp, r["lp"], lr.lp_tol(r, V), "logprob")
            assert torch.equal(stats[:, 0].cpu().double(), r["m"])
            near(stats[:, 1], r["S"], r["S"] * lr.sum_tol(r, V), "sum")
            if want_entropy:
                near(H, r["H"], lr.H_tol(r, V), "entropy")
            again = m.token_logprobs(c["dx"], c["dids"], inv_t=c["dinv"], allow=c["dallow"], want_entropy=want_entropy)
            assert torch.equal(lp, again[0]) and torch.equal(stats, again[1])


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
def test_gradient(rows, V, dtype, masked):
    m = gc.pkg()
    for stride, shift in ((0, 0), (3, 1)):
        c = make(rows, V, dtype, 11 * rows + V, masked, stride, shift)
        r = lr.score(c["x"], c["ids"], c["inv_t"], c["allow"])
        g, h = torch.randn(rows, generator=c["g"]), 0.1 * torch.randn(rows, generator=c["g"])
        stats, H = torch.stack([r["m"], r["S"]], 1).float().to(DEV), r["H"].float().to(DEV)
        for with_h in (False, True):
            want, size = lr.grad(r, g.double(), h.double() if with_h else torch.zeros(rows, dtype=torch.float64))
            mem = torch.full((rows, V + 5), 77.0, dtype=dtype, device=DEV)
            out = m.token_logprobs_grad(c["dx"], c["dids"], stats, d_logprob=g.to(DEV), entropy=H if with_h else None, d_entropy=h.to(DEV) if with_h else None,
                                        inv_t=c["dinv"], allow=c["dallow"], out=mem[:, :V])
            near(out, want, lr.grad_tol(r, size, want, V, dtype, h=h if with_h else None), "gradient")
            assert bool((mem[:, V:] == 77.0).all()), "written beyond the row"
        own = m.token_logprobs_grad(c["dx"], c["dids"], stats, d_logprob=g.to(DEV), entropy=H, d_entropy=h.to(DEV), inv_t=c["dinv"], allow=c["dallow"], out=c["dx"])
        assert own.data_ptr() == c["dx"].data_ptr()  # (in place)
        near(own, want, lr.grad_tol(r, size, want, V, dtype, h=h), "gradient in place")


SPECIAL = ["none_allowed", "all_minus_inf", "lowest", "some_lowest", "id_masked", "no_id", "id_past_the_row", "nan_masked", "inf_masked", "nan", "inf", "cold", "hot", "t_zero",
           "t_nan", "t_inf", "t_negative", "huge", "one_allowed", "id_minus_inf"]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [5, 1000, 40001])
def test_special_rows(dtype, V):
    m = gc.pkg()
    rows = len(SPECIAL)
    c = make(rows, V, dtype, 5, masked=True)
    x, ids, inv_t, allow = c["x"], c["ids"], c["inv_t"], c["allow"]
    at = {n: i for i, n in enumerate(SPECIAL)}
    allow[:, 0] = True
    ids[ids == 1] = 0
    allow[:, 1] = False
    allow[at["none_allowed"]] = False
    x[at["all_minus_inf"]] = -math.inf
    x[at["lowest"]] = torch.finfo(dtype).min
    x[at["some_lowest"], ::2] = torch.finfo(dtype).min
    ids[at["id_masked"]] = 1
    ids[at["no_id"]] = -1
    ids[at["id_past_the_row"]] = V
    x[at["nan_masked"], 1] = math.nan
    x[at["inf_masked"], 1] = math.inf
    x[at["nan"], 0] = math.nan
    x[at["inf"], 0] = math.inf
    inv_t[at["cold"]] = 1000.0
    inv_t[at["hot"]] = 1e-3
    for n, v in (("t_zero", 0.0), ("t_nan", math.nan), ("t_inf", math.inf), ("t_negative", -1.0)):
        inv_t[at[n]] = v
    x[at["huge"], 0] = 1e9
    x[at["huge"], 2] = 1e9
    allow[at["huge"], 2] = True
    allow[at["one_allowed"]] = False
    allow[at["one_allowed"], 0] = True
    ids[at["one_allowed"]] = 0
    x[at["id_minus_inf"], ids[at["id_minus_inf"]].long()] = -math.inf
    c["dx"].copy_(x)
    d = dict(inv_t=inv_t.to(DEV), allow=lr.pack_allow(allow).to(DEV))
    r = lr.score(x, ids, inv_t, allow)
    lp, stats, H = m.token_logprobs(c["dx"], ids.to(DEV), want_entropy=True, **d)
    near(lp, r["lp"], torch.nan_to_num(lr.lp_tol(r, V)), "logprob")
    near(H, r["H"], torch.nan_to_num(lr.H_tol(r, V)), "entropy")
    ok = [i for n, i in at.items() if n not in ("nan", "inf", "t_zero", "t_nan", "t_inf", "t_negative")]
    assert torch.equal(stats[ok, 0].cpu().double(), r["m"][ok])
    near(stats[ok, 1], r["S"][ok], (r["S"] * lr.sum_tol(r, V))[ok], "sum")
    g, h = torch.randn(rows, generator=c["g"]), torch.full((rows,), 0.01)
    want, size = lr.grad(r, g.double(), h.double())
    out = m.token_logprobs_grad(c["dx"], ids.to(DEV), stats, d_logprob=g.to(DEV), entropy=H, d_entropy=h.to(DEV), **d)
    near(out[ok], want[ok], lr.grad_tol(r, size, want, V, dtype)[ok], "gradient")
    bad = [i for i in range(rows) if i not in ok]
    keep = allow[bad] & ~torch.isneginf(x[bad])
    assert bool(torch.isnan(out[bad].cpu().float())[keep].all())
    for n in ("none_allowed", "all_minus_inf"):
        assert stats[at[n]].tolist() == [-math.inf, 0.0] and H[at[n]].item() == 0.0 and lp[at[n]].item() == -math.inf and not out[at[n]].any()


def test_gradient_of_rows_without_derivatives_is_zero_and_they_are_not_read():
    m = gc.pkg()
    for dtype in (F32, BF16):
        c = make(6, 5003, dtype, 3)
        c["dx"][1::2] = math.nan
        ids = c["dids"].clone()
        ids[3] = -1
        g = torch.ones(6, device=DEV)
        g[1] = g[5] = 0.0
        stats = torch.tensor([[1.0, 2.0]] * 6, device=DEV)
        out = m.token_logprobs_grad(c["dx"], ids, stats, d_logprob=g)
        assert not out[1::2].any() and bool(torch.isfinite(out[::2].float()).all()) and bool(out[::2].any())


def test_gradient_against_differences():
    """Central differences of the kernel's own log-probability and entropy by every logit of a row. A step of 2^-6: the third derivatives of both are below 8 in
    size at t = 1.25 (t^3 times 1 + the exponents' size), so the difference quotient is off by 8 / 6 * 2^-12 = 3.3e-4 at most, and by the outputs'
    error over the step, 2 * 4e-6 * 2^6 / 2 = 2.6e-4."""
    m = gc.pkg()
    V, step = 37, 2.0 ** -6
    c = make(1, V, F32, 19, sigma=1.0)
    inv_t = torch.tensor([1.25], device=DEV)
    x = c["dx"][0].clone()
    many = x.repeat(2 * V, 1)
    for v in range(V):
        many[2 * v, v] += step
        many[2 * v + 1, v] -= step
    lp, _, H = m.token_logprobs(many, c["dids"].repeat(2 * V), inv_t=inv_t.repeat(2 * V), want_entropy=True)
    _, stats, H0 = m.token_logprobs(x[None], c["dids"], inv_t=inv_t, want_entropy=True)
    one = torch.ones(1, device=DEV)
    by_lp = m.token_logprobs_grad(x[None], c["dids"], stats, d_logprob=one, inv_t=inv_t)[0]
    by_H = m.token_logprobs_grad(x[None], c["dids"], stats, entropy=H0, d_entropy=one, inv_t=inv_t)[0]
    for f, d in ((lp, by_lp), (H, by_H)):
        quotient = (f[0::2] - f[1::2]).double() / (2 * step)
        assert float((quotient - d.double()).abs().max()) < 6e-4


def tokens(n, seed, with_ref=True, with_weight=True):
    g = torch.Generator().manual_seed(seed)
    lp = -3.0 * torch.rand(n, generator=g)
    t = dict(lp=lp, old=lp + 0.3 * torch.randn(n, generator=g), adv=torch.randn(n, generator=g), ref=lp + 0.3 * torch.randn(n, generator=g) if with_ref else None,
             H=5.0 * torch.rand(n, generator=g), w=None)
    if with_weight:
        t["w"] = torch.rand(n, generator=g) / n
        t["w"][torch.rand(n, generator=g) < 0.2] = 0.0
    return t


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 511, 512, 513, 1024, 1025, 5000, 32768, 70001, 300000])
@pytest.mark.parametrize("kind", ["plain", "all"])
def test_policy_loss(n, kind):
    """Everything in 64 bits and rounded once: half a step each."""
    m = gc.pkg()
    every = kind == "all"
    t = tokens(n, n, every, every)
    if every and n > 4:  # far off the old policy, and tokens of weight 0 with anything in them
        t["old"][:2] = torch.tensor([-60.0, 60.0])
        t["adv"][0] = -1.0
        t["w"][3] = 0.0
        t["lp"][3], t["old"][3], t["adv"][3], t["ref"][3], t["H"][3] = math.nan, math.inf, math.nan, -math.inf, math.nan
    o = dict(clip_low=0.2, clip_high=0.28, dual_clip=3.0, kl_coef=0.05, entropy_coef=0.01) if every else {}
    sums, g, h, size = lr.policy(t["lp"], t["old"], t["adv"], t["ref"], t["w"], t["H"] if every else None, **o)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    for _ in range(2):
        got = m.policy_loss(d["lp"], d["old"], d["adv"], ref_logprob=d["ref"], entropy=d["H"] if every else None, weight=d["w"], **o)
        near(got[0], sums, lr.EPS * sums.abs() + 1e-12 * size, "sums")
        near(got[1], g, lr.EPS * g.abs() * 1.001 + 2.0 ** -149, "d_logprob")
        if every:
            near(got[2], h, lr.EPS * h.abs() * 1.001 + 2.0 ** -149, "d_entropy")
        else:
            assert got[2] is None


def test_policy_loss_of_no_tokens():
    m = gc.pkg()
    none = torch.empty(0, device=DEV)
    sums, g, h = m.policy_loss(none, none, none, entropy=none)
    assert sums.tolist() == [0.0] * 5 and g.numel() == 0 and h.numel() == 0
    logits = torch.empty((0, 100), device=DEV)
    sums, lp, H, d = m.policy_loss_rows(logits, torch.empty(0, dtype=torch.int32, device=DEV), none, none)
    assert sums.tolist() == [0.0] * 5 and lp.numel() == 0 and d.shape == (0, 100)
    lp, stats, H = m.token_logprobs(logits, torch.empty(0, dtype=torch.int32, device=DEV), want_entropy=True)
    assert lp.numel() == 0 and stats.shape == (0, 2) and H.numel() == 0
    assert m.token_logprobs_grad(logits, torch.empty(0, dtype=torch.int32, device=DEV), stats).shape == (0, 100)


# rows of one workgroup and of several, of all builds (shares of up to 256 vectors, of 4 and of 12 times as many); sums over up to 64 and 1024 rows, of rows of three parts up to 4096, over more in a second launch
ROWS = [(600, 777), (520, 12400), (513, 25001), (1030, 1100), (4096, 261), (4097, 300), (1, 1), (1, 129), (7, 1000), (16, 50257), (3, 151936), (5, 262144), (130, 3), (140, 1001), (130, 20480), (129, 20485), (128, 40961), (130, 50257), (128, 81921), (128, 151936),
        (128, 160007)]


POLICY_CASES = [(rows, V, dtype, kind) for rows, V in ROWS for dtype in (F32, BF16) for kind in ("plain", "entropy", "bonus", "masked")] + [(4100, 12500, F32, "bonus"), (1027, 24700, F32, "masked")] \
    + [(5, 1048575, dtype, kind) for dtype in (F32, BF16) for kind in ("plain", "entropy", "bonus", "masked")] + [(2, V, F32, "masked") for V in (786407, 786409)] \
    + [(32772, 9, F32, "bonus"), (32769, 17, BF16, "masked")]  # the longest, 64 full shares, more rows than a grid has in its second dimension


@pytest.mark.parametrize("rows,V,dtype,kind", POLICY_CASES)
def test_policy_loss_rows(rows, V, dtype, kind):
    m = gc.pkg()
    c = make(rows, V, dtype, 13 * rows + V, kind == "masked", 0 if kind == "plain" else 3, 0 if kind == "plain" else 1)
    r = lr.score(c["x"], c["ids"], c["inv_t"], c["allow"])
    g = c["g"]
    old, ref, adv = (r["lp"] + 0.3 * torch.randn(rows, generator=g)).float(), (r["lp"] + 0.3 * torch.randn(rows, generator=g)).float(), torch.randn(rows, generator=g)
    w = None if kind == "plain" else torch.rand(rows, generator=g) / rows
    o = dict(clip_low=0.2, clip_high=0.28, dual_clip=3.0, kl_coef=0.05, entropy_coef=0.01 if kind in ("bonus", "masked") else 0.0)
    want_entropy = kind != "plain"
    ratio = (r["lp"] - old.double()).exp()
    for border in (0.8, 1.28, 3.0):  # no token stands where an error in its log-probability could move it over
        assert bool(((ratio - border).abs() > 1.5 * border * lr.lp_tol(r, V)).all())
    ids = c["dids"].clone()
    counts = torch.ones(rows, dtype=torch.bool)
    if w is not None and rows > 4:  # rows that count for nothing, whatever they hold
        w[1] = 0.0
        ids[2] = -1
        counts[1] = counts[2] = False
        c["dx"][1:3] = math.nan
    live_w = torch.full((rows,), 1.0 / rows) if w is None else torch.where(counts, w, torch.zeros_like(w))
    sums, dg, dh, size = lr.policy(r["lp"], old, adv, ref, live_w, r["H"] if want_entropy else None, **o)
    want, gsize = lr.grad(r, dg, dh)
    # an error in the log-probability goes into the ratio and the KL term, relative to their size
    off = lr.lp_tol(r, V)
    gtol = live_w.double() * (ratio * adv.double().abs() + o["kl_coef"] * (ref.double() - r["lp"]).exp()) * (1.01 * off + 4 * lr.EPS)
    tol = lr.grad_tol(r, gsize, want, V, dtype) + r["t"][:, None] * gtol[:, None] * (r["p"] + 1.0 * (torch.arange(V)[None] == r["at"][:, None]))
    Htol = lr.H_tol(r, V)
    tol = tol + dh.abs()[:, None] * r["p"] * r["t"][:, None] * Htol[:, None]
    args = dict(ref_logprob=ref.to(DEV), weight=None if w is None else w.to(DEV), inv_t=c["dinv"], allow=c["dallow"], want_entropy=want_entropy, **o)
    stol = (live_w.double() * (ratio * adv.double().abs() + o["kl_coef"] * (ref.double() - r["lp"]).exp().clamp(min=1.0)) * off).sum() + (live_w.double() * Htol).sum() + lr.EPS * sums.abs() + 1e-12 * size
    klt = (live_w.double() * ((ref.double() - r["lp"]).exp() + 1) * off).sum()
    for where in ("own", "in place"):
        got = m.policy_loss_rows(c["dx"], ids, old.to(DEV), adv.to(DEV), out=c["dx"] if where == "in place" else None, **args)
        near(got[0], sums, stol + klt, "sums")
        near(got[1], torch.where(counts, r["lp"], torch.zeros_like(r["lp"])), off, "logprob")
        if want_entropy:
            near(got[2], torch.where(counts, r["H"], torch.zeros_like(r["H"])), Htol, "entropy")
        else:
            assert got[2] is None
        near(got[3], want, tol, "gradient " + where)


def test_policy_loss_rows_is_what_its_parts_give():
    """One call against the three it stands for, and the same bits twice."""
    m = gc.pkg()
    for rows in (20, 200):
        c = make(rows, 12345, F32, 23)
        old = torch.full((rows,), -7.0, device=DEV)
        adv = torch.linspace(-1, 1, rows, device=DEV)
        o = dict(kl_coef=0.1, entropy_coef=0.02)
        one = m.policy_loss_rows(c["dx"], c["dids"], old, adv, ref_logprob=old, inv_t=c["dinv"], **o)
        two = m.policy_loss_rows(c["dx"], c["dids"], old, adv, ref_logprob=old, inv_t=c["dinv"], **o)
        assert all(torch.equal(a, b) for a, b in zip(one, two))
        lp, stats, H = m.token_logprobs(c["dx"], c["dids"], inv_t=c["dinv"], want_entropy=True)
        sums, g, h = m.policy_loss(lp, old, adv, ref_logprob=old, entropy=H, **o)
        d = m.token_logprobs_grad(c["dx"], c["dids"], stats, d_logprob=g, entropy=H, d_entropy=h, inv_t=c["dinv"])
        for a, b in zip(one, (sums, lp, H, d)):
            assert float((a - b).abs().max()) <= 2e-5 * max(1e-6, float(b.abs().max()))


@pytest.mark.parametrize("lengths", [[1, 1], [0, 3], [0, 0], [5, 0, 7, 1000], [513, 2, 1025, 4097, 3, 1], "65", "300"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_loss(lengths, smoothing):
    """The sums over an answer in 64 bits, all outputs rounded once; 1e-12 for the order of the sums."""
    m = gc.pkg()
    g = torch.Generator().manual_seed(31)
    if isinstance(lengths, str):
        lengths = torch.randint(0, 40, (2 * int(lengths),), generator=g).tolist()
    for before, behind, extra in ((0, 0, False), (3, 700, True)):
        off = [before]
        for n in lengths:
            off.append(off[-1] + n)
        rows, P = off[-1] + behind, len(lengths) // 2
        lp = -5.0 * torch.rand(rows, generator=g)
        ref = lp + torch.randn(rows, generator=g) if extra else None
        w = torch.rand(P, generator=g) if extra else None
        if extra and P > 1:
            w[0] = 0.0
        beta = 0.1 if extra else 5.0  # (with 5 and no reference the losses go to both ends)
        loss, each, reward, d = lr.preference(lp, off, ref, w, beta, smoothing)
        for _ in range(2):
            got = m.preference_loss(lp.to(DEV), torch.tensor(off, dtype=torch.int32, device=DEV), ref_logprob=None if ref is None else ref.to(DEV),
                                    weight=None if w is None else w.to(DEV), beta=beta, label_smoothing=smoothing)
            scale = 1e-10 * (1.0 + each.abs())
            near(got[0], loss.reshape(1), lr.EPS * loss.abs() + scale.sum(), "loss")
            near(got[1], each, lr.EPS * each.abs() + scale, "pair_loss")
            near(got[2], reward, lr.EPS * reward.abs() + 1e-10, "reward")
            near(got[3], d, lr.EPS * d.abs() * 1.001 + 1e-10 * d.abs() + 2.0 ** -149, "d_logprob")


def test_preference_offsets_past_the_rows_end_there():
    m = gc.pkg()
    lp = -torch.rand(10, device=DEV)
    a = m.preference_loss(lp, torch.tensor([0, 4, 10], dtype=torch.int32, device=DEV))
    b = m.preference_loss(lp, torch.tensor([0, 4, 1 << 20], dtype=torch.int32, device=DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_drawn_answers_scored_and_trained_on():
    """The operators as they are used: tokens drawn by the batched sampler under a temperature and a mask, scored with both, a policy step on them at once (the
    ratio is 1: the gradient is that of the plain policy gradient), and pairs of the same answers through the preference loss."""
    m = gc.pkg()
    rows, V = 24, 32771
    c = make(rows, V, F32, 41, masked=True)
    seed, step = torch.arange(rows, dtype=torch.int64, device=DEV), torch.zeros(rows, dtype=torch.int64, device=DEV)
    smp = m.BatchSampler(c["dx"], c["dinv"], seed, step, allow=c["dallow"]).run()
    ids = smp.token.cpu()
    assert bool(c["allow"][torch.arange(rows), ids.long()].all())
    r = lr.score(c["x"], ids, c["inv_t"], c["allow"])
    lp, stats, H = m.token_logprobs(c["dx"], smp.token, inv_t=c["dinv"], allow=c["dallow"], want_entropy=True)
    near(lp, r["lp"], lr.lp_tol(r, V), "logprob")
    near(smp.prob, r["lp"].exp(), 4e-6 * r["lp"].exp(), "the sampler's probability of an open row")
    adv = torch.randn(rows, generator=c["g"])
    sums, lp2, _, d = m.policy_loss_rows(c["dx"], smp.token, lp, adv.to(DEV), inv_t=c["dinv"], allow=c["dallow"])
    g = -adv.double() / rows
    want, size = lr.grad(r, g, torch.zeros(rows, dtype=torch.float64))
    near(d, want, lr.grad_tol(r, size, want, V, F32, extra=2e-5), "policy gradient")
    off = [0, 5, 12, 12, 20]
    off_d = torch.tensor(off, dtype=torch.int32, device=DEV)
    loss, each, reward, g = m.preference_loss(lp, off_d, beta=0.3)
    _, _, _, want_g = lr.preference(lp.cpu(), off, beta=0.3)
    d = m.token_logprobs_grad(c["dx"], smp.token, stats, d_logprob=g, inv_t=c["dinv"], allow=c["dallow"])
    want, size = lr.grad(r, want_g, torch.zeros(rows, dtype=torch.float64))
    near(d, want, lr.grad_tol(r, size, want, V, F32), "preference gradient")
    assert not d[20:].any()


def test_captured_steps_replayed():
    """A scoring call, a policy step of few rows (two launches), one of many (rows in registers), a token loss and a preference step in one captured graph,
    replayed four times on changed inputs with eager calls between; every replay against the eager results, to the bit."""
    m = gc.pkg()
    assert m.lib().ws_probe() == 0
    few, many = make(6, 60000, BF16, 51), make(140, 6000, F32, 52)
    off = torch.tensor([0, 40, 70, 71, 140], dtype=torch.int32, device=DEV)
    old = {k: torch.full((c["rows"],), -8.0, device=DEV) for k, c in (("few", few), ("many", many))}
    adv = {k: torch.linspace(-1, 1, c["rows"], device=DEV) for k, c in (("few", few), ("many", many))}
    long = {k: (v * 1.0).to(DEV) for k, v in tokens(3000, 3).items()}
    starts = few["dx"].clone(), many["dx"].clone(), long["lp"].clone()

    def prepare(k):
        few["dx"].copy_(torch.roll(starts[0], 13 * k, 1))
        many["dx"].copy_(torch.roll(starts[1], 7 * k, 1))
        long["lp"].copy_(starts[2] + 0.01 * k)

    def steps():
        out = []
        for k, c in (("few", few), ("many", many)):
            out += m.policy_loss_rows(c["dx"], c["dids"], old[k], adv[k], ref_logprob=old[k], inv_t=c["dinv"], kl_coef=0.1, entropy_coef=0.01)
        lp, stats, H = m.token_logprobs(few["dx"], few["dids"], want_entropy=True)
        lp2, stats2, _ = m.token_logprobs(many["dx"], many["dids"])
        loss, each, reward, g = m.preference_loss(lp2, off)
        out += [lp, stats, H, lp2, loss, each, reward, g, m.token_logprobs_grad(many["dx"], many["dids"], stats2, d_logprob=g)]
        out += m.policy_loss(long["lp"], long["old"], long["adv"], ref_logprob=long["ref"], entropy=long["H"], weight=long["w"], kl_coef=0.1)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = []
        for k in range(4):
            prepare(k)
            eager.append([t.clone() for t in steps()])
        prepare(0)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        held = steps()
        graph.capture_end()
        for k in range(4):
            prepare(k)
            graph.replay()
            between = steps()
            side.synchronize()
            for i, (a, b, e) in enumerate(zip(held, eager[k], between)):
                assert torch.equal(a, b), (k, i)
                assert torch.equal(e, b), (k, i)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_parts_that_do_not_wait_for_each_other_give_the_same_bits(dtype):
    """ws_policy.spins = 1: a part looks once and then works the missing parts' sums out itself, while their gradient may already be going over the logits. To the bit what
    waiting gives, in place or not, and the sums' and parts' words are left as the next call needs them (replays of a captured graph). In place has bits of its own: which
    thread adds up which logits goes by the boundaries of the memory that the gradient is written to."""
    m = gc.pkg()
    for rows, V, masked in ((1, 151936, False), (6, 100003, True), (40, 65537, False), (200, 50257, False), (2, 1048575, True)):
        c = make(rows, V, dtype, 61 + rows, masked, 3, 1)
        old, adv = torch.full((rows,), -7.0, device=DEV), torch.linspace(-1, 1, rows, device=DEV)
        args = dict(ref_logprob=old, inv_t=c["dinv"], allow=c["dallow"], kl_coef=0.1, entropy_coef=0.02)
        want = m.policy_loss_rows(c["dx"], c["dids"], old, adv, **args)
        start = c["dx"].clone()
        own = [t.clone() for t in m.policy_loss_rows(c["dx"], c["dids"], old, adv, out=c["dx"], **args)]
        for _ in range(4):
            c["dx"].copy_(start)
            got = m.policy_loss_rows(c["dx"], c["dids"], old, adv, spins=1, **args)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            got = m.policy_loss_rows(c["dx"], c["dids"], old, adv, spins=1, out=c["dx"], **args)
            assert all(torch.equal(a, b) for a, b in zip(got, own))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c["dx"].copy_(start)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            held = m.policy_loss_rows(c["dx"], c["dids"], old, adv, spins=1, out=c["dx"], **args)
            graph.capture_end()
            for _ in range(3):
                c["dx"].copy_(start)
                graph.replay()
                side.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(held, own))
        torch.cuda.current_stream().wait_stream(side)


def test_sums_of_a_second_launch_replayed():
    """Rows of one and of two parts, more than meet in one launch: the second launch adds up and breaks the parts' words. Captured, replayed on changed logits, eager calls between."""
    m = gc.pkg()
    assert m.lib().ws_probe() == 0
    for rows, V in ((1030, 5000), (1030, 40000)):
        c = make(rows, V, BF16, 57)
        old, adv = torch.full((rows,), -8.0, device=DEV), torch.linspace(-1, 1, rows, device=DEV)
        start = c["dx"].clone()

        def step():
            return m.policy_loss_rows(c["dx"], c["dids"], old, adv, ref_logprob=old, inv_t=c["dinv"], kl_coef=0.1, entropy_coef=0.01)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = []
            for k in range(3):
                c["dx"].copy_(torch.roll(start, 5 * k, 1))
                eager.append([t.clone() for t in step()])
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            held = step()
            graph.capture_end()
            for k in range(3):
                c["dx"].copy_(torch.roll(start, 5 * k, 1))
                graph.replay()
                between = step()
                side.synchronize()
                assert all(torch.equal(a, b) and torch.equal(e, b) for a, b, e in zip(held, eager[k], between)), (rows, V, k)
        torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("rows,V,stride", [(5, 40, 40), (5, 40, 48), (1, 40, 100), (5, 1, 1), (5, 1, 3), (1, 1, 1)])
def test_gradients_of_rows_apart_are_contiguous(rows, V, stride):
    m = gc.pkg()
    x = torch.randn(rows, stride, device=DEV)[:, :V]
    ids, v = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.ones(rows, device=DEV)
    lp, stats, _ = m.token_logprobs(x, ids)
    for d in (m.token_logprobs_grad(x, ids, stats, d_logprob=v), m.policy_loss_rows(x, ids, lp, -rows * v)[3]):
        assert d.shape == (rows, V) and d.is_contiguous()
        want = -torch.softmax(x.double(), 1)
        want[:, 0] += 1.0
        assert float((d.double() - want).abs().max()) <= 60 * lr.EPS  # (sums and powers as in loss_ref.sum_tol: 42 half steps and the exponents' 16)


def test_rows_far_apart():
    """Offsets beyond 32 bits: three rows 1.5e9 elements apart, of logits and of their gradient."""
    m = gc.pkg()
    V, stride = 5003, 1500000001
    c = make(3, V, BF16, 71)
    mem, out = torch.empty(3 * stride, dtype=BF16, device=DEV), torch.empty(3 * stride, dtype=BF16, device=DEV)
    far, far_out = mem.view(3, stride)[:, :V], out.view(3, stride)[:, :V]
    far.copy_(c["x"])
    old, adv = torch.full((3,), -7.0, device=DEV), torch.ones(3, device=DEV)
    near_by = m.policy_loss_rows(c["dx"], c["dids"], old, adv, entropy_coef=0.1)
    away = m.policy_loss_rows(far, c["dids"], old, adv, entropy_coef=0.1, out=far_out)
    # (rows begin elsewhere against the 16-byte boundaries, so a thread has other logits: sums differ in their last bits, within twice what either may be off)
    assert float((near_by[1] - away[1]).abs().max()) <= 2 * float(lr.lp_tol(lr.score(c["x"], c["ids"]), V).max())
    assert float((near_by[3].float() - away[3].float()).abs().max()) <= 2 ** -8 * float(near_by[3].float().abs().max())
    lp, stats, H = m.token_logprobs(far, c["dids"], want_entropy=True)
    r = lr.score(c["x"], c["ids"])
    near(lp, r["lp"], lr.lp_tol(r, V), "logprob")
    near(H, r["H"], lr.H_tol(r, V), "entropy")
    g = m.token_logprobs_grad(far, c["dids"], stats, d_logprob=adv, out=far_out)
    want, size = lr.grad(r, torch.ones(3, dtype=torch.float64), torch.zeros(3, dtype=torch.float64))
    near(g, want, lr.grad_tol(r, size, want, V, BF16), "gradient")


def test_scores_without_a_workspace():
    """Through the C entry point: every row is one workgroup's then."""
    import ctypes as C
    m = gc.pkg()
    for rows, V in ((2, 151936), (1, 40000), (1, 1048575)):
        c = make(rows, V, F32, 81)
        r = lr.score(c["x"], c["ids"], c["inv_t"])
        d = m.LossRows(c["dx"].data_ptr(), m.DTYPE_F32, rows, V, V, c["dids"].data_ptr(), c["dinv"].data_ptr())
        assert m.lib().ws_token_logprobs_workspace(C.byref(d)) > 0
        lp, stats, H = torch.empty(rows, device=DEV), torch.empty((rows, 2), device=DEV), torch.empty(rows, device=DEV)
        m.check(m.lib().ws_token_logprobs(torch.cuda.current_stream().cuda_stream, C.byref(d), lp.data_ptr(), stats.data_ptr(), H.data_ptr(), None, 0), "ws_token_logprobs")
        # (a thread adds V / 256 terms here, as everywhere the tolerance says)
        near(lp, r["lp"], lr.lp_tol(r, V), "logprob")
        near(H, r["H"], lr.H_tol(r, V), "entropy")
        assert torch.equal(stats[:, 0].cpu().double(), r["m"])


def test_calls_on_two_streams_at_once():
    m = gc.pkg()
    cases = [make(8, 90000, BF16, 91 + i) for i in range(2)]
    old = torch.full((8,), -7.0, device=DEV)
    adv = torch.linspace(-1, 1, 8, device=DEV)
    call = lambda c: m.policy_loss_rows(c["dx"], c["dids"], old, adv, inv_t=c["dinv"], entropy_coef=0.02)  # noqa: E731
    want = [call(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(call(c))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_arguments_that_are_refused():
    m = gc.pkg()
    x, ids, v = torch.zeros((4, 100), device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, device=DEV)
    st = torch.ones((4, 2), device=DEV)
    words = torch.zeros((4, 4), dtype=torch.int32, device=DEV)
    bad = [lambda: m.token_logprobs(x.half(), ids), lambda: m.token_logprobs(x[:, ::2], ids), lambda: m.token_logprobs(x[0], ids), lambda: m.token_logprobs(x, ids.long()),
           lambda: m.token_logprobs(x, ids[:3]), lambda: m.token_logprobs(x, ids.cpu()), lambda: m.token_logprobs(x, ids, inv_t=v.double()),
           lambda: m.token_logprobs(x, ids, allow=words[:, :3]), lambda: m.token_logprobs(x, ids, allow=words[:3]), lambda: m.token_logprobs(x[:1].expand(4, 100), ids),
           lambda: m.token_logprobs_grad(x, ids, None, d_logprob=v), lambda: m.token_logprobs_grad(x, ids, st[:3], d_logprob=v), lambda: m.token_logprobs_grad(x, ids, st, d_entropy=v),
           lambda: m.token_logprobs_grad(x, ids, st, d_logprob=v, out=x.bfloat16()), lambda: m.token_logprobs_grad(x, ids, st, d_logprob=v, out=x[:3]),
           lambda: m.token_logprobs_grad(x.view(-1)[:396].view(4, 99), ids, st, d_logprob=v, out=x.view(-1)[4:].view(4, 99)),
           lambda: m.policy_loss_rows(x, None, v, v), lambda: m.policy_loss_rows(x, ids, None, v), lambda: m.policy_loss_rows(x, ids, v, v, kl_coef=0.1),
           lambda: m.policy_loss_rows(x, ids, v, v, dual_clip=0.5), lambda: m.policy_loss(v, v, v, entropy_coef=0.1), lambda: m.policy_loss(v, v[:3], v),
           lambda: m.policy_loss(v, v, v, clip_low=2.0), lambda: m.preference_loss(v, ids[:1]), lambda: m.preference_loss(v, ids), lambda: m.preference_loss(v, ids[:3], label_smoothing=2.0),
           lambda: m.preference_loss(v, ids[:3], ref_logprob=v[:2])]
    for i, call in enumerate(bad):
        with pytest.raises(m.WsError):
            call()
            raise AssertionError(i)


FIRST_CALL = """
import sys, torch
sys.path[:0] = [{root!r}]
from __graft_entry__ import load_package
m = load_package()
x = torch.randn(3, 70001, device="cuda:0")
ids = torch.zeros(3, dtype=torch.int32, device="cuda:0")
v = torch.zeros(3, device="cuda:0")
side = torch.cuda.Stream()
torch.cuda.synchronize()
assert m.lib().ws_probe() == 0
graph = torch.cuda.CUDAGraph()
with torch.cuda.stream(side):
    graph.capture_begin()
    lp, stats, _ = m.token_logprobs(x, ids)
    sums, lp2, H, d = m.policy_loss_rows(x, ids, v, v + 1.0, entropy_coef=0.1)
    graph.capture_end()
    for k in range(3):
        x.add_(0.25)
        graph.replay()
        want = m.token_logprobs(x, ids), m.policy_loss_rows(x, ids, v, v + 1.0, entropy_coef=0.1)
        side.synchronize()
        assert torch.equal(lp, want[0][0]) and torch.equal(d, want[1][3]) and torch.equal(sums, want[1][0])
print("captured first")
"""


def test_first_calls_of_a_process_under_capture():
    """ws_probe loads the kernels, so a captured call may be the first that needs them."""
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=gc.ROOT)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]
