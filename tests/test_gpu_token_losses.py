"""GPU parity of the log-probability, policy and preference operators with their definitions in 64 bits.

Tolerances are counted in roundings.  u = 2^-24 is half a step of a float.
  logp, lse: an exponential is off by 2^-22 (hardware exp2) plus the roundings of its argument d = z - m, 2 u |d|, which
  weigh at most e^-|d| |d| < 0.37; a sum of n terms over 32 threads or more adds the roundings of its longest chain
  (n / 32 / 8 terms at most, counted as 64 here for the sizes below) and of ten merges with two exponentials each:
  (64 + 20 * 4 + 4) u = 150 u relative to the sum, hence absolute in log s; then log, differences and the sum m + log s
  round at most 4 times at the magnitude of |logp| + |lse|.
  Everything behind it is the derivative of a formula times that, plus a handful of roundings of its own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
# one class to many, around 16-byte vectors, warps, thread blocks and the kernels' own limits
CLASSES = [1, 2, 7, 8, 9, 31, 64, 255, 257, 1000, 1001, 2047, 2048, 2056, 4099, 8200, 16390, 32000, 33001, 65544, 70003]


def rows_of(rows, classes, dtype, pad=0, skip=0, seed=0, spread=3.0):
    """[rows, classes] logits whose first element lies `skip` elements behind an aligned address."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.randn(skip + rows * (classes + pad) + 8, generator=g, device="cuda") * spread
    flat = flat.to(dtype)
    return torch.as_strided(flat, (rows, classes), (classes + pad, 1), skip)


def ints(rows, classes, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, classes, (rows,), generator=g, device="cuda", dtype=torch.int32)


def floats(n, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, generator=g, device="cuda") * scale


def one(x):
    return torch.tensor([x], dtype=torch.float32, device="cuda")


def stats64(z, y):
    z = z.double()
    top = z.amax(1)
    top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    return z.gather(1, y.long().clamp(0, z.shape[1] - 1)[:, None])[:, 0] - lse, lse


def near(got, want, tol, what):
    off = (got.double() - want).abs()
    same = (got.double() == want) | (torch.isnan(got.double()) & torch.isnan(want))
    bad = ~(same | (off <= tol))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max()):.3g} x the tolerance"


def logp_tol(logp, lse):
    return U * (150 + 4 * (logp.abs() + lse.abs()))


def check_gradient(got, z, y, coef, coef_tol, lse_tol):
    """got = coef (onehot - p) rounded once; coef_tol, lse_tol [rows]: what coef and log s may be off by."""
    p = torch.softmax(z.double(), 1)
    hot = torch.zeros_like(p)
    rows = torch.arange(z.shape[0], device="cuda")
    ok = (y >= 0) & (y < z.shape[1])
    hot[rows[ok], y[ok].long()] = 1.0
    want = torch.where((coef != 0)[:, None], coef[:, None] * (hot - p), torch.zeros_like(p))
    info = torch.finfo(got.dtype)
    # p: exponential 4 u, its argument 2 u |d| <= u (2 * 0.37 / p) p, division and two products 4 u, sum lse_tol
    tol = coef.abs()[:, None] * (p * (8 * U + lse_tol[:, None]) + U) + coef_tol[:, None] * (p + hot)
    tol = tol + want.abs() * (info.eps / 2 + 2 * U) + info.smallest_normal * info.eps / 2
    near(got, want, tol, "dlogits")


# ------------------------------------------------------------------------------------------------ log-probabilities

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_token_logprobs(dtype, classes):
    from renaissance_b200 import ops
    for rows, pad, skip in ((1, 0, 0), (5, 0, 0), (19, 3, 1), (33, 8, 8)):
        z = rows_of(rows, classes, dtype, pad, skip, seed=rows)
        y = ints(rows, classes)
        if rows > 4:
            y[1], y[3] = -1, classes
        out = ops.token_logprobs(z, y)
        logp, lse = stats64(z, y)
        off = (y < 0) | (y >= classes)
        logp, lse = logp.masked_fill(off, 0), lse.masked_fill(off, 0)
        near(out["logp"], logp, logp_tol(logp, lse), "logp")
        near(out["lse"], lse, logp_tol(logp, lse), "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [1, 9, 1000, 4099, 40000])
def test_extreme_logits(dtype, classes):
    """Minus infinity and the type's lowest value as masks, in part of a row and in all of it; infinity and NaN."""
    from renaissance_b200 import ops
    z = rows_of(9, classes, dtype, seed=3)
    y = torch.zeros(9, dtype=torch.int32, device="cuda")
    low = torch.finfo(dtype).min
    z[0] = -math.inf
    z[1] = low                              # all alike: a uniform distribution
    z[2, 1:] = -math.inf
    z[3, 1:] = low
    z[4, 0] = -math.inf                     # the label itself is masked
    z[5, classes // 2] = math.nan
    z[6, classes - 1] = math.inf
    y[8] = -1
    z[8] = math.nan                         # does not count: not read
    out = ops.token_logprobs(z, y)
    logp, lse = out["logp"].tolist(), out["lse"].tolist()
    assert logp[0] == lse[0] == -math.inf
    assert abs(logp[1] + math.log(classes)) <= U * (150 + 8 * math.log(classes))
    assert logp[2] == logp[3] == 0.0
    assert logp[4] == -math.inf and (math.isfinite(lse[4]) if classes > 1 else lse[4] == -math.inf)
    assert math.isnan(logp[5]) and math.isnan(lse[5]) and math.isnan(logp[6])
    assert math.isfinite(logp[7])
    assert logp[8] == lse[8] == 0.0


# ------------------------------------------------------------------------------------------------ policy loss

def policy64(z, y, old, adv, ref, w, lo, hi, k, scaling):
    """(loss_partial, logp, coef = scaling * d loss / d logp, what each may be off by, rows that count)."""
    classes = z.shape[1]
    logp, lse = stats64(z, y)
    counts = (y >= 0) & (y < classes) & (w != 0) & ~torch.isinf(lse)
    w, old, adv = w.double(), old.double(), adv.double()
    lo, hi = float(torch.tensor(1.0) - torch.tensor(lo)), float(torch.tensor(1.0) + torch.tensor(hi))
    ratio = torch.exp(logp - old)
    kept, cut = ratio * adv, ratio.clamp(lo, hi) * adv
    loss = -torch.minimum(kept, cut)
    slope = torch.where(kept <= cut, -kept, torch.zeros_like(kept))
    t = logp_tol(logp, lse)
    rel = t + U * (4 + (logp - old).abs())                  # of the ratio
    loss_tol, slope_tol = kept.abs() * rel, slope.abs() * rel
    if ref is not None:
        gap = ref.double() - logp
        loss = loss + k * (torch.expm1(gap) - gap)
        slope = slope - k * torch.expm1(gap)
        gap_tol = t + U * gap.abs()
        loss_tol = loss_tol + k * (torch.expm1(gap).abs() + 4 * U) * gap_tol + 6 * U * k * (torch.expm1(gap).abs() + gap.abs())
        slope_tol = slope_tol + k * torch.exp(gap) * gap_tol + 6 * U * k * torch.expm1(gap).abs()
    zero = torch.zeros_like(logp)
    pick = lambda x: torch.where(counts, x, zero)
    part, coef = pick(loss * w), pick(slope * w * scaling)
    part_tol = pick((loss_tol + 4 * U * loss.abs()) * w.abs())
    coef_tol = pick((slope_tol + 4 * U * slope.abs()) * w.abs() * scaling)
    return part, pick(logp), coef, part_tol, pick(t), coef_tol


def policy_inputs(rows, classes, dtype, pad, skip, seed, kl, masked):
    z = rows_of(rows, classes, dtype, pad, skip, seed)
    y = ints(rows, classes, seed + 1)
    logp = stats64(z, y)[0]
    moved = floats(rows, seed + 2, 0.3).double()
    for border in (math.log(0.8), math.log(1.28)):          # off the kinks, where the gradient jumps
        moved = torch.where((moved - border).abs() < 1e-3, torch.full_like(moved, border + 2e-3), moved)
    old = (logp - moved).float()
    ref = (logp + floats(rows, seed + 3, 0.4).double()).float() if kl else None
    adv = floats(rows, seed + 4)
    w = floats(rows, seed + 5).abs() + 0.1
    if masked and rows > 3:
        y[1] = classes
        w[2] = 0
        z[2] = math.nan                                     # behind the mask: not read
        adv[3] = 0
    return z, y, old, adv, ref, w / w.sum()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_policy_loss(dtype, classes):
    from renaissance_b200 import ops
    for rows, pad, skip, kl in ((1, 0, 0, False), (6, 0, 0, True), (21, 5, 1, True), (40, 8, 8, False)):
        z, y, old, adv, ref, w = policy_inputs(rows, classes, dtype, pad, skip, 10 * rows, kl, True)
        k = 0.05 if kl else 0.0
        scaling = 4096.0
        out = ops.policy_loss_fused(z, y, old, adv, one(scaling), 0.2, 0.28, ref, k, w)
        part, logp, coef, part_tol, t, coef_tol = policy64(z, y, old, adv, ref, w, 0.2, 0.28, k, scaling)
        near(out["logp"], logp, t, "logp")
        near(out["loss_partial"], part, part_tol, "loss_partial")
        near(out["loss"], part.sum().reshape(1), part_tol.sum() + U * part.sum().abs() + 1e-45, "loss")
        z = torch.where((w == 0)[:, None], torch.zeros_like(z), z)
        check_gradient(out["dlogits"], z, y, coef, coef_tol, t)


@pytest.mark.parametrize("classes", [9, 1000, 5001, 32000])
def test_policy_loss_gradient_matches_differences(classes):
    """Float logits: the gradient along a random direction against central differences of the 64-bit loss."""
    from renaissance_b200 import ops
    z, y, old, adv, ref, w = policy_inputs(12, classes, torch.float32, 0, 0, 77, True, True)
    out = ops.policy_loss_fused(z, y, old, adv, one(1.0), 0.2, 0.28, ref, 0.05, w)
    z = torch.where((w == 0)[:, None], torch.zeros_like(z), z).double()
    d = torch.randn(z.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda", dtype=torch.float64)
    h = 1e-5
    f = lambda s: policy64(z + s * h * d, y, old, adv, ref, w, 0.2, 0.28, 0.05, 1.0)[0].sum()
    slope = (f(1) - f(-1)) / (2 * h)
    got = (out["dlogits"].double() * d).sum()
    # the loss's third derivative is of order 10 along d: h^2 * 10; float gradients: 100 u of each product
    assert abs(float(got - slope)) < 10 * h * h * classes + 200 * U * float((out["dlogits"].double() * d).abs().sum())


def test_policy_loss_defaults_and_clipped_rows():
    from renaissance_b200 import ops
    z = rows_of(8, 100, torch.float32, seed=2)
    y = ints(8, 100)
    logp = stats64(z, y)[0].float()
    adv = torch.tensor([1.0, 1, -1, -1, 1, -1, 0, 2], device="cuda")
    move = torch.tensor([0.5, -0.5, -0.5, 0.5, 0, 0, 1, -1], device="cuda")     # log ratio
    out = ops.policy_loss_fused(z, y, logp - move, adv, one(1.0))
    want = policy64(z, y, logp - move, adv, None, torch.full((8,), 0.125, device="cuda"), 0.2, 0.2, 0.0, 1.0)
    near(out["loss_partial"], want[0], want[3], "loss_partial")
    # ratio above its bound with a gain, below it with a loss: clipped, nothing flows
    gone = (out["dlogits"] == 0).all(1).tolist()
    assert gone == [True, False, True, False, False, False, True, False]


@pytest.mark.parametrize("classes", [16, 3000, 20000])
def test_policy_loss_rows_without_a_distribution(classes):
    from renaissance_b200 import ops
    z, y, old, adv, ref, w = policy_inputs(7, classes, torch.bfloat16, 0, 0, 5, True, False)
    z[3] = -math.inf
    y[5] = 0
    z[5, 0] = math.nan
    out = ops.policy_loss_fused(z, y, old, adv, one(1.0), 0.2, 0.28, ref, 0.05, w)
    assert float(out["loss_partial"][3]) == 0 and float(out["logp"][3]) == 0 and not out["dlogits"][3].any()
    assert math.isnan(float(out["logp"][5])) and math.isnan(float(out["loss"])) and out["dlogits"][5].isnan().all()
    others = [0, 1, 2, 4, 6]
    assert out["dlogits"][others].isfinite().all() and out["loss_partial"][others].isfinite().all()


# ------------------------------------------------------------------------------------------------ preference loss

def preference64(z, y, starts, ref, beta, eps, scaling):
    rows, classes = z.shape
    logp, lse = stats64(z, y)
    counts = (y >= 0) & (y < classes) & ~torch.isinf(lse)
    seqs = len(starts) - 1
    owner = torch.full((rows,), -1, dtype=torch.int64)
    for q in range(seqs):
        owner[starts[q]:starts[q + 1]] = q
    owner = owner.cuda()
    counts &= owner >= 0
    logp = torch.where(counts, logp, torch.zeros_like(logp))
    t = torch.where(counts, logp_tol(logp, lse), torch.zeros_like(logp))
    S = torch.stack([logp[starts[q]:starts[q + 1]].sum() for q in range(seqs)])
    S_tol = torch.stack([t[starts[q]:starts[q + 1]].sum() for q in range(seqs)]) + U * S.abs() + 1e-45
    gap = S - (ref.double() if ref is not None else 0.0)
    x = beta * (gap[0::2] - gap[1::2])
    x_tol = abs(beta) * (S_tol[0::2] + S_tol[1::2])
    pairs = seqs // 2
    softplus = lambda v: v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))
    part = ((1 - eps) * softplus(-x) + eps * softplus(x)) / pairs
    pull = beta * (eps * torch.sigmoid(x) - (1 - eps) * torch.sigmoid(-x)) / pairs * scaling
    pull_tol = abs(beta) * scaling / pairs * x_tol * 0.25 + 2 * U * pull.abs()
    coef = torch.zeros_like(logp)
    coef_tol = torch.zeros_like(logp)
    for q in range(seqs):
        coef[starts[q]:starts[q + 1]] = pull[q // 2] * (1 if q % 2 == 0 else -1)
        coef_tol[starts[q]:starts[q + 1]] = pull_tol[q // 2]
    coef, coef_tol = torch.where(counts, coef, torch.zeros_like(coef)), torch.where(counts, coef_tol, torch.zeros_like(coef))
    return part, x_tol / pairs + 2 * U * part, S, S_tol, logp, t, coef, coef_tol


def check_preference(z, y, starts, ref, beta=0.1, eps=0.0, scaling=1.0, front=0):
    from renaissance_b200 import ops
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out = ops.preference_loss_fused(z, y, st, ref, one(scaling), beta, eps)
    part, part_tol, S, S_tol, logp, t, coef, coef_tol = preference64(z, y, starts, ref, beta, eps, scaling)
    near(out["logp"], logp, t, "logp")
    near(out["seq_logp"], S, S_tol, "seq_logp")
    near(out["loss_partial"], part, part_tol, "loss_partial")
    near(out["loss"], part.sum().reshape(1), part_tol.sum() + 2 * U * part.sum(), "loss")
    check_gradient(out["dlogits"], torch.where((coef == 0)[:, None], torch.zeros_like(z), z), y, coef, coef_tol, t)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_preference_loss(dtype, classes):
    for starts, behind, pad, skip in (([0, 1, 2], 0, 0, 0), ([0, 3, 3, 10, 14], 2, 5, 1), ([2, 7, 12, 12, 12, 20, 33], 1, 8, 8)):
        rows = starts[-1] + behind
        z = rows_of(rows, classes, dtype, pad, skip, seed=rows)
        y = ints(rows, classes)
        y[starts[0]::5] = -1
        ref = floats(len(starts) - 1, 9, 3.0) - 20
        check_preference(z, y, starts, ref, 0.3, 0.1, 4096.0)


def test_preference_loss_far_apart_pairs_and_no_reference():
    """Margins so large that a sigmoid is 0 or 1 in floats, both ways; sequences without rows; no reference."""
    z = rows_of(40, 300, torch.float32, seed=4, spread=8.0)
    y = ints(40, 300)
    check_preference(z, y, [0, 10, 20, 30, 40], None, 0.5)
    check_preference(z, y, [0, 0, 40], torch.tensor([900.0, -900.0], device="cuda"), 1.0, 0.0)
    check_preference(z, y, [0, 40, 40], torch.tensor([900.0, -900.0], device="cuda"), 1.0, 0.25)
    check_preference(z, y, [0, 0, 0], torch.tensor([0.5, -1.0], device="cuda"))
    out = check_preference(z, y, [0, 10, 20, 30, 40], None, 0.0)
    assert not out["dlogits"].any()


def test_preference_loss_many_pairs_and_long_sequences():
    """2000 pairs of zero to three rows; two sequences of 20 000 rows."""
    lens = [(i * 7) % 4 for i in range(4000)]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    z = rows_of(starts[-1], 33, torch.bfloat16, seed=8)
    check_preference(z, ints(starts[-1], 33), starts, floats(4000, 3, 2.0), 0.2, 0.1, 1e5)
    z = rows_of(40_000, 17, torch.float32, seed=8)
    y = ints(40_000, 17)
    ref = torch.stack([stats64(z[:20_000], y[:20_000])[0].sum(), stats64(z[20_000:], y[20_000:])[0].sum()]).float()
    check_preference(z, y, [0, 20_000, 40_000], ref, 0.1, 0.0, 1e3)


def test_preference_rows_outside_and_without_distribution():
    from renaissance_b200 import ops
    z = rows_of(12, 500, torch.float16, seed=6)
    y = ints(12, 500)
    z[0] = z[1] = z[11] = math.nan          # outside every sequence
    y[3] = -1
    z[3] = math.nan                         # no label
    z[6] = -math.inf                        # no distribution
    out = ops.preference_loss_fused(z, y, torch.tensor([2, 6, 11], dtype=torch.int32, device="cuda"), None, one(512.0), 0.2)
    assert out["loss"].isfinite().all() and out["dlogits"].isfinite().all()
    for r in (0, 1, 3, 6, 11):
        assert not out["dlogits"][r].any() and float(out["logp"][r]) == 0
    assert out["dlogits"][2].any() and out["dlogits"][10].any()


def test_preference_bounds_from_the_device_are_clamped():
    """Bounds below 0, past the rows or not ascending: no access outside the buffers, whatever the sums are."""
    from renaissance_b200 import ops
    z = rows_of(12, 64, torch.float32, seed=6)
    y = ints(12, 64)
    for starts in ([-5, 6, 99], [9, 3, 12], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [0, 100, 5]):
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        out = ops.preference_loss_fused(z, y, st, None, one(1.0), 0.2)
        assert out["dlogits"].isfinite().all()
    out = ops.preference_loss_fused(z, y, torch.tensor([-5, 6, 99], dtype=torch.int32, device="cuda"), None, one(1.0), 0.2)
    want = ops.preference_loss_fused(z, y, torch.tensor([0, 6, 12], dtype=torch.int32, device="cuda"), None, one(1.0), 0.2)
    assert torch.equal(out["dlogits"], want["dlogits"]) and torch.equal(out["loss"], want["loss"])


# ------------------------------------------------------------------------------------------------ one number for a row

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [100, 1000, 2048, 5001, 32000, 50021, 131072, 140000])
def test_a_rows_logp_does_not_depend_on_batch_or_operator(dtype, classes):
    """Few rows are cut among more thread blocks than many; the sums are the same ones, so that a ratio of the policy
    with itself is exactly 1."""
    from renaissance_b200 import ops
    rows = 1500
    z = rows_of(rows, classes, dtype, seed=classes)
    y = ints(rows, classes)
    w = torch.full((rows,), 1.0 / rows, device="cuda")
    many = ops.token_logprobs(z, y)
    for n in (1, 3, 100):
        few = ops.token_logprobs(z[:n], y[:n])
        assert torch.equal(few["logp"], many["logp"][:n]) and torch.equal(few["lse"], many["lse"][:n])
    for n in (2, rows):
        adv = floats(n, 5)
        out = ops.policy_loss_fused(z[:n], y[:n], many["logp"][:n], adv, one(1.0), weights=w[:n])
        assert torch.equal(out["logp"], many["logp"][:n])
        assert torch.equal(out["loss_partial"], -adv * w[:n])           # ratio 1
        st = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
        assert torch.equal(ops.preference_loss_fused(z[:n], y[:n], st, None, one(1.0))["logp"], many["logp"][:n])


# ------------------------------------------------------------------------------------------------ how they are called

def test_no_rows():
    from renaissance_b200 import ops
    z = torch.empty((0, 50), device="cuda", dtype=torch.float16)
    y = torch.empty(0, dtype=torch.int32, device="cuda")
    f = torch.empty(0, device="cuda")
    assert ops.token_logprobs(z, y)["logp"].numel() == 0
    assert float(ops.policy_loss_fused(z, y, f, f, one(1.0))["loss"]) == 0.0
    out = ops.preference_loss_fused(z, y, torch.zeros(3, dtype=torch.int32, device="cuda"), None, one(1.0))
    assert abs(float(out["loss"]) - math.log(2)) < 1e-6


def test_given_gradient_buffer_keeps_its_padding():
    """dlogits as the left columns of a wider buffer, at an alignment other than the logits'."""
    from renaissance_b200 import ops
    for classes, zpad, zskip, dpad, dskip in ((1001, 23, 0, 7, 1), (1000, 24, 0, 24, 8), (777, 0, 3, 0, 0), (33001, 7, 0, 1, 5)):
        for dtype in DTYPES:
            z, y, old, adv, ref, w = policy_inputs(9, classes, dtype, zpad, zskip, 3, True, False)
            flat = torch.full((dskip + 9 * (classes + dpad) + 16,), 7.0, dtype=dtype, device="cuda")
            d = torch.as_strided(flat, (9, classes), (classes + dpad, 1), dskip)
            want = ops.policy_loss_fused(z, y, old, adv, one(64.0), 0.2, 0.28, ref, 0.05, w)
            got = ops.policy_loss_fused(z, y, old, adv, one(64.0), 0.2, 0.28, ref, 0.05, w, dlogits=d)
            assert got["dlogits"].data_ptr() == d.data_ptr() and torch.equal(d, want["dlogits"])
            d.fill_(7.0)
            assert (flat == 7.0).all()
            st = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
            want = ops.preference_loss_fused(z, y, st, None, one(64.0))
            ops.preference_loss_fused(z, y, st, None, one(64.0), dlogits=d)
            assert torch.equal(d, want["dlogits"])
            d.fill_(7.0)
            assert (flat == 7.0).all()


def test_results_are_reproducible_and_other_streams_agree():
    from renaissance_b200 import ops
    z, y, old, adv, ref, w = policy_inputs(300, 5000, torch.bfloat16, 0, 0, 3, True, True)
    st = torch.tensor([0, 100, 150, 200, 300], dtype=torch.int32, device="cuda")
    first = ops.policy_loss_fused(z, y, old, adv, one(64.0), 0.2, 0.28, ref, 0.05, w)
    pref = ops.preference_loss_fused(z, y, st, None, one(64.0))
    side = torch.cuda.Stream()
    scale = one(64.0)
    torch.cuda.synchronize()
    for _ in range(3):
        a = ops.policy_loss_fused(z, y, old, adv, scale, 0.2, 0.28, ref, 0.05, w, stream=side)
        b = ops.preference_loss_fused(z, y, st, None, scale, stream=side)
        c = ops.policy_loss_fused(z, y, old, adv, scale, 0.2, 0.28, ref, 0.05, w)
        torch.cuda.synchronize()
        for k in ("loss", "loss_partial", "logp"):
            assert torch.equal(a[k], first[k]) and torch.equal(c[k], first[k])
        bits = lambda t: t.view(torch.int16)        # one row is NaN in the preference loss, which does not mask it
        assert torch.equal(bits(a["dlogits"]), bits(first["dlogits"])) and torch.equal(bits(b["dlogits"]), bits(pref["dlogits"]))
        assert torch.equal(bits(b["loss"]), bits(pref["loss"]))


def test_captured_calls_replay_beside_eager_ones():
    """Two captured graphs and eager calls on one stream's inputs: replays on different streams do not disturb one
    another."""
    from renaissance_b200 import ops
    z, y, old, adv, ref, w = policy_inputs(200, 4100, torch.float16, 0, 0, 3, True, False)
    st = torch.tensor([0, 100, 200], dtype=torch.int32, device="cuda")
    scale = one(64.0)
    call = lambda: (ops.policy_loss_fused(z, y, old, adv, scale, 0.2, 0.28, ref, 0.05, w),
                    ops.preference_loss_fused(z, y, st, None, scale), ops.token_logprobs(z, y))
    want = call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out, torch.cuda.Stream()))
    for _ in range(4):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        now = call()
        torch.cuda.synchronize()
        for got in [now] + [o for _, o, _ in graphs]:
            for a, b in zip(got, want):
                for k in a:
                    assert torch.equal(a[k].nan_to_num(), b[k].nan_to_num()), k
    for g, out, _ in graphs:                # the inputs' buffers are what is captured, not their values
        z.mul_(0.5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[2]["logp"], ops.token_logprobs(z, y)["logp"])


def test_python_checks_on_device_tensors():
    from renaissance_b200 import _lib, ops
    z = rows_of(4, 64, torch.float16)
    y, f = ints(4, 64), floats(4, 1)
    with pytest.raises(TypeError):
        ops.token_logprobs(z.double(), y)
    with pytest.raises(TypeError):
        ops.token_logprobs(z, y.long())
    with pytest.raises(ValueError):
        ops.token_logprobs(z, y[:3])
    with pytest.raises(ValueError):
        ops.token_logprobs(z.t(), y)
    with pytest.raises(ValueError):
        ops.token_logprobs(z[:1].expand(4, 64), y)
    with pytest.raises(ValueError):
        ops.policy_loss_fused(z, y, f, f, one(1.0), dlogits=torch.empty_like(z)[:, :32])
    with pytest.raises(_lib.Trb200Error):
        ops.policy_loss_fused(z, y, f, f, one(1.0), dlogits=z)
    with pytest.raises(_lib.Trb200Error):
        ops.policy_loss_fused(z, y, f, f, one(1.0), kl_coef=0.1)
    with pytest.raises(_lib.Trb200Error):
        ops.policy_loss_fused(z, y, f, f, one(1.0), clip_low=1.5)
    with pytest.raises(ValueError):
        ops.preference_loss_fused(z, y, torch.zeros(4, dtype=torch.int32, device="cuda"), None, one(1.0))
    with pytest.raises(TypeError):
        ops.policy_loss_fused(z, y, f.cpu(), f, one(1.0))


def test_offsets_past_32_bits():
    """Logits of more than 2^32 bytes and 2^31 elements: the last rows against the same rows alone."""
    from renaissance_b200 import ops
    rows, classes = 17000, 131071
    z = torch.empty((rows, classes), dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    y = ints(rows, classes)
    old, adv = floats(rows, 3, 0.1) - 12, floats(rows, 4)
    w = torch.full((rows,), 0.25, device="cuda")
    out = ops.policy_loss_fused(z, y, old, adv, one(64.0), weights=w)
    tail = slice(rows - 40, rows)
    alone = ops.policy_loss_fused(z[tail], y[tail], old[tail], adv[tail], one(64.0), weights=w[tail])
    assert torch.equal(out["logp"][tail], alone["logp"]) and torch.equal(out["dlogits"][tail], alone["dlogits"])
    logp, lse = stats64(z[tail], y[tail])
    near(out["logp"][tail], logp, U * (400 + 4 * (logp.abs() + lse.abs())), "logp")
    del out, alone
    st = torch.tensor([0, rows - 40, rows], dtype=torch.int32, device="cuda")
    got = ops.preference_loss_fused(z, y, st, torch.tensor([-12.0 * (rows - 40), -480.0], device="cuda"), one(64.0), 0.01)
    p = torch.softmax(z[tail].double(), 1)
    pull = got["dlogits"][tail].double() / -(p - torch.nn.functional.one_hot(y[tail].long(), classes))
    at = pull.gather(1, y[tail].long()[:, None])
    assert (at.amax() - at.amin()) <= at.abs().amax() * 2.0 ** -7


@pytest.mark.parametrize("classes", [1000, 33001])
def test_captured_branches_that_join_before_a_loss(classes):
    """One graph, two streams: the policy's and the reference's log-probabilities side by side, both waited for by the
    loss, which begins while the kernel in front of it still runs.  Replays see new logits, as the same calls in a row
    do."""
    from renaissance_b200 import ops
    rows = 300
    z, y, old, adv, ref, w = policy_inputs(rows, classes, torch.bfloat16, 0, 0, 3, True, False)
    other = rows_of(rows, classes, torch.bfloat16, seed=11)
    scale = one(64.0)

    def loss(side=None):
        main = torch.cuda.current_stream()
        if side is None:
            was, before = ops.token_logprobs(z, y), ops.token_logprobs(other, y)
        else:
            side.wait_stream(main)
            with torch.cuda.stream(side):
                before = ops.token_logprobs(other, y)
            was = ops.token_logprobs(z, y)
            main.wait_stream(side)
        return ops.policy_loss_fused(z, y, was["logp"], adv, scale, 0.2, 0.28, before["logp"], 0.05)

    loss()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = loss(side)
    for step in range(5):
        z.mul_(0.9)
        other.add_(z)
        for k in out:
            out[k].fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        want, apart = loss(), loss(torch.cuda.Stream())
        torch.cuda.synchronize()
        for k in out:
            assert torch.equal(out[k].nan_to_num(), want[k].nan_to_num()), (k, step)
            assert torch.equal(apart[k].nan_to_num(), want[k].nan_to_num()), (k, step)
