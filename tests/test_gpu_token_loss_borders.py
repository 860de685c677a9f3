"""The token losses where a formula taken as it stands loses its digits, or where a row leaves the ordinary range.  The
definitions in 64 bits, and how tolerances are counted, are those of test_gpu_token_losses."""
import math

import pytest
import torch

from test_gpu_token_losses import (DTYPES, U, check_gradient, floats, ints, logp_tol, near, one, policy64, preference64, rows_of,
                                   stats64)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ KL term

@pytest.mark.parametrize("classes", [50, 5001])
def test_kl_term_keeps_its_digits_next_to_the_reference(classes):
    """kl = exp(x) - x - 1 with x = ref - logp as floats, from |x| = 1e-7 to 80: eight roundings of a series or twelve of a
    difference.  No advantage, so that the loss is the KL term alone."""
    from renaissance_b200 import ops
    size = [s * 10.0 ** -k * m for k in range(8) for m in (1.0, 2.5, 4.9, 5.1) for s in (1, -1)] + [20.0, -20.0, 80.0, -80.0, 0.0]
    rows = len(size)
    z, y = rows_of(rows, classes, torch.float32, seed=1), ints(rows, classes)
    logp = ops.token_logprobs(z, y)["logp"]
    ref = logp + torch.tensor(size, device="cuda")
    zero, w = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    out = ops.policy_loss_fused(z, y, logp, zero, one(1.0), ref_logp=ref, kl_coef=1.0, weights=w)
    assert torch.equal(out["logp"], logp)
    x = (ref - logp).double()
    series = torch.where(x.abs() < 1e-2, x * x * (0.5 + x / 6 + x * x / 24 + x ** 3 / 120 + x ** 4 / 720), torch.expm1(x) - x)
    near(out["loss_partial"], series, 20 * U * series, "kl")
    assert (out["loss_partial"][x == 0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [50, 5001])
def test_kl_term_of_an_impossible_class_is_infinite(dtype, classes):
    """logp = -inf (a masked class was chosen): exp(ref - logp) - (ref - logp) - 1 grows without bound, it is not NaN.  The
    same where the reference gives the class no chance, and where the exponential overflows."""
    from renaissance_b200 import ops
    z, y = rows_of(4, classes, dtype, seed=2), torch.zeros(4, dtype=torch.int32, device="cuda")
    z[1, 0] = -math.inf
    logp = ops.token_logprobs(z, y)["logp"]
    ref = logp.clone()
    ref[1], ref[2], ref[3] = -3.0, -math.inf, float(logp[3]) + 100.0
    out = ops.policy_loss_fused(z, y, logp.clamp_min(-5.0), torch.ones(4, device="cuda"), one(1.0), ref_logp=ref, kl_coef=0.1)
    assert math.isfinite(float(out["loss_partial"][0])) and (out["loss_partial"][1:] == math.inf).all()
    assert float(out["loss"]) == math.inf


# ------------------------------------------------------------------------------------------------ preference loss

@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
def test_preference_loss_of_an_impossible_answer(eps):
    """A label whose logit is minus infinity makes S = -inf.  In the other answer x = +inf: the loss is eps * inf, without
    smoothing 0; in the preferred one x = -inf and the loss is (1 - eps) * inf.  Gradients are finite, the other pair's
    numbers the formula's."""
    from renaissance_b200 import ops
    z, y = rows_of(8, 300, torch.float32, seed=4), ints(8, 300)
    logp, _ = stats64(z, y)
    st = torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32, device="cuda")
    x = 0.5 * (logp[4:6].sum() - logp[6:8].sum())
    soft = lambda v: torch.nn.functional.softplus(v)
    other = ((1 - eps) * soft(-x) + eps * soft(x)) / 2
    for row, sign in ((3, 1), (0, -1)):
        w = z.clone()
        w[row, int(y[row])] = -math.inf
        out = ops.preference_loss_fused(w, y, st, None, one(1.0), 0.5, eps)
        part = out["loss_partial"].tolist()
        factor = eps if sign > 0 else 1 - eps
        assert part[0] == (math.inf if factor else 0.0)
        tol = 0.5 * float(logp_tol(logp, logp)[4:].sum()) + 8 * U
        assert abs(part[1] - float(other)) <= tol
        assert float(out["loss"]) == (math.inf if factor else part[1])
        assert out["dlogits"].isfinite().all()
        pull = 0.5 / 2 * (eps if sign > 0 else -(1 - eps))      # beta / pairs * (eps sigmoid(x) - (1 - eps) sigmoid(-x))
        coef = torch.tensor([pull, pull, -pull, -pull], dtype=torch.float64, device="cuda")
        lse = stats64(w, y)[1]
        check_gradient(out["dlogits"][:4], w[:4], y[:4], coef, 2 * U * coef.abs(), U * (150 + 4 * lse.abs())[:4])


# ------------------------------------------------------------------------------------------------ large logits

# shifts of a row's logits, and factors: maxima on both sides of 256 and of 2^100, ordinary rows among them
MOVES = {torch.float16: [(0, 1), (245, 1), (-262, 1), (300, 1), (-1000, 1), (6e4, 1), (0, 100), (-6e4, 1), (0, 1), (250, 1)],
         torch.bfloat16: [(0, 1), (245, 1), (-262, 1), (300, 1), (-1000, 1), (1e30, 1), (0, 1e30), (-1e30, 1), (0, 100), (250, 1),
                          (3e38, 1), (-3e38, 1), (1e28, 1)]}
MOVES[torch.float32] = MOVES[torch.bfloat16] + [(1e4, 1), (-1e4, 3)]
FAR_CLASSES = [1, 9, 100, 200, 300, 450, 700, 1000, 1501, 2048, 2057, 5001, 16400, 33001, 70003, 140000]


def far_rows(rows, classes, dtype, pad, skip, seed):
    """(logits, labels, the same logits in 64 bits minus their row's maximum: the same distribution)."""
    z = rows_of(rows, classes, dtype, pad, skip, seed)
    y = ints(rows, classes, seed + 1)
    for i in range(rows):
        shift, factor = MOVES[dtype][i % len(MOVES[dtype])]
        z[i] = (z[i].double() * factor + shift).to(dtype)
        if factor > 1:
            y[i] = int(z[i].float().argmax())               # any other class would have no chance at all
    w = z.double()
    return z, y, w - w.amax(1, keepdim=True)


def spare_columns(rows, classes, dtype):
    """A gradient buffer inside a wider one, at an odd alignment."""
    flat = torch.full((1 + rows * (classes + 3) + 8,), 7.0, dtype=dtype, device="cuda")
    return flat, torch.as_strided(flat, (rows, classes), (classes + 3, 1), 1)


def kept_off(flat, d):
    d.fill_(7.0)
    return bool((flat == 7.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", FAR_CLASSES)
def test_policy_loss_with_large_logits(dtype, classes):
    """A distribution does not change when all its logits move: loss and gradient to the tolerances of the logits minus
    their maximum.  Up to 256 the 16-bit gradient's exponent is rounded at the logits' own size, 2^-16 of the result."""
    from renaissance_b200 import ops
    rows = 2 * len(MOVES[dtype])
    for pad, skip, given in ((0, 0, False), (5, 1, True)):
        z, y, zero = far_rows(rows, classes, dtype, pad, skip, 7)
        logp, log_sum = stats64(zero, y)
        moved = torch.where(floats(rows, 9) < 0, -0.1, 0.1).double()
        old, ref = (logp - moved).float(), (logp + 0.2).float()
        adv, w = floats(rows, 11), floats(rows, 12).abs() + 0.1
        flat, d = spare_columns(rows, classes, dtype) if given else (None, None)
        out = ops.policy_loss_fused(z, y, old, adv, one(64.0), 0.2, 0.28, ref, 0.05, w, dlogits=d)
        part, want, coef, part_tol, t, coef_tol = policy64(zero, y, old, adv, ref, w, 0.2, 0.28, 0.05, 64.0)
        near(out["logp"], want, t, "logp")
        near(out["loss_partial"], part, part_tol, "loss_partial")
        check_gradient(out["dlogits"], zero, y, coef, coef_tol, t + 2.0 ** -16 * (dtype != torch.float32))
        got = ops.token_logprobs(z, y)
        assert torch.equal(got["logp"], out["logp"])
        near(got["lse"], log_sum + z.double().amax(1), t + U * (log_sum + z.double().amax(1)).abs(), "lse")
        assert not given or (out["dlogits"].data_ptr() == d.data_ptr() and kept_off(flat, d))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", FAR_CLASSES)
def test_preference_loss_with_large_logits(dtype, classes):
    from renaissance_b200 import ops
    rows = 2 * len(MOVES[dtype])
    starts = [0, 3, rows // 2, rows // 2, rows - 1]
    for pad, skip, given in ((0, 0, False), (5, 1, True)):
        z, y, zero = far_rows(rows, classes, dtype, pad, skip, 5)
        y[1] = -1
        flat, d = spare_columns(rows, classes, dtype) if given else (None, None)
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        S = preference64(zero, y, starts, None, 0.1, 0.1, 64.0)[2]
        ref = (S + floats(4, 3)).float()
        out = ops.preference_loss_fused(z, y, st, ref, one(64.0), 0.1, 0.1, dlogits=d)
        part, part_tol, S, S_tol, logp, t, coef, coef_tol = preference64(zero, y, starts, ref, 0.1, 0.1, 64.0)
        near(out["logp"], logp, t, "logp")
        near(out["seq_logp"], S, S_tol, "seq_logp")
        near(out["loss_partial"], part, part_tol, "loss_partial")
        check_gradient(out["dlogits"], zero, y, coef, coef_tol, t + 2.0 ** -16 * (dtype != torch.float32))
        assert not given or kept_off(flat, d)


# ------------------------------------------------------------------------------------------------ rows that move

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("classes", [9, 100, 777, 1001, 2047, 2049, 5001, 33001, 50021])
def test_a_row_that_moves_keeps_its_logp_to_its_alignment(dtype, classes):
    """The same rows in another order, at other strides and offsets: bit for bit the same where a row's address modulo 16
    bytes is, a ratio of exactly 1 in the loss among it; elsewhere within twice what one sum may be off by."""
    from renaissance_b200 import ops
    rows, item = 48, torch.finfo(dtype).bits // 8
    wide = 16 // item
    z, y = rows_of(rows, classes, dtype, seed=3), ints(rows, classes)
    first = ops.token_logprobs(z, y)
    where = lambda t: (t.data_ptr() + torch.arange(rows, device="cuda") * t.stride(0) * item) % 16
    tol = 2 * logp_tol(*stats64(z, y))
    order = torch.randperm(rows, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    moves = 0
    for pad, skip, perm in ((0, 0, order), (-classes % wide, 0, order), (5, 1, order), (0, wide, order), (wide, 3, torch.arange(rows, device="cuda"))):
        w = rows_of(rows, classes, dtype, pad, skip)
        w.copy_(z[perm])
        got = ops.token_logprobs(w, y[perm])
        same = where(w) == where(z)[perm]
        moves += int((~same).sum())
        for k in ("logp", "lse"):
            assert torch.equal(got[k][same], first[k][perm][same])
            assert ((got[k].double() - first[k][perm].double()).abs() <= tol[perm]).all()
        adv = floats(rows, 5)
        out = ops.policy_loss_fused(w, y[perm], first["logp"][perm], adv, one(1.0), weights=torch.ones(rows, device="cuda"))
        assert torch.equal(out["logp"], got["logp"])
        assert torch.equal(out["loss_partial"][same], -adv[same])
    # an aligned stride keeps every row's alignment, wherever it goes
    a, b = (rows_of(rows, classes, dtype, -classes % wide, s) for s in (0, 2 * wide))
    a.copy_(z)
    b.copy_(z[order])
    assert torch.equal(ops.token_logprobs(b, y[order])["logp"], ops.token_logprobs(a, y)["logp"][order])
    assert moves > 0


# ------------------------------------------------------------------------------------------------ digits of the ratio

@pytest.mark.parametrize("classes", [16, 1000, 5001])
def test_ratio_has_more_digits_than_the_stored_logp(classes):
    """Five classes near the maximum, the chosen one 100 below it, nothing else: log s is good to 10 u (five exponentials of
    4 u, nine additions and merges that change nothing but add to one another), the float that logp is stored as to 64 u.
    Of the ratio: 10 u, 1 u for log s and for the difference, 4 u for its exponential, 3 u of products."""
    from renaissance_b200 import ops
    rows = 256
    z = torch.full((rows, classes), -math.inf, device="cuda")
    z[:, :5] = 3.0 + rows_of(rows, 5, torch.float32, seed=1, spread=0.3)
    z[:, 9] = -97.0 + floats(rows, 2)
    y = torch.full((rows,), 9, dtype=torch.int32, device="cuda")
    logp, _ = stats64(z, y)
    old = (logp + 0.1 * floats(rows, 3).double()).float()
    adv, w = -torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda")         # no upper bound for a loss
    out = ops.policy_loss_fused(z, y, old, adv, one(1.0), 1.0, 10.0, weights=w)
    ratio = torch.exp(logp - old.double())
    near(out["loss_partial"], ratio, 20 * U * ratio, "ratio")
    # a policy that has not moved
    out = ops.policy_loss_fused(z, y, out["logp"], adv, one(1.0), 1.0, 10.0, weights=w)
    assert (out["loss_partial"] == 1).all()
    z[3, 9] = z[4, 7] = -math.inf                           # impossible now as it was then: no ratio; z[4] is as before
    old = ops.token_logprobs(z, y)["logp"]
    out = ops.policy_loss_fused(z, y, old, adv, one(1.0), 1.0, 10.0, weights=w)
    assert out["loss_partial"][3].isnan() and (out["loss_partial"][4:] == 1).all()
    z[5, 2], z[6, 1] = math.nan, math.inf
    out = ops.policy_loss_fused(z, y, torch.full_like(old, -100.0), adv, one(1.0), 1.0, 10.0, weights=w)
    assert out["loss_partial"][5:7].isnan().all() and out["loss_partial"][7:].isfinite().all()
