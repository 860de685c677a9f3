"""The token losses where a formula taken as it stands loses its digits, or where a row leaves the ordinary range.  The
definitions in 64 bits, and how tolerances are counted, are those of test_gpu_token_losses."""
import math

import pytest
import torch

from test_gpu_token_losses import DTYPES, U, check_gradient, floats, ints, logp_tol, near, one, rows_of, stats64

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
