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
