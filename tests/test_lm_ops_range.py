"""Layer normalisation near the ends of the number range: both memory layouts
give what the formula gives wherever fp32 holds the formula's own steps, and the
same infinities where it does not.  Distillation at the ends of its temperatures."""
import numpy as np
import pytest

from test_lm_ops import BF16, F16, F32, check_distill, check_ln, distill_inputs, ln_inputs, place, quantise, run_distill, run_ln, vec

pytestmark = pytest.mark.gpu

# features: fewer than the lanes that share a column, a whole strip in registers, runs of features
FEATURES = [1, 5, 33, 300, 1500, 2500]


def far_positions(n, f, name):
    """positions around 3e19, whose square is more than fp32 holds, one or two
    steps of bf16 apart; the first one without any spread"""
    x, dy, gamma, beta = ln_inputs(n, f, name)
    step = 2.0 ** 57
    x = quantise(208 * step + np.rint(x) * step, name)
    x[0] = 208 * step
    return x, dy, gamma, beta


@pytest.mark.parametrize("name", [F32, BF16])
@pytest.mark.parametrize("f", FEATURES)
def test_means_whose_square_overflows(hip, f, name):
    x, dy, gamma, beta = far_positions(9, f, name)
    for axis in (0, 1):
        for how in ("plain", "turned"):
            check_ln(run_ln(hip, x, dy, gamma, beta, axis, how, name), x, dy, gamma, beta, name)


@pytest.mark.parametrize("f", FEATURES)
def test_infinite_means_and_variances(hip, f):
    """what is stored of a position that holds infinities, or whose variance is
    more than fp32 holds, does not depend on the layout"""
    n, be = 6, hip
    x, _, gamma, beta = ln_inputs(n, f, F32)
    x[1, 0], x[2, f // 2], x[3, f - 1] = np.inf, -np.inf, np.nan
    if f > 1:
        x[4, 0], x[4, f - 1] = np.inf, -np.inf
        x[5] = np.where(np.arange(f) % 2, 1e20, -1e20)
    for axis in (0, 1):
        for how in ("plain", "turned"):
            tx, ty = place(be, x, axis, how, F32), place(be, (n, f), axis, how, F32)
            mean, var = (be.empty((1, n) if axis == 0 else (n, 1)) for _ in range(2))
            be.compound_fprop_ln(tx, mean, var, vec(be, gamma, axis), vec(be, beta, axis), ty, 1e-5, axis=axis)
            y, mean, var = (t.get() for t in (ty, mean, var))
            y, mean, var = (y.T if axis == 0 else y), mean.ravel(), var.ravel()
            assert mean[1] == np.inf and mean[2] == -np.inf and np.isnan(mean[3])
            assert np.isnan(var[1:4]).all() and np.isnan(y[1:4]).all() and np.isfinite(y[0]).all()
            if f > 1:
                assert np.isnan(mean[4]) and np.isnan(var[4]) and np.isnan(y[4]).all()
                # an infinite variance: 1 / std is 0
                assert abs(mean[5]) <= 1e20 and var[5] == np.inf and np.array_equal(y[5], beta[0].astype(np.float32))



@pytest.mark.parametrize("spread,size", [(1e15, 1e25), (1e-15, 1e-25)])
@pytest.mark.parametrize("f", [5, 300, 1500, 2500])
def test_gradients_where_deviation_times_error_leaves_the_range(hip, f, spread, size):
    """(x - mean) dy alone is outside fp32, the normalised deviation times dy is not"""
    x, dy, gamma, beta = ln_inputs(9, f, F32, shift=0.0)
    x, dy = quantise(x * spread, F32), quantise(dy * size, F32)
    eps = 1e-5 if spread > 1 else float(np.float32(1e-36))
    for axis in (0, 1):
        for how in ("plain", "turned"):
            check_ln(run_ln(hip, x, dy, gamma, beta, axis, how, F32, eps), x, dy, gamma, beta, F32, eps)


@pytest.mark.parametrize("name", [F32, F16, BF16])
@pytest.mark.parametrize("tau", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
def test_distillation_at_the_ends_of_its_temperatures(hip, tau, name):
    z, ids, t, weight = distill_inputs(9, 700, 11, name, name)
    if name == F16:
        weight = weight / max(tau, 1.0)                 # (gradients that the type holds)
    for axis in (0, 1):
        check_distill(run_distill(hip, z, ids, t, weight, tau, axis, "plain", name, name), z, ids, t, weight, tau, name)
