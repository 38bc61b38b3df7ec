"""The activations of the gated Dense at chosen arguments, relative to the result.

Weights of zero leave act(bias_g[n]) * bias_u[n], so the argument is any float32 value and no sum rounds.  The tolerances count,
for x the argument and t the exponential's: two roundings of the factor before the exponential and at most seven of t for the tanh
form (4 |t| 2^-23), two for the others (|t| 2^-23); 2^-22 for the exponential, 2^-23 for the reciprocal, 2^-24 each for the sum, the product
with x, the product with the other factor: (|t| or 4 |t|) + 5 units of 2^-23.  A reciprocal below 2^-126 may be 0.
GELU is max(x, 0) - a 2^Q(a): 3.1e-8 for the polynomial (2^-9 of the result down to -6 where that is less), half a unit of each of the
Horner sums, 2^-22 for the exponential, half a unit of the result and of the product."""

import numpy as np
import pytest

from test_gpu_mx import ACTS, Mx, Out, dev32, lib, run_gated  # noqa: F401  (lib is the fixture)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def rounded(x):
    return np.asarray(x, dtype=np.float32).astype(np.float64)


def arguments():
    x = np.concatenate([np.linspace(-14, 14, 2801), np.linspace(-110, 110, 441), -np.exp2(np.linspace(-40, 6, 461)), np.exp2(np.linspace(-40, 6, 461)),
                        [0.0, -0.0, 1e-38, -1e-38, 1e-42, 300.0, -300.0, 1e6, -1e6, 3e38, -3e38]])
    return rounded(x)


def exact(x, act):
    from scipy.special import expit, log_ndtr

    with np.errstate(over='ignore'):
        if act == 'silu':
            return x * expit(x)
        if act == 'sigmoid':
            return expit(x)
        if act == 'gelu':
            return x * np.exp(log_ndtr(x))
        return x * expit(2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3))


def exponent_roundings(x):
    """Half a unit of every Horner sum of log2 Phi(-a), carried to the end: an absolute error of the exponent.  The sums are those
    of the parabola-like series itself, so its leading terms say how large they are: below 0.46 a^2 + 1.16 a + 1, whatever the order."""
    a = np.minimum(np.abs(x), 64.0)
    return 9 * U * (0.47 * a * a + 1.16 * a + 1)


def tolerance(x, act, want):
    """for a factor of 1 behind the activation"""
    if act == 'gelu':
        a = np.abs(x)
        power = np.abs(np.where(x < 0, want, want - x))               # a Phi(-a)
        poly = np.where((x <= 0) & (x >= -6), np.minimum(3.1e-8, 2.0 ** -9 * power), 3.1e-8)
        tail = np.where(a > 13, power, 0.0)                          # the power is 0 there
        return poly + tail + power * (2.0 ** -22 + np.log(2) * exponent_roundings(x)) + 2 * U * np.abs(want) + 2.0 ** -126
    t = np.abs(x) if act != 'gelu_tanh' else np.abs(1.6 * (x + 0.044715 * x ** 3))
    per = 4 if act == 'gelu_tanh' else 1
    rel = np.minimum((per * t + 5) * 2.0 ** -23, 1.0)
    return rel * np.abs(want) + 2.0 ** -126 * (1.0 if act == 'sigmoid' else 1 + np.abs(x))


def gated_of(lib, x, factor, act, kind, m):
    n, k = x.size, 32
    zero = Mx(np.zeros((n, k), dtype=np.uint8), np.full((n, 1), 127, dtype=np.uint8))
    a = Mx(np.full((m, k), 2, dtype=np.uint8), np.full((m, 1), 127, dtype=np.uint8))
    out = Out(kind, m, n)
    run_gated(lib, a, zero, zero, dev32(x), dev32(factor), out, act)
    got = out.get()
    assert lib.device_status() == 0
    assert all(np.array_equal(got[0], row, equal_nan=True) for row in got[1:])
    return got[0]


@pytest.mark.parametrize('act', ['silu', 'sigmoid', 'gelu', 'gelu_tanh'])
@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('m', [3, 300])         # both kernels
def test_activation_relative_to_its_result(lib, act, kind, m):  # noqa: F811
    x = arguments()
    want = exact(x, act)
    got = gated_of(lib, x, np.ones_like(x), act, kind, m)
    tol = tolerance(x, act, want)
    if kind == 'bf16':
        tol = tol + (np.abs(want) + tol) * 2.0 ** -8
    far = np.abs(got - want) > tol
    assert not far.any(), [(x[i], got[i], want[i], tol[i]) for i in np.flatnonzero(far)[:8]]


@pytest.mark.parametrize('m', [3, 300])
def test_gelu_keeps_a_bfloat16_step_down_to_minus_six(lib, m):  # noqa: F811
    """The polynomial's 2^-9 of the result, the exponential's and the exponent's roundings, and half a step of bfloat16."""
    x = rounded(np.linspace(-6, -0.5, 4000))
    want = exact(x, 'gelu')
    got = gated_of(lib, x, np.ones_like(x), 'gelu', 'bf16', m)
    rel = 2.0 ** -9 + 2.0 ** -22 + np.log(2) * exponent_roundings(x) + 2 * U
    assert (np.abs(got - want) <= np.abs(want) * (rel + 2.0 ** -8 * (1 + rel))).all()


@pytest.mark.parametrize('act', ['silu', 'sigmoid', 'gelu', 'gelu_tanh'])
@pytest.mark.parametrize('m', [3, 300])
def test_activation_times_a_factor(lib, act, m):  # noqa: F811
    rng = np.random.default_rng(ACTS.index(act))
    x, u = rounded(rng.normal(0, 4, 3000)), rounded(rng.normal(0, 1, 3000) * np.exp2(rng.integers(-20, 20, 3000)))
    want = exact(x, act)
    got = gated_of(lib, x, u, act, 'f32', m)
    tol = (tolerance(x, act, want) + U * np.abs(want)) * np.abs(u)
    assert (np.abs(got - want * u) <= tol).all()


@pytest.mark.parametrize('m', [3, 300])
def test_infinite_and_nan_arguments(lib, m):  # noqa: F811
    x = np.array([np.inf, -np.inf, np.nan, 1.0] * 500)
    for act, want in (('sigmoid', [1.0, 0.0, np.nan]), ('gelu', [np.inf, 0.0, np.nan]), ('relu', [np.inf, 0.0, np.nan]), ('none', [np.inf, -np.inf, np.nan]),
                      ('silu', [np.inf, np.nan, np.nan])):      # x / (1 + exp(-x)) at -infinity is a quotient of infinities
        got = gated_of(lib, x, np.ones_like(x), act, 'f32', m)
        assert np.array_equal(got[:3], np.array(want), equal_nan=True), act
        assert np.array_equal(got, np.tile(got[:4], 500), equal_nan=True), act
