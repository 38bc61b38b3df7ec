"""The graph oracle's MXFP4 rounding and the host packing against the definition, where either can go wrong (CPU)."""

import numpy as np
import pytest

import mx_reference as R
from aie4ml_b200.quant_utils import from_mx, to_mx
from oracle import oracle


@pytest.mark.parametrize('what', [np.nan, np.inf, -np.inf])
def test_oracle_makes_the_whole_block_nan(what):
    x = np.random.default_rng(0).standard_normal((4, 80))
    x[1, 40], x[2, 0], x[2, 79] = what, what, what
    got = oracle.mx_round(x)
    assert np.array_equal(got, R.values(*R.quantize(x)), equal_nan=True)
    assert np.isnan(got[1, 32:64]).all() and not np.isnan(got[1, :32]).any() and np.isnan(got[2, 64:]).all()


def test_oracle_next_to_powers_of_two():
    """One step of float64 below a power of two the logarithm rounds up to it; the exponent must not."""
    x = np.zeros((60, 32))
    x[:, 0] = np.nextafter(np.exp2(np.arange(60) - 30.0), 0.0)
    x[:, 1] = np.exp2(np.arange(60) - 32.0) * 1.25
    assert np.array_equal(oracle.mx_round(x), R.values(*R.quantize(x)))
    assert np.array_equal(oracle.mx_round(2 * x), 2 * oracle.mx_round(x))


def test_oracle_keeps_shapes_and_small_values():
    x = np.random.default_rng(1).standard_normal((2, 3, 50)) * 2.0 ** -126
    x[1, 2] = 0.0
    want = R.values(*R.quantize(x.reshape(-1, 50))).reshape(x.shape)
    assert np.array_equal(oracle.mx_round(x), want)


@pytest.mark.parametrize('value', [2.0 ** 128, -2.0 ** 130, 1e39, 2.0 ** 131, 1e40, -1e60, 1e300])
def test_host_packing_beyond_float32(value):
    """No scale byte stands for a block that large: NaN, as the kernel makes of the infinity that a float32 holds of it."""
    x = np.random.default_rng(2).standard_normal((3, 70))
    x[1, 33] = value
    codes, tiles = to_mx(x)
    with np.errstate(over='ignore'):
        want = R.quantize(x.astype(np.float32).astype(np.float64))
    got = from_mx(codes, tiles, 3, 70)
    assert np.isnan(got[1, 32:64]).all() and np.isfinite(got[1, :32]).all()
    assert np.array_equal(tiles, R.tile_scales(want[1], 70))


def test_host_packing_up_to_the_largest_float32():
    x = np.zeros((2, 32))
    x[0, :3] = np.finfo(np.float32).max, -np.finfo(np.float32).max, 1e38
    x[1, 0] = 2.0 ** 127
    codes, tiles = to_mx(x)
    want = R.quantize(x)
    assert (want[1] < 255).all() and np.array_equal(tiles, R.tile_scales(want[1], 32))
    assert np.array_equal(from_mx(codes, tiles, 2, 32), R.values(*want).astype(np.float32))
