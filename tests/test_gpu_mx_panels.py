"""Products whose weights are more than one panel of the pair kernel's tile order (32 MB of codes): Dense and gated, a narrower last
panel, fewer tiles than pairs and several tiles to a pair.  Sums are exact: codes up to 4 and scales of 2^-1 .. 2^1 make products that are
multiples of 2^-4 of at most 64, and 8200 of them stay below 2^24 such units."""

import numpy as np
import pytest

import mx_reference as R
from test_gpu_mx import Mx, Out, dev32, lib, run_dense, run_gated, torch  # noqa: F401  (lib is the fixture)

pytestmark = pytest.mark.gpu


def operand(rng, rows, cols):
    codes = rng.integers(0, 7, (rows, cols)).astype(np.uint8) | (rng.integers(0, 2, (rows, cols)).astype(np.uint8) << 3)
    return Mx(codes, rng.integers(126, 129, (rows, R.ceil_div(cols, 32))).astype(np.uint8), spare=0)


def on_device(q):
    t = torch()
    v = t.from_numpy(R.VALUES).cuda()[t.from_numpy(q.np_codes).cuda().int()]
    scale = t.exp2(t.from_numpy(q.np_scales).cuda().double() - 127)
    return v * scale.repeat_interleave(32, 1)[:, :q.cols]


@pytest.mark.parametrize('m,k,n', [(300, 8200, 8500),      # 68 tiles of Dense: panels of 31 and 3 columns of tiles, fewer tiles than pairs
                                   (1030, 8200, 8200),     # 165 tiles of Dense: panels of 31 and 2, two and three tiles to a pair
                                   (140, 4100, 33100)])    # panels of 60, 60 and 10
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('kind', ['f32', 'mx'])
def test_panels(lib, m, k, n, gated, kind):  # noqa: F811
    rng = np.random.default_rng(m + n + gated)
    a, w = operand(rng, m, k), operand(rng, n, k)
    b = rng.integers(-1024, 1025, n) / 16.0
    bias = dev32(b)
    x = on_device(a)
    want = (x @ on_device(w).T + bias.double()).cpu().numpy()
    out = Out(kind, m, n)
    if gated:
        u = operand(rng, n, k)
        want = (want.astype(np.float32) * (x @ on_device(u).T).float().cpu().numpy()).astype(np.float64)
        run_gated(lib, a, w, u, bias, None, out, 'none')
    else:
        run_dense(lib, a, w, bias, out, 0)
    got = out.get()
    assert lib.device_status() == 0
    if kind == 'mx':
        codes, scales = (np.concatenate(p) for p in zip(*(R.quantize(want[i:i + 64]) for i in range(0, m, 64))))
        assert np.array_equal(got[1], scales)
        assert np.array_equal(R.values(*got), R.values(codes, scales))
    else:
        assert np.array_equal(got, want)
