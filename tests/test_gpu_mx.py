"""MXFP4 operators on the GPU against their definition in 64 bits.

Quantisation is exact, so codes, scales and the places around them are compared for equality.  Products are compared for
equality too wherever every partial sum is exact in float32 whatever its order: with scales of 2^-1 .. 2^1 the products are
multiples of 2^-4 below 144, and 4096 of them stay below 2^24 such units.  Elsewhere the tolerance counts roundings:
K + 2 additions of at most 2^-23 (truncation) of the sum of magnitudes, and half a step of the output type.
"""

import numpy as np
import pytest

import mx_reference as R

pytestmark = pytest.mark.gpu

F = {'bf16': 0, 'f32': 1, 'mx': 3}
ACTS = ['none', 'relu', 'silu', 'gelu', 'gelu_tanh', 'sigmoid']


@pytest.fixture(scope='module')
def lib():
    from aie4ml_b200 import lib as a4c

    return a4c


def torch():
    import torch

    return torch


def stream():
    return torch().cuda.current_stream().cuda_stream


def up(n, to=32):
    return -(-n // to) * to


class Mx:
    """An operand on the device; the pitch holds spare columns full of ones and the rows behind the last have NaN scales."""

    def __init__(self, codes, scales, spare=32):
        t = torch()
        self.rows, self.cols = codes.shape
        self.pitch = up(self.cols) + spare
        self.np_codes, self.np_scales = codes, scales
        self.codes = t.from_numpy(R.pack_codes(codes, self.pitch, fill=0x77)).cuda()
        self.scales = t.from_numpy(R.tile_scales(scales, self.cols, row_fill=255)).cuda()

    @property
    def args(self):
        return self.codes.data_ptr(), self.pitch, self.scales.data_ptr()

    @property
    def values(self):
        return R.values(self.np_codes, self.np_scales)


def random_mx(rng, rows, cols, lo=126, hi=128, spare=32):
    return Mx(rng.integers(0, 16, (rows, cols)).astype(np.uint8), rng.integers(lo, hi + 1, (rows, R.ceil_div(cols, 32))).astype(np.uint8), spare)


def bf16_round(x):
    """float64 (exact in float32) -> nearest bfloat16 values"""
    return torch().from_numpy(np.asarray(x, dtype=np.float32)).bfloat16().float().numpy().astype(np.float64)


class Out:
    """An output with guard rows and columns around it, all of which must survive."""

    def __init__(self, kind, rows, cols):
        t = torch()
        self.kind, self.rows, self.cols = kind, rows, cols
        # float outputs: every third has a pitch that no wide store can use
        self.ld = up(cols) + 32 if kind == 'mx' else cols + 3 if (rows + cols) % 3 == 0 else up(cols, 8) + 8
        width = self.ld // 2 if kind == 'mx' else self.ld
        dtype = {'mx': t.uint8, 'bf16': t.bfloat16, 'f32': t.float32}[kind]
        self.buf = t.full((rows + 2, width), 0x55 if kind == 'mx' else -7.0, dtype=dtype, device='cuda')
        self.scales = t.full((R.ceil_div(rows, 128) * R.ceil_div(cols, 128) * 512,), 0xEE, dtype=t.uint8, device='cuda') if kind == 'mx' else None

    @property
    def args(self):
        return self.buf[1:].data_ptr(), F[self.kind], self.ld, self.scales.data_ptr() if self.scales is not None else None

    def get(self):
        torch().cuda.synchronize()
        guard = 0x55 if self.kind == 'mx' else -7.0
        b = self.buf.float().cpu().numpy() if self.kind != 'mx' else self.buf.cpu().numpy()
        used = R.ceil_div(self.cols, 2) if self.kind == 'mx' else self.cols
        assert (b[0] == guard).all() and (b[-1] == guard).all() and (b[1:-1, used:] == guard).all(), 'written beyond the output'
        body = b[1:-1, :used]
        if self.kind != 'mx':
            return body.astype(np.float64)
        codes = np.stack([body & 15, body >> 4], axis=2).reshape(self.rows, -1)
        assert (codes[:, self.cols:] == 0).all()
        tiled = self.scales.cpu().numpy()
        scales = R.untile_scales(tiled, self.rows, R.ceil_div(self.cols, 128) * 128)
        blocks = R.ceil_div(self.cols, 32)
        assert (scales[:, blocks:] == 0).all(), 'blocks beyond the row end'
        return codes[:, :self.cols], scales[:, :blocks]


# ---- quantisation -------------------------------------------------------------------------------

def awkward(rng, rows, cols):
    """Normal values over many binades, exact ties, zeros of both signs, subnormals, and blocks with NaN and infinity."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-130, 120, (rows, 1)))
    flat = x.reshape(-1)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0])
    n = flat.size
    pick = rng.random(n)
    base = np.exp2(rng.integers(-20, 20, (rows, 1)) * np.ones((1, cols))).reshape(-1)
    flat[:] = np.where(pick < 0.3, ties[rng.integers(0, 10, n)] * base, flat)
    flat[:] = np.where((pick > 0.3) & (pick < 0.35), -0.0, flat)
    if rows > 4:
        x[1] = 0.0
        x[2] = 2.0 ** -127 * np.round(rng.standard_normal(cols) * 8) / 8
        x[3, : max(1, cols // 3)] = np.nan
        x[4, -1] = np.inf
    return x


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 31), (1, 33), (1, 4096), (5, 256), (127, 128), (129, 257), (777, 1000), (300, 8191)])
@pytest.mark.parametrize('offset', [0, 1])
def test_quantize(lib, dtype, rows, cols, offset):
    t = torch()
    rng = np.random.default_rng(rows * 131 + cols)
    td = {'bf16': t.bfloat16, 'f32': t.float32}[dtype]
    ldx = up(cols, 8) + (8 if offset == 0 else 5)        # offset 1: neither base nor pitch allow wide loads
    store = t.full((rows * ldx + 8,), float('nan'), dtype=td, device='cuda')
    x = store[offset:offset + rows * ldx].view(rows, ldx)
    x[:, :cols] = t.from_numpy(awkward(rng, rows, cols)).to(td).cuda()
    want_codes, want_scales = R.quantize(x[:, :cols].double().cpu().numpy())
    out = Out('mx', rows, cols)
    ptr, _, ld, sc = out.args
    lib.check(lib.load().a4c_quantize_mx(x.data_ptr(), F[dtype], ldx, ptr, ld, sc, rows, cols, stream()), 'quantize')
    codes, scales = out.get()
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)
    tiled = out.scales.cpu().numpy()
    assert np.array_equal(tiled, R.tile_scales(want_scales, cols)), 'rows beyond the last are written as 0'
    back = Out(dtype, rows, cols)
    ptr_b, f, ld_b, _ = back.args
    lib.check(lib.load().a4c_dequantize_mx(ptr, ld, sc, ptr_b, f, ld_b, rows, cols, stream()), 'dequantize')
    got, want = back.get(), R.values(want_codes, want_scales)
    assert np.array_equal(got, want, equal_nan=True)
    wide = t.empty(rows, up(cols, 8), dtype=td, device='cuda')          # the wide stores
    lib.check(lib.load().a4c_dequantize_mx(ptr, ld, sc, wide.data_ptr(), f, up(cols, 8), rows, cols, stream()), 'dequantize')
    assert np.array_equal(wide[:, :cols].double().cpu().numpy(), want, equal_nan=True)


def test_quantize_is_a_projection(lib):
    """What has been quantised comes back as it is, from either type."""
    t = torch()
    rng = np.random.default_rng(5)
    q = random_mx(rng, 200, 320, 3, 250)
    q.np_codes[:, ::32] = 7                        # every block reaches its top binade
    q = Mx(q.np_codes, q.np_scales)
    for td, f in ((t.bfloat16, 0), (t.float32, 1)):
        y = t.empty(200, 320, dtype=td, device='cuda')
        lib.check(lib.load().a4c_dequantize_mx(*q.args, y.data_ptr(), f, 320, 200, 320, stream()), 'dequantize')
        out = Out('mx', 200, 320)
        lib.check(lib.load().a4c_quantize_mx(y.data_ptr(), f, 320, out.args[0], out.ld, out.args[3], 200, 320, stream()), 'quantize')
        codes, scales = out.get()
        assert np.array_equal(codes, q.np_codes) and np.array_equal(scales, q.np_scales)


# ---- Dense --------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 32, 16), (3, 33, 5), (1, 4096, 200), (16, 64, 128), (17, 65, 129), (31, 255, 33), (64, 256, 256), (100, 257, 96),
          (128, 512, 384), (129, 1000, 777), (200, 130, 1024), (256, 2048, 256), (333, 1000, 65), (385, 4096, 640),
          (190, 300, 1100), (531, 224, 1129)]


# enough tiles of 256 x 256 (and of 256 x 128 pairs of features) that a CTA pair works through several
WIDE = [(1030, 300, 2600), (2600, 64, 5000), (3001, 520, 4500), (300, 257, 9700)]


def run_dense(lib, a, w, bias, out, relu):
    lib.check(lib.load().a4c_dense_mx(*a.args, *w.args, bias.data_ptr() if bias is not None else None, *out.args, a.rows, a.cols, w.rows, relu,
                                      stream()), 'dense')


def exact_bias(rng, n):
    """multiples of 1/16 up to 64: the sums stay exact"""
    return rng.integers(-1024, 1025, n) / 16.0


@pytest.mark.parametrize('m,k,n', SHAPES + WIDE)
@pytest.mark.parametrize('kind', ['bf16', 'f32', 'mx'])
def test_dense_exact(lib, m, k, n, kind):
    t = torch()
    rng = np.random.default_rng(m * 7919 + k * 31 + n)
    a, w = random_mx(rng, m, k), random_mx(rng, n, k, spare=0)
    b = exact_bias(rng, n) if (m + n) % 2 else None
    relu = int(k % 2)
    want = a.values @ w.values.T + (b if b is not None else 0.0)
    if relu:
        want = np.maximum(want, 0.0)
    out = Out(kind, m, n)
    run_dense(lib, a, w, t.from_numpy(np.asarray(b, dtype=np.float32)).cuda() if b is not None else None, out, relu)
    got = out.get()
    assert lib.device_status() == 0
    if kind == 'mx':
        codes, scales = (np.concatenate(p) for p in zip(*(R.quantize(want[i:i + 512]) for i in range(0, m, 512))))
        assert np.array_equal(got[1], scales)
        assert np.array_equal(R.values(*got), R.values(codes, scales))      # a zero's sign is free
    else:
        assert np.array_equal(got, bf16_round(want) if kind == 'bf16' else want)


@pytest.mark.parametrize('m,k,n', [(1, 4096, 300), (40, 1000, 130), (300, 4096, 260)])
def test_dense_wide_scales(lib, m, k, n):
    """Scales over 20 binades: the order of the sum shows, and the tolerance counts it."""
    rng = np.random.default_rng(m + k + n)
    a, w = random_mx(rng, m, k, 117, 137), random_mx(rng, n, k, 117, 137)
    out = Out('f32', m, n)
    run_dense(lib, a, w, None, out, 0)
    err = np.abs(out.get() - a.values @ w.values.T)
    assert (err <= (k + 2) * 2.0 ** -23 * (np.abs(a.values) @ np.abs(w.values.T))).all()


def test_dense_extreme_scales(lib):
    """Blocks of scale 2^-127 and 2^113 each on its own; NaN blocks make their row (or column) NaN and nothing else."""
    rng = np.random.default_rng(9)
    a, w = random_mx(rng, 140, 96), random_mx(rng, 150, 96)
    a.np_scales[3], w.np_scales[:] = 0, 127
    a.np_scales[4] = 240
    a.np_scales[7, 1], w.np_scales[11, 2] = 255, 255
    a, w = Mx(a.np_codes, a.np_scales), Mx(w.np_codes, w.np_scales)
    out = Out('f32', 140, 150)
    run_dense(lib, a, w, None, out, 0)
    got = out.get()
    with np.errstate(over='ignore'):
        want = (a.values @ w.values.T).astype(np.float32).astype(np.float64)
    nan = np.zeros((140, 150), dtype=bool)
    nan[7, :], nan[:, 11] = True, True
    assert np.array_equal(np.isnan(got), nan)
    keep = ~nan
    keep[3] = False
    assert np.array_equal(got[keep], want[keep])
    assert (np.abs(got[3][~nan[3]] - want[3][~nan[3]]) <= 96 * 2.0 ** -126).all()


def test_dense_relu_keeps_nan(lib):
    rng = np.random.default_rng(10)
    a, w = random_mx(rng, 5, 64), random_mx(rng, 40, 64)
    a.np_scales[2, 0] = 255
    a = Mx(a.np_codes, a.np_scales)
    out = Out('bf16', 5, 40)
    run_dense(lib, a, w, None, out, 1)
    got = out.get()
    assert np.isnan(got[2]).all() and not np.isnan(np.delete(got, 2, axis=0)).any()


# ---- gated --------------------------------------------------------------------------------------

def run_gated(lib, a, wg, wu, bg, bu, out, act):
    p = [None if b is None else b.data_ptr() for b in (bg, bu)]
    lib.check(lib.load().a4c_gated_dense_mx(*a.args, *wg.args, *wu.args, *p, *out.args, a.rows, a.cols, wg.rows, ACTS.index(act), stream()), 'gated')


def gated_sums(a, wg, wu, bg, bu):
    z = 0.0
    return a.values @ wg.values.T + (bg if bg is not None else z), a.values @ wu.values.T + (bu if bu is not None else z)


def dev32(x):
    return None if x is None else torch().from_numpy(np.asarray(x, dtype=np.float32)).cuda()


@pytest.mark.parametrize('m,k,n', SHAPES + WIDE)
@pytest.mark.parametrize('kind', ['bf16', 'f32', 'mx'])
def test_gated_exact(lib, m, k, n, kind):
    rng = np.random.default_rng(m * 7907 + k * 37 + n)
    a, wg, wu = random_mx(rng, m, k), random_mx(rng, n, k, spare=0), random_mx(rng, n, k, spare=64)
    bg = exact_bias(rng, n) if m % 2 else None
    bu = exact_bias(rng, n) if n % 2 else None
    act = 'relu' if k % 2 else 'none'
    g, u = gated_sums(a, wg, wu, bg, bu)
    want = (R.activate(g, act).astype(np.float32) * u.astype(np.float32)).astype(np.float64)     # one rounding
    out = Out(kind, m, n)
    run_gated(lib, a, wg, wu, dev32(bg), dev32(bu), out, act)
    got = out.get()
    assert lib.device_status() == 0
    if kind == 'mx':
        codes, scales = (np.concatenate(p) for p in zip(*(R.quantize(want[i:i + 512]) for i in range(0, m, 512))))
        assert np.array_equal(got[1], scales)
        assert np.array_equal(R.values(*got), R.values(codes, scales))
    else:
        assert np.array_equal(got, bf16_round(want) if kind == 'bf16' else want)


@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('kind', ['bf16', 'f32'])
def test_gated_activations(lib, act, kind):
    """Exact sums between about -40 and 40, so that what is measured is the activation: the exponential's stated error is
    2 + 1.2 |x| units in the last place, the quotient's 2, and five more roundings; the error function's polynomial form adds an
    absolute 2^-22, which x multiplies."""
    rng = np.random.default_rng(ACTS.index(act))
    m, k, n = 150, 64, 160
    a, wg, wu = random_mx(rng, m, k, 124, 125), random_mx(rng, n, k, 125, 126), random_mx(rng, n, k, 124, 126)
    bg, bu = exact_bias(rng, n) / 8, exact_bias(rng, n) / 8
    g, u = gated_sums(a, wg, wu, bg, bu)
    want = R.activate(g, act) * u
    out = Out(kind, m, n)
    run_gated(lib, a, wg, wu, dev32(bg), dev32(bu), out, act)
    z = np.abs(g) if act != 'gelu_tanh' else np.abs(1.6 * (g + 0.044715 * g ** 3))
    rel = (2 + 1.2 * z + 2 + 5 + 3 * z) * 2.0 ** -23              # 3 z: roundings of the exponent's argument
    tol = np.minimum(rel, 1.0) * np.abs(want) + 2.0 ** -22 * (1 + np.abs(g)) * np.abs(u)
    if kind == 'bf16':
        tol = tol + (np.abs(want) + tol) * 2.0 ** -8
    assert (np.abs(out.get() - want) <= tol).all()


@pytest.mark.parametrize('act', ['silu', 'gelu', 'gelu_tanh', 'sigmoid'])
@pytest.mark.parametrize('kind', ['bf16', 'f32', 'mx'])
def test_gated_activations_many_rows(lib, act, kind):
    """The same in the pair kernel, four and more tiles to a pair, each with its columns' own biases; the first rows alone then take the
    other kernel and give the same bits (exact sums, the same arithmetic behind them)."""
    rng = np.random.default_rng(100 + ACTS.index(act))
    m, k, n = 4100, 64, 2500
    a, wg, wu = random_mx(rng, m, k, 124, 125), random_mx(rng, n, k, 125, 126), random_mx(rng, n, k, 124, 126)
    bg, bu = exact_bias(rng, n) / 8, exact_bias(rng, n) / 8
    g, u = gated_sums(a, wg, wu, bg, bu)
    want = R.activate(g, act) * u
    out = Out(kind, m, n)
    run_gated(lib, a, wg, wu, dev32(bg), dev32(bu), out, act)
    got = out.get()
    assert lib.device_status() == 0
    few = Mx(a.np_codes[:37], a.np_scales[:37])
    some = Out(kind, 37, n)
    run_gated(lib, few, wg, wu, dev32(bg), dev32(bu), some, act)
    first = some.get()
    if kind == 'mx':
        ref_codes, ref_scales = (np.concatenate(p) for p in zip(*(R.quantize(want[i:i + 512]) for i in range(0, m, 512))))
        ref, val = R.values(ref_codes, ref_scales), R.values(*got)
        # a result next to a border between two codes, or a block's largest next to a power of two, may go either way
        step = 4 * np.repeat(np.exp2(ref_scales.astype(np.float64) - 127), 32, axis=1)[:, :n]
        assert (np.abs(val - ref) <= step).all() and (val != ref).mean() < 1e-3
        assert np.array_equal(R.values(*first), val[:37])
        return
    z = np.abs(g) if act != 'gelu_tanh' else np.abs(1.6 * (g + 0.044715 * g ** 3))
    rel = (2 + 1.2 * z + 2 + 5 + 3 * z) * 2.0 ** -23
    tol = np.minimum(rel, 1.0) * np.abs(want) + 2.0 ** -22 * (1 + np.abs(g)) * np.abs(u)
    if kind == 'bf16':
        tol = tol + (np.abs(want) + tol) * 2.0 ** -8
    assert (np.abs(got - want) <= tol).all()
    assert np.array_equal(first, got[:37])


@pytest.mark.parametrize('which', ['gate', 'other'])
def test_gated_one_bias_many_rows(lib, which):
    """Only one of the two biases, several tiles to a pair, a last tile of columns beyond the features."""
    rng = np.random.default_rng(31)
    m, k, n = 2600, 64, 4999
    a, wg, wu = random_mx(rng, m, k), random_mx(rng, n, k), random_mx(rng, n, k)
    b = exact_bias(rng, n)
    bg, bu = (b, None) if which == 'gate' else (None, b)
    g, u = gated_sums(a, wg, wu, bg, bu)
    out = Out('f32', m, n)
    run_gated(lib, a, wg, wu, dev32(bg), dev32(bu), out, 'none')
    assert np.array_equal(out.get(), (g.astype(np.float32) * u.astype(np.float32)).astype(np.float64))


@pytest.mark.parametrize('m', [7, 700])
@pytest.mark.parametrize('act', ['silu', 'gelu', 'gelu_tanh', 'sigmoid'])
def test_gated_keeps_nan(lib, m, act):
    """A NaN in either factor is a NaN in the output, and only there."""
    rng = np.random.default_rng(m)
    n, k = 2300, 64
    a, wg, wu = random_mx(rng, m, k), random_mx(rng, n, k), random_mx(rng, n, k)
    a.np_scales[4, 1], wg.np_scales[33, 0], wu.np_scales[90, 1] = 255, 255, 255
    a, wg, wu = (Mx(q.np_codes, q.np_scales) for q in (a, wg, wu))
    out = Out('f32', m, n)
    run_gated(lib, a, wg, wu, None, None, out, act)
    want = np.zeros((m, n), dtype=bool)
    want[4, :], want[:, 33], want[:, 90] = True, True, True
    assert np.array_equal(np.isnan(out.get()), want)


def test_gated_far_arguments(lib):
    """Sums of +-2^14 and more: sigmoid ends at 0 and 1 without NaN."""
    rng = np.random.default_rng(77)
    a, wg, wu = random_mx(rng, 20, 256, 133, 134), random_mx(rng, 64, 256, 133, 134), random_mx(rng, 64, 256)
    for act in ('silu', 'gelu', 'gelu_tanh', 'sigmoid'):
        out = Out('f32', 20, 64)
        run_gated(lib, a, wg, wu, None, None, out, act)
        g, u = gated_sums(a, wg, wu, None, None)
        far = np.abs(g) > 200
        assert far.mean() > 0.9
        s = np.where(g > 0, 1.0 if act == 'sigmoid' else g, 0.0)
        got = out.get()
        assert not np.isnan(got).any()
        assert (np.abs(got - s * u)[far] <= 2.0 ** -22 * np.abs(s * u)[far]).all()


def test_shapes_at_random(lib):
    """Sixty shapes over the whole range of rows, K and features, each exact: whatever tile, split or kernel a size selects."""
    rng = np.random.default_rng(20)
    t = torch()
    for i in range(60):
        m, k, n = (int(round(hi ** rng.random())) for hi in (3000, 2000, 2500))
        a, w, u = random_mx(rng, m, k), random_mx(rng, n, k), random_mx(rng, n, k)
        x = t.from_numpy(a.values).cuda()
        g, h = ((x @ t.from_numpy(q.values).cuda().T).cpu().numpy() for q in (w, u))      # exact in any order
        out = Out('f32', m, n)
        if i % 2:
            run_dense(lib, a, w, None, out, 0)
            want = g
        else:
            run_gated(lib, a, w, u, None, None, out, 'none')
            want = (g.astype(np.float32) * h.astype(np.float32)).astype(np.float64)
        assert np.array_equal(out.get(), want), (m, k, n, i)
    assert lib.device_status() == 0


# ---- as they are used ---------------------------------------------------------------------------

def test_feed_forward_block(lib):
    """quantise -> gated (MXFP4 out) -> dense, on a side stream, captured and replayed with new inputs."""
    t = torch()
    L = lib.load()
    rng = np.random.default_rng(21)
    m, d, f = 77, 320, 700
    wg, wu, wd = random_mx(rng, f, d, 122, 123), random_mx(rng, f, d, 122, 123), random_mx(rng, d, f, 122, 123)
    x = t.empty(m, d, dtype=t.bfloat16, device='cuda')
    xq = t.empty(m, up(d) // 2, dtype=t.uint8, device='cuda')
    xs = t.empty(L.a4c_mx_scale_bytes(m, d), dtype=t.uint8, device='cuda')
    hq = t.empty(m, up(f) // 2, dtype=t.uint8, device='cuda')
    hs = t.empty(L.a4c_mx_scale_bytes(m, f), dtype=t.uint8, device='cuda')
    y = t.empty(m, d, dtype=t.float32, device='cuda')

    def block():
        s = stream()
        lib.check(L.a4c_quantize_mx(x.data_ptr(), 0, d, xq.data_ptr(), up(d), xs.data_ptr(), m, d, s), 'quantize')
        lib.check(L.a4c_gated_dense_mx(xq.data_ptr(), up(d), xs.data_ptr(), *wg.args, *wu.args, None, None, hq.data_ptr(), 3, up(f), hs.data_ptr(),
                                       m, d, f, 2, s), 'gated')
        lib.check(L.a4c_dense_mx(hq.data_ptr(), up(f), hs.data_ptr(), *wd.args, None, y.data_ptr(), 1, d, None, m, f, d, 0, s), 'dense')

    def check_against(xv):
        codes, scales = R.quantize(xv)
        a = R.values(codes, scales)
        h = R.activate(a @ wg.values.T, 'silu') * (a @ wu.values.T)
        got_h = R.values(np.stack([hq.cpu().numpy() & 15, hq.cpu().numpy() >> 4], 2).reshape(m, -1)[:, :f], R.untile_scales(hs.cpu().numpy(), m, f))
        # the intermediate: at most one step of its block away from the definition's, and nearly everywhere equal
        ref_codes, ref_scales = R.quantize(h)
        ref_h = R.values(ref_codes, ref_scales)
        step = 4 * np.repeat(np.exp2(ref_scales.astype(np.float64) - 127), 32, axis=1)[:, :f]
        assert (np.abs(got_h - ref_h) <= step).all() and (got_h != ref_h).mean() < 1e-3
        # the last product: exact in its own operands up to the order of 700 additions
        want = got_h @ wd.values.T
        assert (np.abs(y.cpu().numpy() - want) <= (f + 2) * 2.0 ** -23 * (np.abs(got_h) @ np.abs(wd.values.T))).all()

    inputs = [t.from_numpy(rng.standard_normal((m, d))).to(t.bfloat16).cuda() for _ in range(3)]
    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(side):
        x.copy_(inputs[0])
        block()
    side.synchronize()
    check_against(inputs[0].double().cpu().numpy())
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        block()
    for xin in inputs[1:]:
        x.copy_(xin)
        graph.replay()
        t.cuda.synchronize()
        check_against(xin.double().cpu().numpy())
    assert lib.device_status() == 0


@pytest.mark.parametrize('m', [1, 16, 150, 600])
def test_same_bits_every_time(lib, m):
    """The split reduction adds in a fixed order; two streams at once do not disturb one another."""
    t = torch()
    rng = np.random.default_rng(m)
    a, w, u = random_mx(rng, m, 2000, 110, 140), random_mx(rng, 300, 2000, 110, 140), random_mx(rng, 300, 2000, 110, 140)
    outs = [Out('f32', m, 300) for _ in range(8)]
    streams = [t.cuda.Stream() for _ in range(2)]
    t.cuda.synchronize()
    for i, o in enumerate(outs):
        with t.cuda.stream(streams[i % 2]):
            run_dense(lib, a, w, None, o, 0) if i < 4 else run_gated(lib, a, w, u, None, None, o, 'silu')
    got = [o.get() for o in outs]
    assert all(np.array_equal(g, got[0]) for g in got[:4]) and all(np.array_equal(g, got[4]) for g in got[4:])


def test_rows_do_not_depend_on_their_batch(lib):
    """Row 0 of a large product equals the product of row 0 up to the order of its sum (exact operands: equal)."""
    rng = np.random.default_rng(3)
    a, w = random_mx(rng, 700, 512), random_mx(rng, 260, 512)
    one = Mx(a.np_codes[:1], a.np_scales[:1])
    big, small = Out('f32', 700, 260), Out('f32', 1, 260)
    run_dense(lib, a, w, None, big, 0)
    run_dense(lib, one, w, None, small, 0)
    assert np.array_equal(big.get()[:1], small.get())


@pytest.mark.parametrize('m', [40, 300, 600])
@pytest.mark.parametrize('gated', [False, True])
def test_nan_and_overflow_in_an_mxfp4_output(lib, m, gated):
    """A block whose float results hold a NaN or an infinity is a NaN block; its neighbours are what they were.  m = 40 takes the
    small tiles, 600 x 6000 the pair kernel."""
    n, k = 6000, 64
    rng = np.random.default_rng(m + gated)
    a, w, u = random_mx(rng, m, k), random_mx(rng, n, k), random_mx(rng, n, k, 127, 127)
    a.np_scales[5] = 255                            # row 5: NaN everywhere
    w.np_scales[70] = 255                           # column 70: NaN
    w.np_scales[200], w.np_codes[200] = 250, 7      # column 200: beyond float32 in rows whose sum does not cancel
    a, w = Mx(a.np_codes, a.np_scales), Mx(w.np_codes, w.np_scales)
    with np.errstate(over='ignore', invalid='ignore'):
        want = (a.values @ w.values.T).astype(np.float32)
        if gated:
            want = want * (a.values @ u.values.T).astype(np.float32)
    out = Out('mx', m, n)
    if gated:
        run_gated(lib, a, w, u, None, None, out, 'none')
    else:
        run_dense(lib, a, w, None, out, 0)
    codes, scales = out.get()
    want_codes, want_scales = R.quantize(want.astype(np.float64))
    sure = np.ones_like(want_scales, dtype=bool)
    sure[:, 200 // 32] = False                      # a partial sum may pass float32's range where the whole does not
    assert np.array_equal(scales[sure], want_scales[sure])
    assert (scales[5] == 255).all() and (scales[:, 2] == 255).all()
    keep = np.repeat(sure & (want_scales != 255), 32, axis=1)[:, :n]
    assert np.array_equal(R.values(codes, np.where(scales == 255, 0, scales))[keep], R.values(want_codes, np.where(want_scales == 255, 0, want_scales))[keep])


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
def test_wide_output_at_any_address(lib, kind):
    """An output whose base is not 16-byte aligned, in the kernel that otherwise stores by bulk copies."""
    t = torch()
    rng = np.random.default_rng(4)
    a, w = random_mx(rng, 300, 96), random_mx(rng, 6400, 96)
    td = {'bf16': t.bfloat16, 'f32': t.float32}[kind]
    store = t.full((300 * 6400 + 16,), -7.0, dtype=td, device='cuda')
    y = store[1:1 + 300 * 6400]
    lib.check(lib.load().a4c_dense_mx(*a.args, *w.args, None, y.data_ptr(), F[kind], 6400, None, 300, 96, 6400, 0, stream()), 'dense')
    want = a.values @ w.values.T
    assert np.array_equal(y.view(300, 6400).double().cpu().numpy(), bf16_round(want) if kind == 'bf16' else want)
    assert float(store[0]) == -7.0 and (store[1 + 300 * 6400:] == -7.0).all()


def test_offsets_beyond_32_bits(lib):
    """5 GB activations: the last rows of quantisation and of both products are what they are on their own."""
    t = torch()
    L = lib.load()
    rows, cols, n = 700000, 4096, 128
    x = t.empty(rows, cols, dtype=t.bfloat16, device='cuda')
    tail = t.randn(500, cols, device='cuda').bfloat16()
    x.zero_()
    x[-500:] = tail
    q = t.empty(rows, cols // 2, dtype=t.uint8, device='cuda')
    s = t.empty(L.a4c_mx_scale_bytes(rows, cols), dtype=t.uint8, device='cuda')
    lib.check(L.a4c_quantize_mx(x.data_ptr(), 0, cols, q.data_ptr(), cols, s.data_ptr(), rows, cols, stream()), 'quantize')
    codes, scales = R.quantize(tail.double().cpu().numpy())
    got = q[-500:].cpu().numpy()
    assert np.array_equal(np.stack([got & 15, got >> 4], 2).reshape(500, -1), codes)
    assert np.array_equal(R.untile_scales(s.cpu().numpy(), rows, cols)[-500:], scales)
    lib.check(L.a4c_dequantize_mx(q.data_ptr(), cols, s.data_ptr(), x.data_ptr(), 0, cols, rows, cols, stream()), 'dequantize')
    assert np.array_equal(x[-500:].double().cpu().numpy(), R.values(codes, scales)) and not x[:-500].any()
    # as the activation of a product, and as its output (K small, N large)
    rng = np.random.default_rng(8)
    w = random_mx(rng, n, cols, spare=0)
    y = t.empty(rows, n, dtype=t.float32, device='cuda')
    lib.check(L.a4c_dense_mx(q.data_ptr(), cols, s.data_ptr(), *w.args, None, y.data_ptr(), 1, n, None, rows, cols, n, 0, stream()), 'dense')
    v = R.values(codes, scales)
    err = np.abs(y[-500:].double().cpu().numpy() - v @ w.values.T)
    assert (err <= (cols + 2) * 2.0 ** -23 * (np.abs(v) @ np.abs(w.values.T))).all() and not y[:-500].any()
    a = random_mx(rng, 600, 32, spare=0)
    big = random_mx(rng, cols, 32, spare=0)
    rep = t.empty(rows, 16, dtype=t.uint8, device='cuda')
    rep[:] = a.codes.repeat(rows // 600 + 1, 1)[:rows]
    # 600 rows repeat, scales are the same throughout: a constant tensor of 2^0
    ones = t.full((L.a4c_mx_scale_bytes(rows, 32),), 0, dtype=t.uint8, device='cuda')
    ones.view(-1, 32, 4, 4)[..., 0] = 127
    lib.check(L.a4c_dense_mx(rep.data_ptr(), 32, ones.data_ptr(), *big.args, None, x.data_ptr(), 0, cols, None, rows, 32, cols, 0, stream()), 'dense')
    last = rows - 1 - (rows - 1) % 600
    want = bf16_round(R.VALUES[a.np_codes[:rows - last]] @ big.values.T)
    assert np.array_equal(x[last:].double().cpu().numpy(), want)
    assert t.equal(x[:600], x[600 * 1000:600 * 1001])
    assert lib.device_status() == 0


def test_two_graphs_in_flight(lib):
    """Two captured blocks on two streams at once: there is no memory between calls that they could share."""
    t = torch()
    rng = np.random.default_rng(12)
    sets = []
    for i, m in enumerate((9, 200)):
        a, w, u = random_mx(rng, m, 640), random_mx(rng, 500, 640), random_mx(rng, 500, 640)
        out = Out('f32', m, 500)
        st, g = t.cuda.Stream(), t.cuda.CUDAGraph()
        run_gated(lib, a, w, u, None, None, out, 'none')
        t.cuda.synchronize()
        with t.cuda.graph(g, stream=st):
            for _ in range(6):
                run_gated(lib, a, w, u, None, None, out, 'none')
        sets.append((st, g, out, (a.values @ w.values.T).astype(np.float32) * (a.values @ u.values.T).astype(np.float32), (a, w, u)))
    for _ in range(5):
        for st, g, *_ in sets:
            with t.cuda.stream(st):
                g.replay()
    t.cuda.synchronize()
    for _, _, out, want, _ in sets:
        assert np.array_equal(out.get(), want.astype(np.float64))
