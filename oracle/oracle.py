"""CPU oracle: a NumPy restatement of the aie4ml AIE kernels' integer arithmetic.

TEST INFRASTRUCTURE ONLY.  Nothing in the shipped package imports this module; it is the
checker that the parity tests, the smoke test and the CPU-baseline leg of the benchmark
compare the CUDA path against.

Every function follows one reference kernel statement by statement (file:line cited per
function, paths relative to the aie4ml project root).  The kernels themselves need AMD's
``adf.h`` / ``aie_api`` (Vitis 2025.2, not redistributable, not vendored by the reference),
so they cannot be compiled outside Vitis; this restatement is parameterised by exactly
what the reference's Python resolver computes (shift, rounding token, dtypes, flags).

Pinning status
--------------
* Host-side quantisation, shift / rounding-token resolution, weight / bias / gamma / beta
  integers and EXP_KQ / EPS_Q0 are pinned against the reference's own Python code through
  the fixtures in ``tests/golden`` (generated by importing the reference).
* Kernel arithmetic (dense, matmul, softmax, layer norm, add): the reference holds no
  golden vectors and its only executable form is the Vitis simulator, so for those:
  **parity unpinned** beyond the kernel sources themselves.
* LayerNorm's reciprocal standard deviation goes through AMD's float ``aie::invsqrt`` /
  ``aie::to_fixed`` whose bits are not determined by the reference sources.  It is defined
  here as ``clamp(round_tok(2^15 * (1.0f / sqrtf((float)var))), 0, 32767)`` in IEEE
  binary32; the CUDA kernel evaluates the same expression with correctly rounded
  ``sqrt`` and ``div``.  **parity unpinned** for that one value.
"""

from __future__ import annotations

import numpy as np

# AIE-API rounding tokens.  The reference's resolver produces floor, ceil, symmetric_inf,
# symmetric_zero and conv_even (src/aie4ml/op_impls/utils/precision.py:13-21);
# positive_inf ("round half up") is the mode the benchmark configurations name.
ROUNDING_TOKENS = (
    'floor',
    'ceil',
    'positive_inf',
    'negative_inf',
    'symmetric_inf',
    'symmetric_zero',
    'conv_even',
    'conv_odd',
)

_INT_RANGE = {
    'int8': (-128, 127),
    'uint8': (0, 255),
    'int16': (-32768, 32767),
    'uint16': (0, 65535),
    'int32': (-(1 << 31), (1 << 31) - 1),
}
_NP_DTYPE = {'int8': np.int8, 'uint8': np.uint8, 'int16': np.int16, 'uint16': np.uint16, 'int32': np.int32}


def round_shift(v, shift: int, tok: str):
    """Arithmetic right shift of integer ``v`` by ``shift`` bits with rounding ``tok``.

    This is the rounding half of the AIE "SRS" step that every ``to_vector<T>(SHIFT)`` in the
    reference kernels performs (e.g. templates/nnet_utils/dense_bias_relu/dense_bias_relu.cpp:154-162
    with the mode set at :9).  ``shift == 0`` is the identity.
    """
    v = np.asarray(v, dtype=np.int64)
    shift = int(shift)
    if shift < 0:
        raise ValueError('shift must be non-negative')
    if shift == 0:
        return v.copy()
    q = v >> shift
    r = v & ((1 << shift) - 1)
    half = 1 << (shift - 1)
    if tok == 'floor':
        inc = np.zeros_like(q, dtype=bool)
    elif tok == 'ceil':
        inc = r != 0
    elif tok == 'positive_inf':
        inc = r >= half
    elif tok == 'negative_inf':
        inc = r > half
    elif tok == 'symmetric_inf':
        inc = np.where(v >= 0, r >= half, r > half)
    elif tok == 'symmetric_zero':
        inc = np.where(v >= 0, r > half, r >= half)
    elif tok == 'conv_even':
        inc = (r > half) | ((r == half) & ((q & 1) == 1))
    elif tok == 'conv_odd':
        inc = (r > half) | ((r == half) & ((q & 1) == 0))
    else:
        raise ValueError(f'unknown rounding token {tok!r}')
    return q + inc.astype(np.int64)


def srs(v, shift: int, tok: str, out_dtype: str):
    """Shift-round-saturate to ``out_dtype``; saturation is always on
    (templates/firmware/variants/dense_bias_relu/parameters.h.jinja:26-29)."""
    lo, hi = _INT_RANGE[out_dtype]
    return np.clip(round_shift(v, shift, tok), lo, hi).astype(_NP_DTYPE[out_dtype])


def _wrap32(v):
    """Two's-complement wrap to 32 bits: the acc32 accumulator lanes are 32 bits wide."""
    return ((np.asarray(v, dtype=np.int64) + (1 << 31)) & 0xFFFFFFFF) - (1 << 31)


def _int_matmul(a, b):
    """Exact integer product of two integer matrices (|values| < 2^16, K < 2^20).

    float64 BLAS is exact here: every partial sum stays far below 2^53."""
    a = np.asarray(a)
    b = np.asarray(b)
    k = a.shape[-1]
    amax = max(1, int(np.abs(a.astype(np.int64)).max(initial=0)))
    bmax = max(1, int(np.abs(b.astype(np.int64)).max(initial=0)))
    if amax * bmax * max(1, k) >= (1 << 52):
        return np.matmul(a.astype(np.int64), b.astype(np.int64))
    return np.rint(np.matmul(a.astype(np.float64), b.astype(np.float64))).astype(np.int64)


def dense(a, w, bias, *, shift: int, tok: str, relu: bool, out_dtype: str = 'int8', acc_bits: int = 32):
    """Dense layer: ``relu?(srs(A @ W + bias))``.

    Follows dense_single::run, templates/nnet_utils/dense_bias_relu/dense_bias_relu.cpp:67-166:
    bias initialises the accumulator (:114-124), int8 x int8 MACs accumulate in acc32 (:132-151),
    ``to_vector<result_t>(SHIFT)`` rounds and saturates, and ReLU is ``max(., 0)`` applied AFTER the
    saturation (:153-157).  The cascade variants (:170-430) add the bias at the chain's end
    instead, which is the same value in wrap-around accumulator arithmetic.

    ``a`` is [..., K] (leading axes flatten into rows), ``w`` is [K, N], ``bias`` [N] int32 or None.
    """
    a = np.asarray(a)
    lead = a.shape[:-1]
    acc = _int_matmul(a.reshape(-1, a.shape[-1]), w)
    if bias is not None:
        acc = acc + np.asarray(bias, dtype=np.int64)[None, :]
    if acc_bits == 32:
        acc = _wrap32(acc)
    y = srs(acc, shift, tok, out_dtype)
    if relu:
        y = np.maximum(y, 0).astype(y.dtype)
    return y.reshape(*lead, -1)


def matmul(a, b, *, shift: int, tok: str, transpose_a: bool = False, transpose_b: bool = False,
           out_dtype: str = 'int8', acc_bits: int = 32):
    """Dynamic MatMul ``srs(A @ B)``; no bias, no ReLU.

    Follows matmul_single::run, templates/nnet_utils/matmul/matmul.cpp:32-118.  TRANSPOSE_A/B
    (:60-77) mean the operand arrives with its last two axes swapped; here the caller passes
    the stored operand and the flag.  Leading axes are independent problems (the reference
    applies the rank-2 contract to each, op_impls/families/matmul/resolver.py:440-463).
    """
    a = np.asarray(a)
    b = np.asarray(b)
    if transpose_a:
        a = np.swapaxes(a, -1, -2)
    if transpose_b:
        b = np.swapaxes(b, -1, -2)
    acc = _int_matmul(a, b)
    if acc_bits == 32:
        acc = _wrap32(acc)
    return srs(acc, shift, tok, out_dtype)


def add(a, b, *, shift: int = 0, tok: str = 'conv_even', out_dtype: str = 'int8'):
    """Elementwise ``srs(a + b, SHIFT)``: elementwise_add_kernel::run,
    templates/nnet_utils/elementwise_add/elementwise_add.cpp:12-37.  On the integer path the
    resolver forces equal types so SHIFT is 0 and this is a saturating add
    (op_impls/families/elementwise/resolver.py:14-33)."""
    acc = np.asarray(a, dtype=np.int64) + np.asarray(b, dtype=np.int64)
    return srs(acc, shift, tok, out_dtype)


# --------------------------------------------------------------------------------------------
# Float-simulation path (AIEConfig.ComputeDtype; passes/force_float_mode.py:22-46).  The reference holds it to
# tolerances against a float model (tests/test_float_sim.py:60-93), so this is a float64 evaluation with the
# storage rounding of each tensor, not a bit-level model of an accumulation order.
# --------------------------------------------------------------------------------------------
def fp8_e4m3_grid() -> np.ndarray:
    """The 127 non-negative finite values of FP8 E4M3 (finite-only variant: 4 exponent bits with bias 7, 3 mantissa
    bits, no infinities, S.1111.111 = NaN), ascending; index = encoding."""
    vals = []
    for code in range(0x7F):
        e, m = code >> 3, code & 7
        vals.append(m * 2.0 ** -9 if e == 0 else (1.0 + m / 8.0) * 2.0 ** (e - 7))
    return np.asarray(vals, dtype=np.float64)


def round_float(values, fmt: str):
    """Round to the storage type ('bfloat16' / 'fp8_e4m3' to nearest even, or 'float32'); returned as float32
    values.  fp8_e4m3 results beyond the largest finite value (448) saturate to it."""
    if fmt == 'fp8_e4m3':
        v = np.asarray(values, dtype=np.float32).astype(np.float64)     # the device rounds a float32 accumulator
        grid = fp8_e4m3_grid()
        mag = np.minimum(np.abs(v), grid[-1])
        hi = np.clip(np.searchsorted(grid, mag, side='left'), 1, len(grid) - 1)
        lo = hi - 1
        d_lo, d_hi = mag - grid[lo], grid[hi] - mag
        pick = np.where(d_lo < d_hi, lo, np.where(d_hi < d_lo, hi, np.where(lo % 2 == 0, lo, hi)))   # tie: even encoding
        return np.copysign(grid[pick], v).astype(np.float32)
    f = np.ascontiguousarray(np.asarray(values, dtype=np.float32))
    if fmt == 'float32':
        return f
    u = f.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32) << 16
    return r.astype(np.uint32).view(np.float32).reshape(f.shape)


def dense_float(a, w, bias, *, relu: bool, fmt: str):
    """``relu?(A @ W + bias)`` on stored (already rounded) operands, result rounded to ``fmt``."""
    a = np.asarray(a, dtype=np.float64)
    acc = a.reshape(-1, a.shape[-1]) @ np.asarray(w, dtype=np.float64)
    if bias is not None:
        acc = acc + np.asarray(bias, dtype=np.float64)[None, :]
    if relu:
        acc = np.maximum(acc, 0.0)
    return round_float(acc, fmt).reshape(*a.shape[:-1], -1)


def matmul_float(a, b, *, transpose_a: bool = False, transpose_b: bool = False, fmt: str):
    a, b = np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64)
    if transpose_a:
        a = np.swapaxes(a, -1, -2)
    if transpose_b:
        b = np.swapaxes(b, -1, -2)
    return round_float(a @ b, fmt)


# --------------------------------------------------------------------------------------------
# MXFP4 products (no counterpart in the reference)
# --------------------------------------------------------------------------------------------

def mx_round(x):
    """The values the MXFP4 form of ``x`` stands for: blocks of 32 along the last axis, scale 2^max(floor(log2 max) - 2, -127),
    E2M1 magnitudes 0 .5 1 1.5 2 3 4 6, nearest even, saturating; a block that holds a NaN or an infinity is NaN."""
    x = np.asarray(x, dtype=np.float64)
    cols = x.shape[-1]
    v = np.zeros((x.size // cols, (cols + 31) // 32 * 32))
    v[:, :cols] = x.reshape(-1, cols)
    v = v.reshape(v.shape[0], -1, 32)
    bad = ~np.isfinite(v).all(axis=2, keepdims=True)
    v = np.where(bad, 0.0, v)
    top = np.abs(v).max(axis=2, keepdims=True)
    e = np.maximum(np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -127)      # frexp: top = m 2^e with 0.5 <= m < 1
    a = np.ldexp(np.abs(v), -e)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    q = np.ldexp(np.minimum(np.round(a / step) * step, 6.0), e)
    return np.where(bad, np.nan, np.copysign(q, v)).reshape(v.shape[0], -1)[:, :cols].reshape(x.shape)


def mx_activate(x, act: str):
    if act == 'relu':
        return np.maximum(x, 0.0)
    if act in ('silu', 'sigmoid'):
        s = 1.0 / (1.0 + np.exp(-x))
        return x * s if act == 'silu' else s
    if act == 'gelu':
        from math import erf

        return 0.5 * x * (1.0 + np.vectorize(erf, otypes=[np.float64])(x / np.sqrt(2.0)))
    if act == 'gelu_tanh':
        return 0.5 * x * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (x + 0.044715 * x ** 3)))
    return x


def mx_product(op: dict, x, params: dict):
    """float64 result of an MXFP4 Dense or gated Dense on the (float) activation ``x``, which it quantises first."""
    a = mx_round(x)
    def linear(w, b):
        y = a @ np.asarray(params[op[w]], dtype=np.float64)
        return y + np.asarray(params[op[b]], dtype=np.float64) if op.get(b) else y
    if op['kind'] == 'dense_mx':
        return mx_activate(linear('weight', 'bias'), 'relu' if op['relu'] else 'none')
    return mx_activate(linear('gate', 'gate_bias'), op['activation']) * linear('up', 'up_bias')


# --------------------------------------------------------------------------------------------
# Softmax
# --------------------------------------------------------------------------------------------

def softmax_numer(out_dtype: str, inv_shift: int) -> int:
    """NUMER of templates/nnet_utils/softmax/softmax.h:22."""
    return 32767 if out_dtype == 'int16' else (255 << int(inv_shift))


def _softmax_finish(score, out_dtype: str, inv_shift: int, use_clb: bool):
    """Row sum, reciprocal and normalisation shared by the four softmax kernels.

    ``inv = floor(NUMER / sum)`` (softmax.cpp:71-75; the tiled kernels reach the same integer
    through batched_reciprocal :108-127, whose correction loops make the float seed irrelevant).
    The linear kernels narrow ``inv`` to int16 without a clamp (:79, :372), the tiled ones clamp
    to [0, 32767] (:218-220); under the resolver's constraints both are the identity, and the
    oracle applies the clamp.  Output is ``srs(score * inv, OUT_SHIFT, floor)`` with
    OUT_SHIFT = INV_SHIFT for uint8 and 0 for int16 (softmax.h:53)."""
    score = np.asarray(score, dtype=np.int64)
    total = score.sum(axis=-1, keepdims=True)
    total = np.where(total > 0, total, 1)
    if use_clb:
        k = np.floor(np.log2(total.astype(np.float64))).astype(np.int64)
        k = np.where((1 << k) > total, k - 1, k)
        k = np.where((1 << (k + 1)) <= total, k + 1, k)
        if out_dtype == 'int16':
            inv = 32767 >> k
        else:
            sh = int(inv_shift) - k
            inv = np.where(sh >= 0, 255 << np.maximum(sh, 0), 255 >> np.maximum(-sh, 0))
    else:
        inv = softmax_numer(out_dtype, inv_shift) // total
    inv = np.clip(inv, 0, 32767)
    out_shift = 0 if out_dtype == 'int16' else int(inv_shift)
    return srs(score * inv, out_shift, 'floor', out_dtype)


def softmax_hccs(x, *, B: int, S: int, Dmax: int, inv_shift: int = 15, use_clb: bool = False,
                 out_dtype: str = 'uint8'):
    """HCCS clipped-linear surrogate softmax over the last axis, int8 in.

    softmax_i8::softmax_row, templates/nnet_utils/softmax/softmax.cpp:20-88 (tiled twin
    :159-239): ``d = min(max - x, Dmax)``, ``score = B - S*d`` narrowed to int16 with
    saturation (:57), then the shared finish."""
    x = np.asarray(x, dtype=np.int64)
    m = x.max(axis=-1, keepdims=True)
    d = np.minimum(m - x, int(Dmax))
    score = np.clip(int(B) - int(S) * d, -32768, 32767)
    return _softmax_finish(score, out_dtype, inv_shift, use_clb)


EXP_A2, EXP_B1, EXP_C0, EXP_ZF = 2811, -11004, 16384, 8


def exp_score16(d, exp_kq: int):
    """``2^(-d*KQ/256)`` in Q14 for d = max - x in [0, 255].

    exp_score16, templates/nnet_utils/softmax/softmax.cpp:252-273, constants from
    templates/firmware/variants/softmax/parameters.h.jinja:18-22.  All int16 with floor shifts
    (the softmax parameter block hard-wires rounding floor, :23-27)."""
    d = np.asarray(d, dtype=np.int64)
    z = np.clip(d * int(exp_kq), -32768, 32767)
    zint = z >> EXP_ZF
    zfrac = z & ((1 << EXP_ZF) - 1)
    t = np.clip((zfrac * EXP_A2) >> EXP_ZF, -32768, 32767)
    inner = t + EXP_B1
    t2 = np.clip((inner * zfrac) >> EXP_ZF, -32768, 32767)
    e = t2 + EXP_C0
    for b in range(4):
        e = np.where((zint & (1 << b)) != 0, e >> (1 << b), e)
    e = np.where(zint >= 16, 0, e)
    return e


def softmax_exp(x, *, exp_kq: int, inv_shift: int = 15, out_dtype: str = 'uint8'):
    """Accurate integer-exp softmax over the last axis, int8 in.

    softmax_exp_i8::run, templates/nnet_utils/softmax/softmax.cpp:333-384 (tiled twin :279-329)."""
    x = np.asarray(x, dtype=np.int64)
    m = x.max(axis=-1, keepdims=True)
    e = exp_score16(m - x, exp_kq)
    return _softmax_finish(e, out_dtype, inv_shift, False)


def exp_kq(in_frac: int, temperature: float = 1.0) -> int:
    """EXP_KQ = round(log2(e) * 2^-in_frac * temperature * 256):
    op_impls/families/softmax/softmax.py:309-337."""
    import math

    return int(round(math.log2(math.e) * (2.0 ** -int(in_frac)) * float(temperature) * (1 << EXP_ZF)))


# --------------------------------------------------------------------------------------------
# LayerNorm
# --------------------------------------------------------------------------------------------

def _round_float_tok(f, tok: str):
    """Round binary32 values to integers with an AIE rounding token."""
    f = np.asarray(f, dtype=np.float32)
    fl = np.floor(f)
    frac = f - fl  # exact: f < 2^16 here
    fl = fl.astype(np.int64)
    if tok == 'floor':
        return fl
    if tok == 'ceil':
        return fl + (frac > 0)
    if tok == 'positive_inf':
        return fl + (frac >= 0.5)
    if tok == 'negative_inf':
        return fl + (frac > 0.5)
    # the argument is never negative here, so the symmetric modes reduce to these
    if tok == 'symmetric_inf':
        return fl + (frac >= 0.5)
    if tok == 'symmetric_zero':
        return fl + (frac > 0.5)
    if tok == 'conv_even':
        return fl + ((frac > 0.5) | ((frac == 0.5) & ((fl & 1) == 1)))
    if tok == 'conv_odd':
        return fl + ((frac > 0.5) | ((frac == 0.5) & ((fl & 1) == 0)))
    raise ValueError(f'unknown rounding token {tok!r}')


def inv_std_q15(var, tok: str):
    """Q15 reciprocal standard deviation of an integer variance >= 1.

    row_statistics, templates/nnet_utils/layer_norm/layer_norm.cpp:33-39:
    ``to_fixed<int32>(invsqrt(to_float(var)), 15)`` clamped to [0, 32767].  AMD's float bits are
    not determined by the reference sources; this restatement evaluates
    ``1.0f / sqrtf((float)var)`` in IEEE binary32, scales by 2^15 (exact) and rounds with the
    op's rounding token."""
    v = np.asarray(var, dtype=np.int64).astype(np.float32)
    inv = (np.float32(1.0) / np.sqrt(v)).astype(np.float32)
    q = _round_float_tok(inv * np.float32(32768.0), tok)
    return np.clip(q, 0, 32767)


def layer_norm(x, gamma, beta, *, eps_q0: int, out_shift: int, tok: str, out_dtype: str = 'int8'):
    """Integer LayerNorm over the last axis (length a power of two), int8 in/out.

    layernorm_i8::run + row_statistics, templates/nnet_utils/layer_norm/layer_norm.cpp:15-121
    (tiled twin :144-231).  gamma is int16 Q7, beta int16 Q15
    (op_impls/families/layernorm/common.py:19-20)."""
    x = np.asarray(x, dtype=np.int64)
    cols = x.shape[-1]
    log2c = int(cols).bit_length() - 1
    if (1 << log2c) != cols:
        raise ValueError('LayerNorm width must be a power of two')
    gamma = np.asarray(gamma, dtype=np.int64)
    beta = np.asarray(beta, dtype=np.int64)
    sum_x = x.sum(axis=-1, keepdims=True)
    sum_sq = (x * x).sum(axis=-1, keepdims=True)
    mu = (sum_x + (cols >> 1)) >> log2c
    centered = _wrap32(sum_sq - 2 * mu * sum_x + cols * mu * mu)
    var = np.maximum(centered >> log2c, 0) + int(eps_q0)
    inv_std = inv_std_q15(var, tok)
    vd = np.clip(x - mu, -32768, 32767)
    fscale = np.clip(round_shift(inv_std * gamma, 7, tok), -32768, 32767)
    acc = _wrap32(vd * fscale + beta)
    return srs(acc, 15 - int(out_shift), tok, out_dtype)


# --------------------------------------------------------------------------------------------
# Host-side quantisation at graph boundaries and for constants
# --------------------------------------------------------------------------------------------

def apply_rounding(values, mode: str):
    """Host rounding of float values: src/aie4ml/quant_utils.py:48-61 (mode = RoundingMode name)."""
    values = np.asarray(values, dtype=np.float64)
    if mode in ('TRN', 'RND_MIN_INF'):
        return np.floor(values)
    if mode in ('TRN_ZERO', 'RND_ZERO'):
        return np.trunc(values)
    if mode == 'RND_INF':
        return np.ceil(values)
    if mode == 'RND_CONV':
        return np.round(values)
    if mode == 'RND':
        return np.where(values >= 0, np.floor(values + 0.5), np.ceil(values - 0.5))
    raise ValueError(f'unsupported rounding mode {mode}')


def handle_overflow(values, width: int, signed: bool, mode: str):
    """Host overflow handling: src/aie4ml/quant_utils.py:64-89 (mode = SaturationMode name)."""
    values = np.asarray(values, dtype=np.int64)
    lo = -(1 << (width - 1)) if signed else 0
    hi = (1 << (width - 1)) - 1 if signed else (1 << width) - 1
    if mode == 'WRAP':
        wrapped = np.mod(values, 1 << width)
        if signed:
            wrapped = np.where(wrapped >= (1 << (width - 1)), wrapped - (1 << width), wrapped)
        return wrapped
    if mode == 'SAT':
        return np.clip(values, lo, hi)
    if mode == 'SAT_ZERO':
        return np.where(values < 0, 0, np.clip(values, 0, hi))
    if mode == 'SAT_SYM':
        return np.clip(values, -hi if signed else lo, hi)
    raise ValueError(f'unsupported saturation mode {mode}')


def quantize(values, *, frac: int, width: int, signed: bool, rounding: str, saturation: str):
    """float -> integer codes: src/aie4ml/simulation.py:260-269 and
    op_impls/families/matmul/common.py:287-304."""
    scale = float(1 << frac) if frac > 0 else 1.0
    rounded = apply_rounding(np.asarray(values, dtype=np.float64) * scale, rounding).astype(np.int64)
    return handle_overflow(rounded, width, signed, saturation)


def dequantize(codes, frac: int):
    """integer codes -> float64: src/aie4ml/simulation.py:248-257."""
    frac = max(0, int(frac))
    return np.asarray(codes, dtype=np.float64) / float(1 << frac)


# --------------------------------------------------------------------------------------------
# Whole lowered graph
# --------------------------------------------------------------------------------------------

def run_plan(plan: dict, inputs: dict) -> dict:
    """Evaluate an exported lowered plan (a plain dict: op list, integer parameters, view ops)
    on integer input codes and return every graph output as integer codes.

    The plan format is what ``CudaModel.export_plan()`` writes: each op names its tensors and
    carries the numeric contract the resolver computed (shift, rounding token, dtypes, flags);
    view ops (slice / concat / transposed operand) are applied with NumPy indexing."""
    env = {name: np.asarray(arr) for name, arr in inputs.items()}
    params = plan['params']
    for op in plan['ops']:
        kind = op['kind']
        if kind == 'dense':
            # a transposed input view (TRANSPOSE_INPUT, dense_bias_relu.cpp:99): the kernel reads A^T of the stored tensor
            lhs = np.swapaxes(env[op['lhs']], -1, -2) if op.get('transpose_lhs', False) else env[op['lhs']]
            env[op['out']] = dense(
                lhs, params[op['weight']], params[op['bias']] if op.get('bias') else None,
                shift=op['shift'], tok=op['rounding'], relu=op['relu'], out_dtype=op['out_dtype'],
                acc_bits=op.get('acc_bits', 32))
        elif kind == 'matmul':
            env[op['out']] = matmul(
                env[op['lhs']], env[op['rhs']], shift=op['shift'], tok=op['rounding'],
                transpose_a=op.get('transpose_lhs', False), transpose_b=op.get('transpose_rhs', False),
                out_dtype=op['out_dtype'], acc_bits=op.get('acc_bits', 32))
        elif kind == 'add':
            env[op['out']] = add(env[op['lhs']], env[op['rhs']], shift=op['shift'], tok=op['rounding'],
                                 out_dtype=op['out_dtype'])
        elif kind == 'dense_f':
            lhs = np.swapaxes(env[op['lhs']], -1, -2) if op.get('transpose_lhs', False) else env[op['lhs']]
            env[op['out']] = dense_float(lhs, params[op['weight']], params[op['bias']] if op.get('bias') else None,
                                         relu=op['relu'], fmt=op['dtype'])
        elif kind in ('dense_mx', 'gated_dense_mx'):
            y = mx_product(op, env[op['lhs']], params)
            env[op['out']] = y if op.get('out_mx') else round_float(y, op['dtype'])   # out_mx: only its MXFP4 form exists
        elif kind == 'matmul_f':
            env[op['out']] = matmul_float(env[op['lhs']], env[op['rhs']], transpose_a=op.get('transpose_lhs', False),
                                          transpose_b=op.get('transpose_rhs', False), fmt=op['dtype'])
        elif kind == 'add_f':
            env[op['out']] = round_float(np.asarray(env[op['lhs']], np.float64) + np.asarray(env[op['rhs']], np.float64),
                                         op['dtype'])
        elif kind == 'layer_norm':
            env[op['out']] = layer_norm(
                env[op['lhs']], params[op['gamma']], params[op['beta']], eps_q0=op['eps_q0'],
                out_shift=op['out_shift'], tok=op['rounding'], out_dtype=op['out_dtype'])
        elif kind == 'softmax':
            if op['approximation'] == 'hccs':
                env[op['out']] = softmax_hccs(
                    env[op['lhs']], B=op['B'], S=op['S'], Dmax=op['Dmax'], inv_shift=op['inv_shift'],
                    use_clb=op['use_clb'], out_dtype=op['out_dtype'])
            else:
                env[op['out']] = softmax_exp(env[op['lhs']], exp_kq=op['exp_kq'], inv_shift=op['inv_shift'],
                                             out_dtype=op['out_dtype'])
        elif kind == 'slice':
            src = env[op['source']]
            for item in op['slices']:
                index = [slice(None)] * src.ndim
                index[op['axis']] = slice(item['start'], item['start'] + item['extent'])
                env[item['output']] = src[tuple(index)]
        elif kind == 'concat':
            env[op['out']] = np.concatenate([env[name] for name in op['inputs']], axis=op['axis'])
        else:
            raise ValueError(f'unknown plan op {kind!r}')
    return {name: env[name] for name in plan['outputs']}
