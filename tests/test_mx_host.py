"""MXFP4 on the host: the definition the GPU tests use, sizes, and every refusal of the four entry points (no GPU)."""

import ctypes

import numpy as np
import pytest

import mx_reference as R
from aie4ml_b200 import lib as a4c


def test_reference_quantiser_by_hand():
    x = np.zeros((1, 64))
    x[0, :8] = [4.0, 6.0, 0.25, 0.75, 1.25, 5.0, -2.5, 7.9]       # scale 1: floor(log2 7.9) = 2
    x[0, 32:] = 2.0 ** -140
    codes, scales = R.quantize(x)
    assert list(codes[0, :8]) == [6, 7, 0, 2, 2, 6, 12, 7]
    assert list(scales[0]) == [127, 0]
    assert (codes[0, 32:] == 0).all()
    x[0, 5] = np.inf
    assert R.quantize(x)[1][0, 0] == 255
    q = R.values(*R.quantize(np.linspace(-3, 3, 64)[None]))
    assert np.abs(q - np.linspace(-3, 3, 64)).max() <= 0.5         # half of the widest step (4 to 6) at scale 1/2


@pytest.mark.parametrize('rows,cols', [(1, 1), (128, 128), (129, 129), (777, 1000), (3, 4097)])
def test_scale_tiles(rows, cols):
    lib = a4c.load()
    s = np.random.default_rng(0).integers(0, 255, (rows, R.ceil_div(cols, 32))).astype(np.uint8)
    tiled = R.tile_scales(s, cols)
    assert tiled.size == lib.a4c_mx_scale_bytes(rows, cols)
    assert np.array_equal(R.untile_scales(tiled, rows, cols), s)


def test_scale_bytes_of_nothing_and_of_much():
    lib = a4c.load()
    assert lib.a4c_mx_scale_bytes(0, 5) == 0 and lib.a4c_mx_scale_bytes(5, 0) == 0 and lib.a4c_mx_scale_bytes(-1, 5) == 0
    assert lib.a4c_mx_scale_bytes(1 << 33, 1 << 20) == (1 << 26) * (1 << 13) * 512


P = 0x10000          # a 16-byte aligned address that no refused call touches
OK = dict(A=P, lda=64, As=P, W=P, ldw=64, Ws=P, U=P, ldu=64, Us=P, b=None, bu=None, Y=P, f=0, ldy=48, Ys=None, M=3, K=64, N=48, act=0)


def dense(**kw):
    d = dict(OK, **kw)
    return a4c.load().a4c_dense_mx(d['A'], d['lda'], d['As'], d['W'], d['ldw'], d['Ws'], d['b'], d['Y'], d['f'], d['ldy'], d['Ys'],
                                   d['M'], d['K'], d['N'], d['act'], None)


def gated(**kw):
    d = dict(OK, **kw)
    return a4c.load().a4c_gated_dense_mx(d['A'], d['lda'], d['As'], d['W'], d['ldw'], d['Ws'], d['U'], d['ldu'], d['Us'], d['b'], d['bu'],
                                         d['Y'], d['f'], d['ldy'], d['Ys'], d['M'], d['K'], d['N'], d['act'], None)


INVALID, ALIGN = a4c.A4C_ERR_INVALID_ARG, a4c.A4C_ERR_ALIGNMENT


@pytest.mark.parametrize('kw,code', [
    (dict(A=None), INVALID), (dict(As=None), INVALID), (dict(W=None), INVALID), (dict(Ws=None), INVALID), (dict(Y=None), INVALID),
    (dict(M=-1), INVALID), (dict(K=0), INVALID), (dict(N=0), INVALID), (dict(N=-5), INVALID),
    (dict(lda=32), INVALID), (dict(ldw=32), INVALID), (dict(ldy=47), INVALID),
    (dict(lda=72), ALIGN), (dict(ldw=80), ALIGN), (dict(A=P + 8), ALIGN), (dict(W=P + 1), ALIGN), (dict(As=P + 4), ALIGN), (dict(Ws=P + 8), ALIGN),
    (dict(Y=P + 1), ALIGN), (dict(Y=P + 2, f=1), ALIGN), (dict(b=P + 2), ALIGN),
    (dict(f=2), INVALID), (dict(f=4), INVALID), (dict(f=-1), INVALID), (dict(Ys=P), INVALID),
    (dict(f=3), INVALID), (dict(f=3, Ys=P), ALIGN), (dict(f=3, Ys=P, ldy=32), INVALID), (dict(f=3, Ys=P + 8, ldy=64), ALIGN),
    (dict(f=3, Ys=P, ldy=64, Y=P + 8), ALIGN), (dict(M=1 << 31), INVALID),
])
def test_products_refuse(kw, code):
    assert dense(**kw) == code
    assert gated(**kw) == code


@pytest.mark.parametrize('kw,code', [(dict(U=None), INVALID), (dict(Us=None), INVALID), (dict(ldu=32), INVALID), (dict(ldu=72), ALIGN),
                                     (dict(U=P + 4), ALIGN), (dict(bu=P + 1), ALIGN), (dict(act=-1), INVALID), (dict(act=6), INVALID)])
def test_gated_refuses(kw, code):
    assert gated(**kw) == code


def test_no_rows_is_no_launch():
    lib = a4c.load()
    assert dense(M=0) == 0 and gated(M=0) == 0
    assert lib.a4c_quantize_mx(P, 0, 64, P, 64, P, 0, 64, None) == 0
    assert lib.a4c_dequantize_mx(P, 64, P, P, 0, 64, 0, 64, None) == 0


@pytest.mark.parametrize('x,f,ldx,q,ldq,s,rows,cols,code', [
    (None, 0, 64, P, 64, P, 1, 64, INVALID), (P, 0, 64, None, 64, P, 1, 64, INVALID), (P, 0, 64, P, 64, None, 1, 64, INVALID),
    (P, 2, 64, P, 64, P, 1, 64, INVALID), (P, 3, 64, P, 64, P, 1, 64, INVALID), (P, 0, 63, P, 64, P, 1, 64, INVALID),
    (P, 0, 64, P, 32, P, 1, 64, INVALID), (P, 0, 64, P, 64, P, -1, 64, INVALID), (P, 0, 64, P, 64, P, 1, 0, INVALID),
    (P, 0, 64, P, 65, P, 1, 64, ALIGN), (P, 0, 64, P + 8, 64, P, 1, 64, ALIGN), (P, 0, 64, P, 64, P + 8, 1, 64, ALIGN),
    (P + 1, 0, 64, P, 64, P, 1, 64, ALIGN), (P + 2, 1, 64, P, 64, P, 1, 64, ALIGN),
    (P, 0, 64, P, 64, P, 1 << 40, 64, a4c.A4C_ERR_TOO_LARGE),
])
def test_quantisers_refuse(x, f, ldx, q, ldq, s, rows, cols, code):
    lib = a4c.load()
    assert lib.a4c_quantize_mx(x, f, ldx, q, ldq, s, rows, cols, None) == code
    assert lib.a4c_dequantize_mx(q, ldq, s, x, f, ldx, rows, cols, None) == code
