"""A feed-forward block of many rows (quantise, gated GELU with biases to MXFP4, Dense): the same bits on every run, and where its hidden
tensor has another 4-bit code than the definition in 64 bits gives, the exact value lies next to the border between the two."""

import numpy as np
import pytest

import mx_reference as R
from test_gpu_mx import lib, random_mx, stream, torch, up  # noqa: F401  (lib is the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('m,d,f', [(4100, 256, 1024), (700, 200, 1500)])
def test_block_of_many_rows(lib, m, d, f):  # noqa: F811
    t, L = torch(), lib.load()
    rng = np.random.default_rng(m)
    wg, wu, wd = random_mx(rng, f, d, 122, 123), random_mx(rng, f, d, 122, 123), random_mx(rng, d, f, 121, 122)
    bg, bu, bd = (t.from_numpy(rng.normal(0, 0.1, n).astype(np.float32)).cuda() for n in (f, f, d))
    x = t.from_numpy(rng.standard_normal((m, d))).to(t.bfloat16).cuda()
    new = lambda rows, cols: (t.empty(rows, up(cols) // 2, dtype=t.uint8, device='cuda'), t.empty(L.a4c_mx_scale_bytes(rows, cols), dtype=t.uint8, device='cuda'))
    args = lambda q: (q[0].data_ptr(), 2 * q[0].shape[1], q[1].data_ptr())
    runs = []
    for _ in range(4):
        xq, hq, y = new(m, d), new(m, f), t.empty(m, d, dtype=t.bfloat16, device='cuda')
        hq[0].zero_()
        lib.check(L.a4c_quantize_mx(x.data_ptr(), 0, d, *args(xq), m, d, stream()), 'quantize')
        lib.check(L.a4c_gated_dense_mx(*args(xq), *wg.args, *wu.args, bg.data_ptr(), bu.data_ptr(), hq[0].data_ptr(), 3, up(f), hq[1].data_ptr(), m, d, f, 3,
                                       stream()), 'gated')
        lib.check(L.a4c_dense_mx(*args(hq), *wd.args, bd.data_ptr(), y.data_ptr(), 0, d, None, m, f, d, 0, stream()), 'dense')
        runs.append((hq, y))
    t.cuda.synchronize()
    assert lib.device_status() == 0
    (codes, tiles), y = runs[0]
    for (c, s), z in runs[1:]:
        assert t.equal(c, codes) and t.equal(s[:m // 128 * 128 * up(f, 128) // 32], tiles[:m // 128 * 128 * up(f, 128) // 32])
        assert t.equal(z.view(t.int16), y.view(t.int16))

    dev = lambda v: t.from_numpy(np.asarray(v)).cuda()
    raw = codes.cpu().numpy()
    h = dev(R.values(np.stack([raw & 15, raw >> 4], 2).reshape(m, -1)[:, :f], R.untile_scales(tiles.cpu().numpy(), m, f)))
    a = dev(R.values(*R.quantize(x.double().cpu().numpy())))
    g, u = (a @ dev(w.values).T + b.double() for w, b in ((wg, bg), (wu, bu)))
    # errors of the sums (additions of float32, each at most 2^-23 of the sum of magnitudes) and of GELU (1e-7, two roundings)
    eg, eu = ((d + 3) * 2.0 ** -23 * (a.abs() @ dev(np.abs(w.values)).T + b.double().abs()) for w, b in ((wg, bg), (wu, bu)))
    act = g * t.special.ndtr(g)
    ea = 1.13 * eg + 1e-7 + 2.0 ** -22 * act.abs()                          # GELU's slope is at most 1.129
    exact = act * u
    eh = ea * (u.abs() + eu) + act.abs() * eu + 2.0 ** -23 * exact.abs()
    ref = dev(np.concatenate([R.values(*R.quantize(p)) for p in np.array_split(exact.cpu().numpy(), 8)]))
    other = h != ref
    # a border is half way between the two codes; next to a power of two of its block's largest magnitude a whole block changes
    top = t.zeros(m, up(f), dtype=t.float64, device='cuda')
    top[:, :f] = exact.abs()
    top = top.view(m, -1, 32)
    worst = t.zeros(m, up(f), dtype=t.float64, device='cuda')
    worst[:, :f] = eh
    largest = top.amax(2)
    edge = t.exp2(t.round(t.log2(largest.clamp(min=1e-30))))
    rescaled = (largest - edge).abs() <= worst.view(m, -1, 32).amax(2)
    near = (exact - (h + ref) / 2).abs() <= eh
    assert (near | rescaled.repeat_interleave(32, 1)[:, :f] | ~other).all()
    assert other.double().mean() < 1e-3
    want = h @ dev(wd.values).T + bd.double()
    tol = (f + 3) * 2.0 ** -23 * (h.abs() @ dev(np.abs(wd.values)).T + bd.double().abs())
    assert ((y.double() - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8).all()
