"""MXFP4 layers in a graph: packing, lowering and refusals on the CPU, execution on the GPU.

On the GPU a graph's result is compared bit for bit with the C calls it stands for, and with the oracle within the
tolerance of the bfloat16 path (rtol 1e-2, atol 5e-2)."""

import json

import numpy as np
import pytest

import mx_reference as R
from aie4ml_b200 import MXFP4, FloatFormat, FloatIntent, GraphBuilder, from_graph, intent
from aie4ml_b200.quant_utils import from_mx, mx_pitch, to_mx
from oracle import oracle

BF16 = FloatIntent(width=16, format=FloatFormat.BF16)
F32 = FloatIntent(width=32, format=FloatFormat.FP32)


@pytest.mark.parametrize('rows,cols', [(1, 1), (5, 33), (130, 257), (64, 1000)])
def test_host_packing(rows, cols):
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-8, 8, (rows, 1)))
    x[0, :1] = 5.0
    x.reshape(-1)[::7] = 0.75
    if rows > 4:
        x[1] = 0.0
        x[2] = 1e-45
        x[3, 0] = np.inf
        x[4, -1] = np.nan
    codes, tiles = to_mx(x)
    want_codes, want_scales = R.quantize(x)
    unbad = np.repeat(want_scales != 255, 32, axis=1)[:, :cols]
    got = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)
    assert codes.shape == (rows, mx_pitch(cols) // 2) and (got[:, cols:] == 0).all()
    assert np.array_equal(tiles, R.tile_scales(want_scales, cols))
    assert np.array_equal(got[:, :cols][unbad], want_codes[unbad])
    assert np.array_equal(from_mx(codes, tiles, rows, cols), R.values(want_codes, want_scales).astype(np.float32), equal_nan=True)
    clean = np.nan_to_num(x, nan=0.0, posinf=0.0)
    assert np.array_equal(oracle.mx_round(clean), R.values(*R.quantize(clean)))


def feed_forward(m=6, d=96, f=160, precision=BF16, activation='silu', bias=True, fusion=None, seed=0, residual=True):
    rng = np.random.default_rng(seed)
    wg, wu, wd = rng.normal(0, d ** -0.5, (d, f)), rng.normal(0, d ** -0.5, (d, f)), rng.normal(0, f ** -0.5, (f, d))
    bg, bu, bd = (rng.normal(0, 0.1, n) if bias else None for n in (f, f, d))
    b = GraphBuilder({'Part': 'cuda_b200', 'AIEConfig': {'FusionPolicy': fusion or {}}}, name='ffn')
    x = b.input('x', (m, d), precision)
    h = b.gated_dense('gate_up', x, wg, wu, MXFP4, precision, activation=activation, bias_gate=bg, bias_up=bu)
    y = b.dense('down', h, wd, MXFP4, precision, bias=bd)
    b.output(b.add('res', x, y, precision) if residual else y)
    return b, (wg, wu, wd, bg, bu, bd)


def test_lowering_and_export():
    b, weights = feed_forward()
    plan = from_graph(b).export_plan()
    assert [op['kind'] for op in plan['ops']] == ['gated_dense_mx', 'dense_mx', 'add_f']
    gated, down = plan['ops'][:2]
    assert (gated['K'], gated['N'], gated['activation'], gated['dtype']) == (96, 160, 'silu', 'bfloat16')
    assert (down['K'], down['N'], down['relu'], down['bias']) == (160, 96, False, 'down/bias')
    values = plan['params'][down['weight']]
    assert values.shape == (160, 96) and np.array_equal(values, from_mx(*to_mx(weights[2].T), 96, 160).T)
    x = np.random.default_rng(1).standard_normal((6, 96)).astype(np.float32)
    (out,) = oracle.run_plan(plan, {'x': x}).values()
    a = oracle.mx_round(x)
    bg, bu = weights[3].astype(np.float32), weights[4].astype(np.float32)
    h = R.activate(a @ plan['params']['gate_up/gate'] + bg, 'silu') * (a @ plan['params']['gate_up/up'] + bu)
    # every tensor of the exported graph is rounded to bfloat16 where it is written
    r = lambda v: oracle.round_float(v, 'bfloat16')
    assert np.array_equal(out, r(x.astype(np.float64) + r(oracle.mx_round(r(h)) @ values + weights[5].astype(np.float32))))


def test_compute_dtype_keeps_the_weights_in_mxfp4():
    b = GraphBuilder({'Part': 'cuda_b200', 'AIEConfig': {'ComputeDtype': 'bfloat16'}}, name='forced')
    x = b.input('x', (4, 32), intent(16, 13))
    b.output(b.dense('fc', x, np.ones((32, 16)) / 8, MXFP4, intent(16, 13), relu=True))
    (op,) = from_graph(b).export_plan()['ops']
    assert op['kind'] == 'dense_mx' and op['relu'] and op['dtype'] == 'bfloat16'


def test_graph_from_json():
    w = np.random.default_rng(0).normal(size=(32, 8))
    spec = {'name': 'g', 'inputs': [{'name': 'x', 'shape': [2, 32], 'precision': {'float': 'float32'}}],
            'params': {'w': {'data': w.tolist(), 'precision': {'float': 'mxfp4'}}},
            'nodes': [{'name': 'fc', 'op': 'mx_dense', 'inputs': ['x', 'w'], 'roles': ['lhs', 'rhs'],
                       'outputs': [{'name': 'y', 'shape': [2, 8], 'precision': {'float': 'float32'}}],
                       'metadata': {'n_in': 32, 'n_out': 8, 'activation': 'relu'}}], 'outputs': ['y']}
    plan = from_graph(json.loads(json.dumps(spec))).export_plan()
    assert plan['ops'][0]['kind'] == 'dense_mx' and plan['ops'][0]['relu']


def refuse(build, error, match):
    b = GraphBuilder({'Part': 'cuda_b200'}, name='bad')
    with pytest.raises(error, match=match):
        build(b)
        from_graph(b).export_plan()


def test_refusals():
    w = np.ones((32, 16))

    def graph(precision=BF16, out=BF16, weights=MXFP4, activation='silu', **kw):
        def build(b):
            x = b.input('x', (4, 32), precision)
            b.output(b.gated_dense('g', x, w, w, weights, out, activation=activation, **kw))
        return build

    refuse(graph(precision=intent(8, 4)), ValueError, "g: gated_dense over MXFP4 weights needs a bfloat16 or float32 lhs, got 'int8'")
    refuse(graph(out=FloatIntent(8, FloatFormat.FP8_E4M3)), ValueError, "float32 output, got 'fp8_e4m3'")
    refuse(graph(out=MXFP4), ValueError, "float32 output, got 'mxfp4'")
    refuse(graph(weights=BF16), ValueError, 'g: gated_dense needs MXFP4 weights')
    refuse(graph(activation='swish'), ValueError, "g: unknown activation 'swish'")
    refuse(graph(bias_up=np.ones(15)), ValueError, 'g: up_bias requires exactly 16 elements, got 15')

    def wrong_shape(b):
        b.gated_dense('g', b.input('x', (4, 31), BF16), w, w, MXFP4, BF16)
    refuse(wrong_shape, ValueError, 'do not match input features 31')

    def int_input(b):
        b.output(b.dense('fc', b.input('x', (4, 32), intent(8, 4)), w, MXFP4, intent(8, 4)))
    refuse(int_input, ValueError, "fc: mx_dense over MXFP4 weights needs a bfloat16 or float32 lhs, got 'int8'")

    def bad_bias(b):
        b.output(b.dense('fc', b.input('x', (4, 32), BF16), w, MXFP4, BF16, bias=np.ones(3)))
    refuse(bad_bias, ValueError, 'fc: bias requires exactly 16 elements, got 3')

    def transposed(b):
        x = b.input('x', (32, 4), BF16)
        b.output(b.dense('fc', b.transpose('t', x, [1, 0]), w, MXFP4, BF16))
    refuse(transposed, NotImplementedError, 'fc: mx_dense over MXFP4 weights has no kernel for a transposed input view')

    def int8_with_mx_weights(b):
        x = b.input('x', (4, 32), BF16)
        b.output(b.dense('fc', x, w, BF16, BF16))
    b = GraphBuilder({'Part': 'cuda_b200'}, name='fine')
    int8_with_mx_weights(b)
    assert from_graph(b).export_plan()['ops'][0]['kind'] == 'dense_f'      # other weights take the path they took


# ---- on the GPU ---------------------------------------------------------------------------------

def by_calls(x, weights, activation, dtype, chain):
    """The same block as C calls on torch tensors; returns the block's output before the residual."""
    import torch

    from aie4ml_b200 import lib as a4c

    L, s = a4c.load(), torch.cuda.current_stream().cuda_stream
    wg, wu, wd, bg, bu, bd = weights
    td, f = (torch.bfloat16, 0) if dtype == 'bfloat16' else (torch.float32, 1)
    m, d = x.shape
    n = wg.shape[1]

    def weight(w):
        codes, tiles = to_mx(w.T)
        return torch.from_numpy(codes).cuda(), torch.from_numpy(tiles).cuda()

    def vec(b):
        return None if b is None else torch.from_numpy(b.astype(np.float32)).cuda()

    def args(q):
        return q[0].data_ptr(), 2 * q[0].shape[1], q[1].data_ptr()

    def new(rows, cols):
        return (torch.zeros(rows, mx_pitch(cols) // 2, dtype=torch.uint8, device='cuda'),
                torch.zeros(L.a4c_mx_scale_bytes(rows, cols), dtype=torch.uint8, device='cuda'))

    g, u, w = weight(wg), weight(wu), weight(wd)
    bias = [vec(b) for b in (bg, bu, bd)]
    p = [None if b is None else b.data_ptr() for b in bias]
    xq, hq = new(m, d), new(m, n)
    y = torch.empty(m, d, dtype=td, device='cuda')
    xd = x.to(td).cuda().contiguous()
    a4c.check(L.a4c_quantize_mx(xd.data_ptr(), f, d, *args(xq), m, d, s), 'q')
    act = {'silu': 2, 'gelu': 3}[activation]
    if chain:
        a4c.check(L.a4c_gated_dense_mx(*args(xq), *args(g), *args(u), p[0], p[1], hq[0].data_ptr(), 3, mx_pitch(n), hq[1].data_ptr(), m, d, n, act, s), 'g')
    else:
        h = torch.empty(m, n, dtype=td, device='cuda')
        a4c.check(L.a4c_gated_dense_mx(*args(xq), *args(g), *args(u), p[0], p[1], h.data_ptr(), f, n, None, m, d, n, act, s), 'g')
        a4c.check(L.a4c_quantize_mx(h.data_ptr(), f, n, *args(hq), m, n, s), 'q')
    a4c.check(L.a4c_dense_mx(*args(hq), *args(w), p[2], y.data_ptr(), f, d, None, m, n, d, 0, s), 'd')
    torch.cuda.synchronize()
    return y.float().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize('m,d,f', [(1, 64, 96), (5, 100, 333), (300, 256, 1024)])
@pytest.mark.parametrize('precision', [BF16, F32])
@pytest.mark.parametrize('chain', [True, False])
def test_block_equals_its_calls(m, d, f, precision, chain):
    import torch

    act = 'silu' if m != 5 else 'gelu'
    b, weights = feed_forward(m, d, f, precision, act, bias=m != 1, fusion={'mx_chain': chain}, residual=False)
    model = from_graph(b)
    model.compile()
    kinds = [op['kind'] for op in model.plan.ops]
    assert kinds == ['quantize_mx', 'gated_dense_mx'] + ([] if chain else ['quantize_mx']) + ['dense_mx']
    assert ('gate_up_out' in model.plan.buffers) == (not chain)
    x = torch.from_numpy(np.random.default_rng(m).standard_normal((m, d)).astype(np.float32))
    got = model.predict(x.numpy())
    assert np.array_equal(got, by_calls(x, weights, act, precision.format.value, chain))
    (want,) = oracle.run_plan(model.export_plan(), {'x': x.to(torch.bfloat16).float().numpy() if precision is BF16 else x.numpy()}).values()
    assert np.allclose(got, want, rtol=1e-2, atol=5e-2)
    # captured and replayed: the same
    model.plan.capture()
    model.plan.run()
    assert np.array_equal(model.plan.tensor_of(b.graph.output_tensor_names[0]).float().cpu().numpy(), got)


@pytest.mark.gpu
def test_fanout_views_and_residual():
    """One input feeds two MXFP4 layers (quantised once), a column slice feeds a third, a Concat collects them, and the hidden
    tensor that is also a graph output keeps its float form."""
    rng = np.random.default_rng(3)
    m, d = 70, 128
    w0, w1, w2 = (rng.normal(0, 0.1, (d, 64)) for _ in range(3))
    ws = rng.normal(0, 0.1, (64, 64))
    b = GraphBuilder({'Part': 'cuda_b200'}, name='views')
    x = b.input('x', (m, d), BF16)
    y0 = b.dense('a', x, w0, MXFP4, BF16, relu=True)
    y1 = b.gated_dense('b', x, w1, w2, MXFP4, BF16, activation='gelu_tanh')
    left, _ = b.split('s', x, [64, 64])
    y2 = b.dense('c', left, ws, MXFP4, BF16)
    cat = b.concat('cat', [y0, y1, y2])
    b.output(b.dense('tail', cat, rng.normal(0, 0.1, (192, 40)), MXFP4, BF16))
    b.output(cat)
    model = from_graph(b)
    model.compile()
    assert [op['kind'] for op in model.plan.ops].count('quantize_mx') == 3
    xv = rng.standard_normal((m, d)).astype(np.float32)
    got = model.predict(xv)
    import torch

    want = oracle.run_plan(model.export_plan(), {'x': torch.from_numpy(xv).bfloat16().float().numpy()})
    for name in got:
        assert np.allclose(got[name], want[name], rtol=1e-2, atol=5e-2), name


@pytest.mark.gpu
def test_residual_block_streams_and_reports(tmp_path):
    from aie4ml_b200.report import profile_plan

    b, _ = feed_forward(64, 128, 256, BF16)
    b.ctx.aie_config['Iterations'] = 4
    model = from_graph(b)
    model.write()
    xs = np.random.default_rng(0).standard_normal((4, 64, 128)).astype(np.float32)
    out = model.predict(xs)                                   # four chunks through the host pipeline
    one, _ = feed_forward(64, 128, 256, BF16)
    single = from_graph(one)
    assert np.array_equal(out, np.concatenate([single.predict(x) for x in xs]))
    rows = {r['kind']: r for r in profile_plan(single.plan, iters=2)}
    assert rows['gated_dense_mx']['ops'] == 4 * 64 * 128 * 256 and rows['quantize_mx']['bytes'] > 64 * 128 * 2
    assert model.dump(tmp_path).exists()
