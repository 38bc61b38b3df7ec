"""Cases that measure the microscaled 4-bit (MXFP4) operators: quantise / dequantise, Dense, gated Dense, and the
feed-forward block they form together.

MXFP4: blocks of 32 values along a row share a power-of-two scale 2**(s - 127) held in one byte (s = 255: not a number); each value is a
4-bit E2M1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign bit), two to a byte, the even column in the low nibble.  Rows of codes start on 16
bytes.  Scales are stored in tiles of 128 rows x 4 blocks (512 bytes): byte (r % 32) * 16 + (r // 32) * 4 + b of a tile belongs to its row r and
block b; tiles of a row group follow one another along the row; places beyond the tensor hold 0.

With ``own`` false, ``run`` computes each operator from elementary torch operations in 32 bits; with ``own`` true it makes the calls
of the framework's C interface that a user's program makes.
"""

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'f32': torch.float32}
FCODE = {'bf16': 0, 'f32': 1, 'mxfp4': 3}
ACTS = {'none': 0, 'relu': 1, 'silu': 2, 'gelu': 3, 'gelu_tanh': 4, 'sigmoid': 5}


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # one token's activations on their way into a 4-bit layer, and back
        {'name': 'round_token', 'op': 'round', 'rows': 1, 'cols': 4096, 'dtype': 'bf16'},
        # an odd batch of float32 features whose last block is ragged
        {'name': 'round_ragged', 'op': 'round', 'rows': 777, 'cols': 1000, 'dtype': 'f32'},
        # a prefill's activations, or a weight matrix of a large layer
        {'name': 'round_large', 'op': 'round', 'rows': 65536, 'cols': 4096, 'dtype': 'bf16'},
        # decoding one token: the weights are read for one row
        {'name': 'dense_token', 'op': 'dense', 'm': 1, 'k': 4096, 'n': 4096, 'relu': False, 'bias': True, 'dtype': 'bf16'},
        # nothing is a multiple of a tile
        {'name': 'dense_ragged', 'op': 'dense', 'm': 333, 'k': 1000, 'n': 777, 'relu': True, 'bias': True, 'dtype': 'bf16'},
        # a batch of 1024 rows, a size of the int8 Dense sweep
        {'name': 'dense_batch', 'op': 'dense', 'm': 1024, 'k': 4096, 'n': 4096, 'relu': True, 'bias': True, 'dtype': 'bf16'},
        # the large end of the same sweep
        {'name': 'dense_large', 'op': 'dense', 'm': 16384, 'k': 8192, 'n': 8192, 'relu': False, 'bias': False, 'dtype': 'bf16'},
        # a few sequences decoding together
        {'name': 'gated_token', 'op': 'gated', 'm': 4, 'k': 4096, 'n': 8192, 'act': 'silu', 'bias': False, 'dtype': 'bf16'},
        # a short prompt on a narrow model, with biases
        {'name': 'gated_prompt', 'op': 'gated', 'm': 1000, 'k': 1024, 'n': 4096, 'act': 'gelu_tanh', 'bias': True, 'dtype': 'bf16'},
        # a long prefill
        {'name': 'gated_large', 'op': 'gated', 'm': 16384, 'k': 4096, 'n': 8192, 'act': 'silu', 'bias': False, 'dtype': 'bf16'},
        # the whole block, 16 sequences decoding together
        {'name': 'ffn_decode', 'op': 'ffn', 'm': 16, 'k': 4096, 'n': 8192, 'act': 'silu', 'bias': False, 'dtype': 'bf16'},
        # the encoder block's feed-forward sizes (256 -> 1024 -> 256) over 512 sequences of 128
        {'name': 'ffn_encoder', 'op': 'ffn', 'm': 65536, 'k': 256, 'n': 1024, 'act': 'gelu', 'bias': True, 'dtype': 'bf16'},
    ]


def _spread(rng, lo, hi):
    """Log-uniform whole number; half of them multiples of 32, the others as they come."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and hi >= 32:
        v = max(32, v // 32 * 32)
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(('round', 'dense', 'gated', 'ffn'))
    dtype = 'bf16'
    if op == 'round':
        dtype = rng.choice(('bf16', 'f32'))
        rows, cols = int(65536 ** rng.random()), _spread(rng, 1, 8192)
        return {'op': op, 'rows': rows, 'cols': cols, 'dtype': dtype}
    while True:
        m, k, n = int(16384 ** rng.random()), _spread(rng, 17, 8192), _spread(rng, 1 if op == 'dense' else 64, 8192)
        if m * k * n * (1 if op == 'dense' else 2 if op == 'gated' else 3) <= 16384 * 8192 * 8192:
            break
    if op == 'dense':
        return {'op': op, 'm': m, 'k': k, 'n': n, 'relu': rng.random() < 0.5, 'bias': rng.random() < 0.5, 'dtype': dtype}
    return {'op': op, 'm': m, 'k': k, 'n': n, 'act': rng.choice(sorted(ACTS)), 'bias': rng.random() < 0.5, 'dtype': dtype}


def _mx_bytes(rows, cols):
    return rows * ((cols + 1) // 2) + rows * ((cols + 31) // 32)


def work(case):
    if case['op'] == 'round':
        size, n = (2 if case['dtype'] == 'bf16' else 4), case['rows'] * case['cols']
        return {'bytes': 2 * n * size + 2 * _mx_bytes(case['rows'], case['cols']), 'flops': 0}
    m, k, n = case['m'], case['k'], case['n']
    if case['op'] == 'dense':
        return {'bytes': _mx_bytes(m, k) + _mx_bytes(n, k) + 2 * m * n + (4 * n if case['bias'] else 0), 'flops': 2 * m * k * n}
    if case['op'] == 'gated':
        return {'bytes': _mx_bytes(m, k) + 2 * _mx_bytes(n, k) + 2 * m * n + (8 * n if case['bias'] else 0), 'flops': 4 * m * k * n}
    return {'bytes': 4 * m * k + 2 * _mx_bytes(n, k) + _mx_bytes(k, n) + (8 * n + 4 * k if case['bias'] else 0), 'flops': 6 * m * k * n}


# ---- inputs --------------------------------------------------------------------------------------

def _pad(n, to):
    return (n + to - 1) // to * to


def _scale_bytes(rows, cols):
    return _pad(rows, 128) // 128 * (_pad(cols, 128) // 128) * 512


def _pack(x):
    """float32 [rows, cols] -> (codes [rows, 16-byte pitch], scale tiles): what a program has in hand after quantising a tensor once."""
    rows, cols = x.shape
    blocks = _pad(cols, 32) // 32
    v = torch.zeros(rows, blocks * 32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, 32)
    e = torch.frexp(v.abs().amax(2))[1] - 3
    v = torch.ldexp(v, -e[:, :, None])
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)     # all borders but .75, 1.75, 3.5 go down
    a = v.abs()
    code = sum((a >= m if i % 2 else a > m).to(torch.uint8) for i, m in enumerate(mids))
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(rows, blocks * 32)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    tiles = torch.zeros(_pad(rows, 128), _pad(blocks, 4), dtype=torch.uint8, device=x.device)
    tiles[:rows, :blocks] = (e + 127).clamp(0, 254).to(torch.uint8)
    tiles = tiles.view(-1, 4, 32, tiles.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()
    return codes.contiguous(), tiles


def _activations(g, rows, cols):
    """Normal values with a few channels that are several times larger, and one row in 64 that is nearly silent."""
    x = torch.randn(rows, cols, generator=g, device='cuda')
    x *= torch.where(torch.rand(cols, generator=g, device='cuda') < 0.01, 8.0, 1.0)
    x *= torch.where(torch.rand(rows, 1, generator=g, device='cuda') < 1 / 64, 1e-3, 1.0)
    return x


def _weights(g, rows, cols):
    return _pack(torch.randn(rows, cols, generator=g, device='cuda') * cols ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    s = {'case': dict(case)}
    dt = DTYPES[case['dtype']]

    def buffer(rows, cols):
        return (torch.empty(rows, _pad(cols, 32) // 2, dtype=torch.uint8, device='cuda'),
                torch.empty(_scale_bytes(rows, cols), dtype=torch.uint8, device='cuda'))

    def bias(n):
        return torch.randn(n, generator=g, device='cuda') * 0.1 if case['bias'] else None

    if case['op'] == 'round':
        rows, cols = case['rows'], case['cols']
        s['x'] = _activations(g, rows, cols).to(dt)
        s['q'] = buffer(rows, cols)
        s['y'] = torch.empty(rows, cols, dtype=dt, device='cuda')
        return s
    m, k, n = case['m'], case['k'], case['n']
    if case['op'] == 'dense':
        s['a'], s['w'], s['b'] = _pack(_activations(g, m, k)), _weights(g, n, k), bias(n)
        s['y'] = torch.empty(m, n, dtype=dt, device='cuda')
        return s
    s['wg'], s['wu'], s['bg'], s['bu'] = _weights(g, n, k), _weights(g, n, k), bias(n), bias(n)
    if case['op'] == 'gated':
        s['a'] = _pack(_activations(g, m, k))
        s['y'] = torch.empty(m, n, dtype=dt, device='cuda')
        return s
    s['x'] = _activations(g, m, k).to(dt)
    s['wd'], s['bd'] = _weights(g, k, n), bias(k)
    s['a'], s['h'] = buffer(m, k), buffer(m, n)
    s['y'] = torch.empty(m, k, dtype=dt, device='cuda')
    return s


# ---- the plain form ------------------------------------------------------------------------------

def _values(packed, rows, cols):
    """Codes and scale tiles -> float32 values."""
    codes, tiles = packed
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), 2).long()].view(rows, -1, 32)
    groups, across = _pad(rows, 128) // 128, _pad(cols, 128) // 128
    s = tiles.view(groups, across, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(groups * 128, across * 4)[:rows, :v.shape[1]]
    scale = torch.ldexp(torch.ones_like(s, dtype=torch.float32), s.int() - 127)
    scale = torch.where(s == 255, torch.nan, scale)
    return (v * scale[:, :, None]).view(rows, -1)[:, :cols]


def _rounded(x):
    """float32 [rows, cols] -> the values its MXFP4 form stands for."""
    rows, cols = x.shape
    blocks = _pad(cols, 32) // 32
    v = x
    if cols % 32:
        v = torch.zeros(rows, blocks * 32, device=x.device)
        v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    top = v.abs().amax(2, keepdim=True)
    e = (torch.frexp(top)[1] - 3).clamp(min=-127)
    v = torch.ldexp(v, -e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    out = torch.ldexp(torch.copysign(a, v), e)
    out = torch.where(torch.isfinite(top), out, torch.nan)
    return out.view(rows, -1)[:, :cols]


def _activate(x, act):
    if act == 'relu':
        return torch.where(x < 0, 0.0, x)
    if act == 'silu':
        return x / (1 + torch.exp(-x))
    if act == 'sigmoid':
        return 1 / (1 + torch.exp(-x))
    if act == 'gelu':
        return 0.5 * x * (1 + torch.erf(x * 0.7071067811865476))
    if act == 'gelu_tanh':
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


def _plus(y, b):
    return y if b is None else y + b


def _plain(s):
    c = s['case']
    dt = DTYPES[c['dtype']]
    if c['op'] == 'round':
        return _rounded(s['x'].float()).to(dt)
    m, k, n = c['m'], c['k'], c['n']
    if c['op'] == 'dense':
        y = _plus(_values(s['a'], m, k) @ _values(s['w'], n, k).T, s['b'])
        return _activate(y, 'relu' if c['relu'] else 'none').to(dt)
    a = _values(s['a'], m, k) if c['op'] == 'gated' else _rounded(s['x'].float())
    h = _activate(_plus(a @ _values(s['wg'], n, k).T, s['bg']), c['act']) * _plus(a @ _values(s['wu'], n, k).T, s['bu'])
    if c['op'] == 'gated':
        return h.to(dt)
    return _plus(_rounded(h) @ _values(s['wd'], k, n).T, s['bd']).to(dt)


# ---- the framework's calls -----------------------------------------------------------------------

_a4c = None


def _own(s):
    global _a4c
    if _a4c is None:
        from aie4ml_b200 import lib
        _a4c = lib
    lib, check = _a4c.load(), _a4c.check
    c = s['case']
    stream = torch.cuda.current_stream().cuda_stream
    y, f = s['y'], FCODE[c['dtype']]

    def ptr(t):
        return None if t is None else t.data_ptr()

    def mx(q):
        return q[0].data_ptr(), 2 * q[0].shape[1], q[1].data_ptr()     # codes, pitch in elements, scales

    if c['op'] == 'round':
        x, (q, ldq, sc) = s['x'], mx(s['q'])
        check(lib.a4c_quantize_mx(x.data_ptr(), f, x.stride(0), q, ldq, sc, c['rows'], c['cols'], stream), 'quantize')
        check(lib.a4c_dequantize_mx(q, ldq, sc, y.data_ptr(), f, y.stride(0), c['rows'], c['cols'], stream), 'dequantize')
        return y
    m, k, n = c['m'], c['k'], c['n']
    if c['op'] == 'dense':
        check(lib.a4c_dense_mx(*mx(s['a']), *mx(s['w']), ptr(s['b']), y.data_ptr(), f, n, None, m, k, n, int(c['relu']), stream), 'dense')
        return y
    if c['op'] == 'gated':
        check(lib.a4c_gated_dense_mx(*mx(s['a']), *mx(s['wg']), *mx(s['wu']), ptr(s['bg']), ptr(s['bu']), y.data_ptr(), f, n, None, m, k, n,
                                     ACTS[c['act']], stream), 'gated dense')
        return y
    x, (h, ldh, hs) = s['x'], mx(s['h'])
    check(lib.a4c_quantize_mx(x.data_ptr(), f, x.stride(0), *mx(s['a']), m, k, stream), 'quantize')
    check(lib.a4c_gated_dense_mx(*mx(s['a']), *mx(s['wg']), *mx(s['wu']), ptr(s['bg']), ptr(s['bu']), h, FCODE['mxfp4'], ldh, hs, m, k, n,
                                 ACTS[c['act']], stream), 'gated dense')
    check(lib.a4c_dense_mx(h, ldh, hs, *mx(s['wd']), ptr(s['bd']), y.data_ptr(), f, k, None, m, n, k, 0, stream), 'dense')
    return y


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definition, in 64 bits -------------------------------------------------------------

def _decode64(packed, rows, cols):
    """Field by field: sign, two exponent bits, one mantissa bit; the scale's byte is looked up at its own address."""
    codes, tiles = packed
    col = torch.arange(cols, device=codes.device)
    row = torch.arange(rows, device=codes.device)
    byte = codes[:, col // 2].int()
    c = torch.where(col % 2 == 0, byte & 15, byte >> 4)
    exp, man = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(exp == 0, man * 0.5, (1 + man * 0.5) * torch.exp2((exp - 1).double()))
    blk = torch.arange((cols + 31) // 32, device=codes.device)
    tile = (row[:, None] // 128) * ((cols + 127) // 128) + blk[None] // 4
    s = tiles[tile * 512 + (row[:, None] % 32) * 16 + (row[:, None] % 128) // 32 * 4 + blk[None] % 4].double()
    scale = torch.exp2(s - 127)[:, col // 32]
    return torch.where(c & 8 != 0, -mag, mag) * scale


def _quantise64(x):
    """Nearest of the sixteen values, ties to the even code, block by block."""
    rows, cols = x.shape
    full = (cols + 31) // 32 * 32
    v = torch.nn.functional.pad(x, (0, full - cols)).view(rows, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    # floor(log2): the logarithm may be a hair off at powers of two, so it is put right by comparison
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    e = torch.where(top > 0, e - 2, -127.0).clamp(min=-127)
    a = (v * torch.exp2(-e)).abs()
    q = torch.zeros_like(a)
    for lower, upper, to_upper_on_tie in ((0.0, 0.5, False), (0.5, 1.0, True), (1.0, 1.5, False), (1.5, 2.0, True), (2.0, 3.0, False),
                                          (3.0, 4.0, True), (4.0, 6.0, False)):
        mid = (lower + upper) / 2
        q = torch.where(a >= mid if to_upper_on_tie else a > mid, upper, q)
    return (torch.sign(v) * q * torch.exp2(e)).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'round':
        return _quantise64(s['x'].double())
    m, k, n = case['m'], case['k'], case['n']

    def linear(a, w, rows, cols, b):
        y = torch.matmul(a, _decode64(w, rows, cols).t())
        return y if b is None else y + b.double()

    if case['op'] == 'dense':
        y = linear(_decode64(s['a'], m, k), s['w'], n, k, s['b'])
        return y.clamp(min=0) if case['relu'] else y
    a = _decode64(s['a'], m, k) if case['op'] == 'gated' else _quantise64(s['x'].double())
    g = linear(a, s['wg'], n, k, s['bg'])
    act = case['act']
    if act == 'relu':
        g = g.clamp(min=0)
    elif act == 'silu':
        g = g * torch.special.expit(g)
    elif act == 'sigmoid':
        g = torch.special.expit(g)
    elif act == 'gelu':
        g = g * torch.special.ndtr(g)
    elif act == 'gelu_tanh':
        g = g * torch.special.expit(2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))
    h = g.mul_(linear(a, s['wu'], n, k, s['bu']))
    if case['op'] == 'gated':
        return h
    return linear(_quantise64(h), s['wd'], k, n, s['bd'])
