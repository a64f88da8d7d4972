"""The linear-attention layers' operators on the GPU against oracle/delta.py.

u = 2^-24; a result of 16 bits adds half a step of its type.

Convolution: width products and sums, the bias: (width + 1) u of the sum of the
terms' sizes, which silu passes on with a slope below 1.1, and 6 u of the result
for the exponential, the sum and the quotient.

Rule: with keys of at most unit length and 0 <= beta <= 1 a step's map of the state
is e^g times a contraction, so what a token rounds is not enlarged by the tokens
behind it. A token rounds each state value three times (the factor, its product,
the update: 2 u, u, u / 2 at most, as random signs), and its prediction and output
are sums of key_dim products: as independent roundings sqrt(key_dim) u of the
products' 2-norm, which is at most the state's norm times |k^| or |q^| (the sum
itself may cancel to nothing, so it is no measure), with a few u from the norms and
the gates. So with s_t the larger norm of the state after the decay and after the
update, in u: r_t = (2 sqrt(key_dim) + 16) s_t is what token t rounds, and E_t^2 =
(e^g E_(t-1))^2 + r_t^2 bounds the state, scale (E_t + r_t) the output, in 2-norms.

Norm: the mean square is off by at most (32 + 8) u where no lane sums more than 32
squares and the rest is a tree; half of it reaches the root; root, quotient, two
products 4 u; the gate 8 u more; residual's addition u of |x| + |residual|, to
which the norm holds y relative through h: (40) u of the row's largest |y| in all."""
import numpy as np
import pytest

from oracle import delta as odelta
from oracle import quant

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ['float32', 'float16', 'bfloat16']
HALF = {'float32': U, 'float16': 2.0 ** -11, 'bfloat16': 2.0 ** -8}
# what a type's smallest step adds where values are subnormal in it
FLOOR = {'float32': 2.0 ** -149, 'float16': 2.0 ** -25, 'bfloat16': 2.0 ** -134}


def _t(x, dtype='float32'):
    import torch
    return torch.tensor(np.asarray(x, dtype=np.float32)).to(getattr(torch, dtype)).cuda()


def _ints(x):
    import torch
    return torch.tensor(np.asarray(x, dtype=np.int32), device='cuda')


def _np(t):
    return t.detach().double().cpu().numpy()


def _random(rng, shape, dtype):
    """A device tensor and its exact values."""
    t = _t(rng.standard_normal(shape), dtype)
    return t, _np(t)


def _layout(rng, counts, spare=2):
    """starts and slots (shuffled rows of a pool) of requests with `counts` new tokens."""
    starts = np.concatenate([[0], np.cumsum(counts)])
    return starts, rng.permutation(len(counts) + spare)[:len(counts)]


# ---------------------------------------------------------------- convolution

CONV_COUNTS = [[1], [1, 1, 1], [33, 0, 1, 2, 3, 31, 32, 64, 65], [0, 0, 200], [2, 300, 0]]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [2, 4, 8])
@pytest.mark.parametrize('counts', CONV_COUNTS, ids=str)
@pytest.mark.parametrize('channels', [1, 100, 1027, 2048])
def test_conv(dtype, width, counts, channels):
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(channels + width + sum(counts))
    starts, slots = _layout(rng, counts)
    tokens, n = starts[-1], len(counts)
    pad = 3
    x, xv = _random(rng, (tokens + pad, channels), dtype)
    w, wv = _random(rng, (channels, width), 'float32')
    state, sv = _random(rng, (n + 2, width - 1, channels), 'float32')
    old = rng.integers(0, 2, n) * 7
    bias, bv = _random(rng, channels, 'float32') if width == 4 else (None, None)
    out = torch.full_like(x, 7.0)
    y = delta.conv(x, w, state, _ints(slots), _ints(starts), _ints(old + counts), bias=bias, silu=width != 2, out=out)
    assert y is out
    got, after = _np(out), sv.copy()
    assert (got[tokens:] == 7).all()
    for b, c in enumerate(counts):
        if not c:
            continue
        rows = slice(starts[b], starts[b] + c)
        before = sv[slots[b]] if old[b] else np.zeros_like(sv[0])
        want, after[slots[b]], size = odelta.conv(before, xv[rows], wv, bv, silu=width != 2)
        assert (np.abs(got[rows] - want) <= 1.1 * (width + 1) * U * size + (6 * U + HALF[dtype]) * np.abs(want)
                + FLOOR[dtype]).all()
    np.testing.assert_array_equal(_np(state), after)     # rows kept, and other requests' untouched


@pytest.mark.parametrize('dtype', TYPES)
def test_conv_step_with_empty_places_and_views(dtype):
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(5)
    n, channels = 7, 260
    wide, _ = _random(rng, (n, channels + 12), dtype)
    x, slots = wide[:, 4:4 + channels], [3, -1, 0, 9, 6, 2, 5]      # -1, 9: outside the pool of 7
    w, wv = _random(rng, (channels, 4), 'float32')
    state, sv = _random(rng, (7, 3, channels), 'float32')
    out = torch.full((n, channels + 3), 7.0, dtype=x.dtype, device='cuda')[:, :channels]
    delta.conv(x, w, state, _ints(slots), lengths=_ints([1, 1, 5, 5, 5, 1, 5]), out=out)
    xv, got, after = _np(x), _np(out), sv.copy()
    for b, s in enumerate(slots):
        if not 0 <= s < 7:
            assert (got[b] == 7).all()
            continue
        before = np.zeros_like(sv[0]) if b in (0, 5) else sv[s]
        want, after[s], size = odelta.conv(before, xv[b:b + 1], wv)
        assert (np.abs(got[b] - want[0]) <= 6 * U * size[0] + (6 * U + HALF[dtype]) * np.abs(want[0]) + FLOOR[dtype]).all()
    np.testing.assert_array_equal(_np(state), after)


# ---------------------------------------------------------------- gated delta rule

def _rule_inputs(rng, tokens, heads, dtype, projected):
    hk, hv, kd, vd = heads
    wide, _ = _random(rng, (tokens, 2 * hk * kd + hv * vd + 8), dtype)       # views of one projection
    q, k, v = wide[:, :hk * kd], wide[:, hk * kd:2 * hk * kd], wide[:, 2 * hk * kd:2 * hk * kd + hv * vd]
    q, k, v = (x.unflatten(-1, (-1, d)) for x, d in ((q, kd), (k, kd), (v, vd)))
    both = _t(rng.standard_normal((tokens, 2 * hv + 1)))
    decay, beta = both[:, :hv], both[:, hv:2 * hv]
    a = dt = None
    if projected:
        a, dt = _t(-rng.uniform(0.01, 8, hv)), _t(rng.uniform(-6, 0, hv))
    else:
        decay, beta = -_t(rng.exponential(0.2, (tokens, hv))), _t(rng.random((tokens, hv)))
    return q, k, v, decay, beta, a, dt


def _opt(t):
    return None if t is None else _np(t)


def _check_rule(heads, counts, dtype, projected, order, norm_eps=1e-6, scale=None, spare=2, pad=2, old=None, step=False):
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(sum(heads) + sum(counts) + len(counts))
    starts, slots = _layout(rng, counts, spare)
    tokens, n = int(starts[-1]), len(counts)
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, tokens + pad, heads, dtype, projected)
    if norm_eps is None:
        q, k = q * 0.05, k * 0.05
    state, sv = _random(rng, (n + spare, heads[1], heads[2], heads[3]), 'float32')
    if old is None:
        old = rng.integers(0, 2, n) * 9
    out = torch.full((tokens + pad, heads[1], heads[3]), 7.0, dtype=v.dtype, device='cuda')
    y = delta.rule(q, k, v, decay, beta, state, _ints(slots), None if step else _ints(starts), _ints(old + np.asarray(counts)),
                   a, dt, order, norm_eps, scale, out)
    assert y is out
    got, after, want = _np(out), sv.copy(), np.full(out.shape, 7.0)
    qv, kv, vv, dv, bv, av, tv = (_opt(x) for x in (q, k, v, decay, beta, a, dt))
    for b, c in enumerate(counts):
        if c:
            rows = slice(starts[b], starts[b] + c)
            before = sv[slots[b]] if old[b] else np.zeros_like(sv[0])
            sizes = np.zeros((c, heads[1]))
            want[rows], after[slots[b]] = odelta.rule(before, qv[rows], kv[rows], vv[rows], dv[rows], bv[rows], av, tv,
                                                      order, norm_eps, scale, sizes)
            rounds = (2 * heads[2] ** 0.5 + 16) * U * sizes
            off, off_out = np.zeros(heads[1]), np.zeros(heads[1])
            for f, r in zip(np.exp(odelta.gates(dv[rows], bv[rows], av, tv)[0]), rounds):
                off = np.hypot(f * off, r)
                off_out += (off + r) ** 2
            off_out = np.sqrt(off_out) * (heads[2] ** -0.5 if scale is None else abs(scale))
            for h in range(heads[1]):
                err = np.linalg.norm(got[rows, h] - want[rows, h])
                assert err <= off_out[h] + HALF[dtype] * np.linalg.norm(want[rows, h]), ('out', b, h)
                err = np.linalg.norm(_np(state[slots[b], h]) - after[slots[b], h])
                assert err <= off[h], ('state', b, h)
    assert (got[tokens:] == 7).all()
    idle = sorted(set(range(n + spare)) - {int(s) for s, c in zip(slots, counts) if c})
    np.testing.assert_array_equal(_np(state)[idle], sv[idle])


HEADS = [(2, 4, 128, 128), (1, 3, 64, 64), (3, 3, 64, 16), (1, 2, 256, 256), (2, 2, 128, 48), (1, 1, 128, 1024)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', HEADS, ids=str)
@pytest.mark.parametrize('n', [1, 3, 70])
def test_rule_step(n, heads, dtype):
    if n == 70 and heads[3] > 128:
        n = 9
    _check_rule(heads, [1] * n, dtype, projected=n != 3, order='tiled' if n == 3 else 'grouped', pad=0, step=True)


def test_rule_step_of_many_heads():
    """Every width of a workgroup's columns."""
    for heads, n in [((16, 32, 128, 128), 1), ((16, 32, 128, 128), 9), ((16, 32, 128, 128), 30), ((2, 4, 128, 64), 200)]:
        _check_rule(heads, [1] * n, 'float32', True, 'grouped', pad=0, step=True)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', HEADS, ids=str)
@pytest.mark.parametrize('counts', [[1], [2], [17], [63], [64], [65], [200], [5, 0, 1, 130, 16, 64, 0, 3]], ids=str)
def test_rule_prompts(counts, heads, dtype):
    _check_rule(heads, counts, dtype, projected=True, order='grouped')


@pytest.mark.parametrize('counts', [[130], [1, 70, 0, 33]], ids=str)
@pytest.mark.parametrize('old', [0, 9])
def test_rule_prompts_with_given_gates_and_keys(counts, old):
    _check_rule((2, 6, 128, 128), counts, 'float32', False, 'tiled', norm_eps=None, scale=0.7,
                old=np.full(len(counts), old))
    _check_rule((2, 6, 64, 128), counts, 'bfloat16', False, 'tiled', norm_eps=1e-3, scale=-2.0,
                old=np.full(len(counts), old))


def test_rule_many_requests():
    rng = np.random.default_rng(1)
    _check_rule((1, 2, 64, 32), rng.integers(0, 90, 150).tolist(), 'float32', True, 'grouped')
    _check_rule((1, 2, 64, 32), [0] * 64 + [70] + [0] * 63 + [1, 100], 'float32', True, 'grouped')


def test_rule_long_prompt():
    _check_rule((1, 2, 128, 32), [3000], 'float32', True, 'grouped')


# ---------------------------------------------------------------- norm

def _check_norm(shape, dtype, out_type, residual, gate, eps=1e-6, cut=0):
    import torch
    from localai_amd import dequant, layer
    rng = np.random.default_rng(sum(shape))
    dim = shape[-1]
    wide = shape[:-1] + (dim + cut,)
    x, _ = _random(rng, wide, dtype)
    x = x[..., cut:]
    w, wv = _random(rng, dim, 'float32')
    r, rv = _random(rng, shape, 'float32') if residual else (None, None)
    z, zv = _random(rng, shape, dtype) if gate else (None, None)
    y = layer.rms_norm(x, w, eps, residual=r, gate=z, dtype=out_type if out_type == 'q8_0' else getattr(torch, out_type))
    xv = _np(x)
    want, h = odelta.rms_norm(xv, wv, eps, rv, zv)
    if residual:
        assert (np.abs(_np(r) - h) <= U * np.abs(h)).all()
    tol = 48 * U * np.abs(want).max(-1, keepdims=True)
    if out_type != 'q8_0':
        assert (np.abs(_np(y) - want) <= tol + HALF[out_type] * np.abs(want) + FLOOR[out_type]).all()
        return
    assert y.shape == (*shape[:-1], dim // 32 * 34) and y.dtype == torch.uint8
    got = np.asarray(quant.dequantize(y.cpu().numpy().tobytes(), 8, shape), np.float64)
    np.testing.assert_array_equal(got, _np(dequant.dequantize_device(y, 8, shape)))
    d = np.repeat(odelta.q8_0(want)[0].astype(np.float64), 32, -1).reshape(shape)
    # half a step of the scale, and the scale's own half step of 2^-11 at 127 times it
    assert (np.abs(got - want) <= d * (0.5 + 127 * 2.0 ** -11) * (1 + 2.0 ** -9) + tol).all()
    blocks = y.cpu().numpy().reshape(-1, 34)
    quants = blocks[:, 2:].view(np.int8)
    assert (np.abs(quants).max(-1) == 127).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('out_type', [*TYPES, 'q8_0'])
@pytest.mark.parametrize('shape', [(1, 64), (5, 256), (3, 1024), (2, 4096), (7, 5120), (2, 20000 // 32 * 32)], ids=str)
@pytest.mark.parametrize('residual', [False, True])
def test_norm(shape, dtype, out_type, residual):
    _check_norm(shape, dtype, out_type, residual, gate=False)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('out_type', [*TYPES, 'q8_0'])
@pytest.mark.parametrize('shape', [(1, 1, 128), (3, 5, 64), (70, 32, 128), (2, 3, 256)], ids=str)
def test_norm_gated(shape, dtype, out_type):
    _check_norm(shape, dtype, out_type, False, gate=True)
    _check_norm(shape, dtype, out_type, True, gate=True, cut=32)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [1, 2, 3, 63, 65, 255, 257, 1023, 1025, 4099, 9999])
def test_norm_of_odd_rows(dtype, dim):
    _check_norm((3, dim), dtype, 'float32', True, gate=True, eps=1e-3)
    _check_norm((3, dim), dtype, dtype, False, gate=False, cut=1)


def test_norm_in_place_and_of_zeros():
    import torch
    from localai_amd import layer
    rng = np.random.default_rng(0)
    x, xv = _random(rng, (9, 2048), 'bfloat16')
    w, wv = _random(rng, 2048, 'float32')
    want = layer.rms_norm(x, w)
    assert layer.rms_norm(x, w, out=x) is x and torch.equal(x, want)
    zeros = torch.zeros(2, 64, device='cuda')
    assert not layer.rms_norm(zeros, w[:64]).any()
    assert not layer.rms_norm(zeros, w[:64], dtype='q8_0').any()
    assert layer.rms_norm(zeros[:0], w[:64]).shape == (0, 64)


def test_norm_blocks_of_values_that_are_not_finite():
    from localai_amd import dequant, layer
    import torch
    x = torch.ones(3, 96, device='cuda')
    x[0, 5], x[1, 40] = float('nan'), float('inf')
    gate = torch.ones_like(x)
    gate[2, 70] = float('nan')
    y = _np(dequant.dequantize_device(layer.rms_norm(x, torch.ones(96, device='cuda'), gate=gate, dtype='q8_0'), 8, (3, 96)))
    assert np.isnan(y[0]).all()                                              # the row's norm is NaN
    assert np.isnan(y[1, 32:64]).all() and (y[1, :32] == 0).all() and (y[1, 64:] == 0).all()
    assert np.isnan(y[2, 64:]).all() and np.isfinite(y[2, :64]).all()
