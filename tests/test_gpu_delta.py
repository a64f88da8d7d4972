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
(e^g E_(t-1))^2 + r_t^2 bounds the state, scale (E_t + r_t) the output, in 2-norms. 64 tokens at once round each operand of a
product to 22 bits (2 u) instead, once, and sum 64 or key_dim products in fp32: of a
token's share fewer and no larger roundings than the three a token of its own.

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


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('counts', [[8], [9], [1, 2, 3], [8, 9, 10], [25, 0, 24, 7, 64]], ids=str)
def test_rule_few_tokens_a_request(counts, dtype):
    """On both sides of what goes token by token in a call of prompts."""
    _check_rule((2, 4, 128, 128), counts, dtype, True, 'tiled')


def test_rule_many_short_requests():
    rng = np.random.default_rng(3)
    _check_rule((1, 4, 64, 64), rng.integers(0, 40, 130).tolist(), 'bfloat16', True, 'grouped')
    _check_rule((1, 4, 64, 64), rng.integers(20, 30, 130).tolist(), 'float32', True, 'grouped')


def test_rule_step_of_many_requests():
    """The widest slices of columns."""
    _check_rule((2, 4, 128, 128), [1] * 520, 'float32', True, 'grouped', pad=0, step=True)


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


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [32, 64, 100, 128, 1032, 2056])
def test_norm_of_rows_at_any_alignment(dim, dtype):
    """Rows, gate, result and weight that begin 0, 1, 4 or 8 values behind an aligned place."""
    import torch
    from localai_amd import layer
    rng = np.random.default_rng(dim)
    base, bv = _random(rng, (5, 3, dim + 8), dtype)
    gate, gv = _random(rng, (5, 3, dim + 8), dtype)
    weight, wv = _random(rng, (dim + 8,), 'float32')
    for x0, g0, w0, o0 in [(0, 0, 0, 0), (8, 0, 4, 8), (4, 8, 0, 0), (0, 4, 4, 8), (8, 8, 1, 0), (1, 0, 0, 0), (0, 0, 0, 4)]:
        out = torch.full((5, 3, dim + 8), 3.0, dtype=base.dtype, device='cuda')
        view = out[..., o0:o0 + dim]
        layer.rms_norm(base[..., x0:x0 + dim], weight[w0:w0 + dim], 1e-6, gate=gate[..., g0:g0 + dim], out=view)
        want, _ = odelta.rms_norm(bv[..., x0:x0 + dim], wv[w0:w0 + dim], 1e-6, gate=gv[..., g0:g0 + dim])
        tol = 40 * U * np.abs(want).max(-1, keepdims=True) + HALF[dtype] * np.abs(want) * (1 + 40 * U) + FLOOR[dtype]
        assert (np.abs(_np(view) - want) <= tol).all(), (x0, g0, w0, o0)
        view[:] = 3.0
        assert (out == 3).all()


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


# ---------------------------------------------------------------- what the rule must not mix

def _finite_case(rng, tokens=150, heads=(2, 4, 128, 32)):
    import torch
    hk, hv, kd, vd = heads
    q, k, v = (torch.tensor(rng.standard_normal((tokens, h, d)), dtype=torch.float32, device='cuda')
               for h, d in ((hk, kd), (hk, kd), (hv, vd)))
    decay, beta = -_t(rng.exponential(0.1, (tokens, hv))), _t(rng.random((tokens, hv)))
    state = _t(rng.standard_normal((1, hv, kd, vd)))
    return q, k, v, decay, beta, state


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('where,value', [(w, float(x)) for w in ('q', 'k', 'v', 'decay', 'beta') for x in ('nan', 'inf', '-inf')
                                         if (w, x) != ('decay', '-inf')])     # (that one forgets everything: finite)
@pytest.mark.parametrize('at', [0, 70, 127])
def test_rule_values_that_are_not_finite_reach_only_what_follows(at, where, value, dtype):
    """Tokens before the one that holds it, heads that do not read it and, of a v, other columns are as without it."""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(at)
    q, k, v, decay, beta, state = _finite_case(rng)
    q, k, v = (x.to(getattr(torch, dtype)) for x in (q, k, v))
    starts = _ints([0, 150])
    call = lambda s: delta.rule(q, k, v, decay, beta, s, starts=starts, order='grouped')
    clean_state = state.clone()
    clean = call(clean_state)
    {'q': q, 'k': k, 'v': v, 'decay': decay, 'beta': beta}[where][(at, 1) if where in ('decay', 'beta') else (at, 0, 5)] = value
    got = call(state)
    heads = {'q': [0, 1], 'k': [0, 1], 'v': [0], 'decay': [1], 'beta': [1]}[where]     # two value heads a key head
    others = [h for h in range(4) if h not in heads]
    assert torch.equal(got[:, others], clean[:, others]) and torch.equal(state[:, others], clean_state[:, others])
    # the piece that holds it goes token by token: rounded elsewhere, no more than that
    near = dict(rtol=HALF[dtype] * 4 + 1e-5, atol=1e-5)
    torch.testing.assert_close(got[:at, heads].float(), clean[:at, heads].float(), **near)
    if where == 'q':
        if not np.isnan(value):
            return     # a norm that is infinite makes q zeros, but for 0 times infinity
        assert torch.isnan(got[at, heads]).all()
        torch.testing.assert_close(got[at + 1:, heads].float(), clean[at + 1:, heads].float(), **near)
        torch.testing.assert_close(state, clean_state, rtol=1e-4, atol=1e-5)
    elif where == 'v':
        columns = [c for c in range(32) if c != 5]
        torch.testing.assert_close(got[:, 0][:, columns].float(), clean[:, 0][:, columns].float(), **near)
        torch.testing.assert_close(state[0, 0][:, columns], clean_state[0, 0][:, columns], rtol=1e-4, atol=1e-5)
        assert not torch.isfinite(got[at:, 0, 5]).any() and not torch.isfinite(state[0, 0, :, 5]).any()
    elif where != 'k' or np.isnan(value):
        assert not torch.isfinite(got[at + 1:, heads]).any() and not torch.isfinite(state[0, heads]).any()


def _against_oracle(args, order='grouped', norm_eps=1e-6, tol=2e-5, starts=None):
    """One request; the 2-norms of output and state within tol of the oracle's largest state."""
    from localai_amd import delta
    q, k, v, decay, beta, state = args
    sizes = np.zeros((len(v), v.shape[1]))
    want, after = odelta.rule(_np(state)[0], _np(q), _np(k), _np(v), _np(decay), _np(beta), order=order, norm_eps=norm_eps,
                              sizes=sizes)
    got = delta.rule(q, k, v, decay, beta, state, starts=_ints([0, len(v)]), order=order, norm_eps=norm_eps)
    for h in range(v.shape[1]):
        assert np.linalg.norm(_np(got)[:, h] - want[:, h]) <= tol * np.linalg.norm(sizes[:, h]) * q.shape[-1] ** -0.5, h
        assert np.linalg.norm(_np(state)[0, h] - after[h]) <= tol * sizes[:, h].max(), h


# Tolerance of the cases below: a token rounds (2 sqrt(128) + 16) u = 2.3e-6 of its state, and what
# it rounds lasts no longer than the state itself, some tens of tokens here: within 2e-5.

def test_rule_forgets_everything():
    rng = np.random.default_rng(2)
    args = _finite_case(rng)
    args[3][40], args[3][64], args[3][100, 1] = -float('inf'), -float('inf'), -3e5
    _against_oracle(args)


def test_rule_equal_keys():
    """The least comfortable system: every k the same, beta 1, nothing forgotten (a sum of powers of A would cancel
    numbers of 1e18)."""
    rng = np.random.default_rng(3)
    q, k, v, decay, beta, state = _finite_case(rng)
    k[:] = k[0]
    decay[:], beta[:] = 0, 1
    _against_oracle((q, k, v, decay, beta, state))
    k[70:] = -k[70:]
    _against_oracle((q, k, v, decay, beta, state))


def test_rule_beta_zero_zero_keys_and_growth():
    rng = np.random.default_rng(4)
    q, k, v, decay, beta, state = _finite_case(rng)
    beta[:50] = 0
    k[60:70], q[65:75] = 0, 0
    decay[80:90] = 0.2      # a state that grows
    decay[130] = 1.5        # faster than a piece takes: token by token
    _against_oracle((q, k, v, decay, beta, state))


@pytest.mark.parametrize('size', [1e-20, 1e-3, 1e12, 3e19])
def test_rule_sizes(size):
    """v and the state of any size (past 1e30 in v or state: token by token)."""
    rng = np.random.default_rng(5)
    q, k, v, decay, beta, state = _finite_case(rng)
    _against_oracle((q * 1e3, k * 1e-3, v * size, decay, beta, state * size))


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('small', [1e-15, 1e-18, 1e-20, 1e-23])
def test_rule_small_keys_and_a_large_state(small, dtype):
    """Keys whose squares leave fp32's range, and a state whose products with them are far above v."""
    import torch
    rng = np.random.default_rng(7)
    q, k, v, decay, beta, state = _finite_case(rng)
    q, k, v = (x.to(getattr(torch, dtype)) for x in (q, k * small, v))
    # (the result's type adds its half step)
    _against_oracle((q, k, v, decay, beta, state * 1e25), tol=2e-5 + 2 * HALF[dtype])


def test_rule_keys_below_the_types_normal_values():
    """f16 keys and queries of a few of its smallest steps."""
    rng = np.random.default_rng(9)
    q, k, v, decay, beta, state = _finite_case(rng)
    _against_oracle(((q * 1e-6).half(), (k * 1e-6).half(), v.half(), decay, beta, state), norm_eps=1e-13, tol=2e-5 + 2 * HALF['float16'])


@pytest.mark.parametrize('dtype', TYPES)
def test_rule_state_values_that_no_key_meets(dtype):
    """One key value is zero in every k and q: what the state holds there, up to fp32's largest, reaches nothing."""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(8)
    q, k, v, decay, beta, state = _finite_case(rng)
    k[:, :, 5], q[:, :, 5] = 0, 0
    q, k, v = (x.to(getattr(torch, dtype)) for x in (q, k, v))
    decay *= 1e-3
    want_state = state.clone()
    state[:, :, 5] = 3e38
    want_state[:, :, 5] = 0
    starts = _ints([0, 150])
    want = delta.rule(q, k, v, decay, beta, want_state, starts=starts)
    got = delta.rule(q, k, v, decay, beta, state, starts=starts)
    # both within the tolerance above, which is of the norm of a head's state
    rows = [i for i in range(128) if i != 5]
    size = want_state.norm(dim=(2, 3)).max().item()
    assert (state - want_state)[:, :, rows].norm().item() <= 4e-5 * 2 * size
    assert (got.float() - want.float()).norm().item() <= 2 * (2e-5 + 2 * HALF[dtype]) * (want.float().norm().item() + size)


def test_rule_large_betas():
    """beta |k|^2 past 2 (a state that overshoots) goes token by token."""
    rng = np.random.default_rng(6)
    q, k, v, decay, beta, state = _finite_case(rng, tokens=70)
    k /= k.norm(dim=-1, keepdim=True)
    beta[20:23] = 4.0
    # an error of these three tokens' grows by up to 3 each: 27 times the tolerance
    _against_oracle((q, k, v, decay, beta, state), norm_eps=None, tol=27 * 2e-5 * 128 ** 0.5)


# ---------------------------------------------------------------- together, as a model uses them

@pytest.mark.parametrize('dtype', TYPES)
def test_prompt_at_once_in_pieces_and_token_by_token(dtype):
    """A layer's convolution, rule and gated norm over a prompt in one call, in two, and its last tokens one by one, with
    paged.extend's tables: the same states and results but for rounding."""
    import torch
    from localai_amd import delta, layer, paged
    rng = np.random.default_rng(7)
    hk, hv, kd, vd, width = 2, 4, 64, 64, 4
    channels, lengths = 2 * hk * kd + hv * vd, [100, 0, 37]
    total = sum(lengths)
    x, z = (_random(rng, (total, n), dtype)[0] for n in (channels, hv * vd))
    w, norm_w = _t(rng.standard_normal((channels, width)) * 0.5), _t(rng.standard_normal(vd))
    decay, beta = _t(rng.standard_normal((total, hv))), _t(rng.standard_normal((total, hv)))
    a, dt = _t(-rng.uniform(0.1, 4, hv)), _t(rng.uniform(-4, 0, hv))
    first = np.concatenate([[0], np.cumsum(lengths)])

    def run(parts):
        states = delta.DeltaCache(2, hk, hv, kd, vd, rows=len(lengths), width=width)
        states.rule_state.normal_()       # what is there before a request starts does not matter
        states.conv_state.normal_()
        cache = paged.PagedKVCache(1, 1, 64, 32, 16, requests=len(lengths))
        out, done = torch.zeros((total, hv, vd), dtype=x.dtype, device='cuda'), np.zeros(len(lengths), int)
        for new in parts:
            step = cache.extend(_ints(new), sum(new) + 3)
            rows = np.concatenate([np.arange(first[b] + done[b], first[b] + done[b] + n) for b, n in enumerate(new)])
            pad = np.concatenate([rows, np.zeros(3, int)])       # three places of padding behind the tokens
            c = states.conv(1, x[pad], w, step)
            q, k, v = states.split(c)
            y = states.rule(1, q, k, v, decay[pad], beta[pad], step, a=a, dt_bias=dt, order='tiled')
            y = layer.rms_norm(y, norm_w, gate=z[pad].unflatten(-1, (hv, vd)))
            out[rows] = y[:len(rows)]
            done += new
            step.check()
        return out, states

    whole, states = run([lengths])
    for parts in ([[64, 0, 30], [36, 0, 7]], [[1, 0, 36], [98, 0, 0], [1, 0, 1]], [[95, 0, 33]] + [[1, 0, 0]] * 5 + [[0, 0, 1]] * 4):
        got, other = run(parts)
        torch.testing.assert_close(got.float(), whole.float(), rtol=8 * HALF[dtype] + 1e-4, atol=8 * HALF[dtype] + 1e-4)
        torch.testing.assert_close(other.rule_state[1, [0, 2]], states.rule_state[1, [0, 2]], rtol=1e-4,
                                   atol=1e-5 + 8 * HALF[dtype])
        torch.testing.assert_close(other.conv_state[1, [0, 2]], states.conv_state[1, [0, 2]], rtol=0, atol=0)
    # against the oracle, the first request
    xv, n = _np(x)[:100], 100
    c, _, _ = odelta.conv(np.zeros((width - 1, channels)), xv, _np(w))
    c = _np(torch.tensor(c).to(x.dtype))
    q, k, v = (c[:, i:j].reshape(n, -1, 64) for i, j in ((0, 128), (128, 256), (256, 512)))
    o, S = odelta.rule(np.zeros((hv, kd, vd)), q, k, v, _np(decay)[:n], _np(beta)[:n], _np(a), _np(dt), 'tiled')
    o, _ = odelta.rms_norm(_np(torch.tensor(o).to(x.dtype)), _np(norm_w), gate=_np(z)[:n].reshape(n, hv, vd))
    torch.testing.assert_close(whole[:n].double().cpu(), torch.tensor(o), rtol=8 * HALF[dtype] + 1e-4, atol=8 * HALF[dtype] + 1e-4)
    torch.testing.assert_close(states.rule_state[1, 0].double().cpu(), torch.tensor(S), rtol=1e-4, atol=1e-5 + 8 * HALF[dtype])


def _calls(rng, dtype='bfloat16', tokens=200, n=3):
    import torch
    heads = (2, 4, 128, 64)
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, tokens, heads, dtype, True)
    starts = _ints([0, 130, 133, tokens])
    state, _ = _random(rng, (n, 4, 128, 64), 'float32')
    x, _ = _random(rng, (tokens, 512), dtype)
    w, _ = _random(rng, (512, 4), 'float32')
    conv_state, _ = _random(rng, (n, 3, 512), 'float32')
    weight, _ = _random(rng, 64, 'float32')
    return dict(q=q, k=k, v=v, decay=decay, beta=beta, a=a, dt=dt, starts=starts, state=state, x=x, w=w,
                conv_state=conv_state, weight=weight, residual=_t(rng.standard_normal((tokens, 512))))


def _run_all(c, stream=None):
    from localai_amd import delta, layer
    conv = delta.conv(c['x'], c['w'], c['conv_state'], starts=c['starts'], stream=stream)
    y = delta.rule(c['q'], c['k'], c['v'], c['decay'], c['beta'], c['state'], starts=c['starts'], a=c['a'],
                   dt_bias=c['dt'], stream=stream)
    step = delta.rule(c['q'][:3], c['k'][:3], c['v'][:3], c['decay'][:3], c['beta'][:3], c['state'], stream=stream)
    z = layer.rms_norm(y, c['weight'], gate=y, stream=stream)
    n = layer.rms_norm(c['x'], c['w'].reshape(-1)[:512], residual=c['residual'], dtype='q8_0', stream=stream)
    return conv, y, step, z, n, c['state'], c['conv_state'], c['residual']


def test_captured_and_replayed():
    import torch
    rng = np.random.default_rng(8)
    c = _calls(rng)
    kept = [c[k].clone() for k in ('state', 'conv_state', 'residual')]

    def reset():
        for k, t in zip(('state', 'conv_state', 'residual'), kept):
            c[k].copy_(t)

    want = [t.clone() for t in _run_all(c)]
    again = [t.clone() for t in _run_all(c)]         # a second step on the states that the first left
    graphs, results = [], []
    for _ in range(2):
        reset()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(_run_all(c))
        graphs.append(g)
    for _ in range(3):
        reset()
        for i, wanted in ((0, want), (1, again)):
            graphs[i].replay()
            torch.cuda.synchronize()
            for t, expected in zip(results[i], wanted):
                assert torch.equal(t, expected)
        reset()
        for t, expected in zip(_run_all(c), want):
            assert torch.equal(t, expected)


def test_streams():
    """Two streams at once, each with its own inputs; results as on one."""
    import torch
    sets = [_calls(np.random.default_rng(s)) for s in (9, 10)]
    twins = [_calls(np.random.default_rng(s)) for s in (9, 10)]
    wants = [_run_all(c) for c in twins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    results = []
    for c, s in zip(sets, streams):
        results.append(_run_all(c, s))
    for s in streams:
        s.synchronize()
    for got, want in zip(results, wants):
        for t, expected in zip(got, want):
            assert torch.equal(t, expected)


@pytest.mark.parametrize('dtype', TYPES)
def test_rule_stays_in_its_workspace(dtype, monkeypatch):
    """Several windows; what lies behind the workspace stays as it was. (The sizes of a window's pieces differ by type.)"""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(11)
    heads, tokens = (8, 128, 128, 16), 1700
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, tokens, heads, dtype, True)
    state, _ = _random(rng, (2, heads[1], heads[2], heads[3]), 'float32')
    behind, made = 8 << 20, []

    def empty(stream, shape, kind):
        if kind is not torch.uint8:
            return torch.empty(shape, dtype=kind, device='cuda')
        made.append(torch.full((shape + behind,), 0xA5, dtype=torch.uint8, device='cuda'))
        return made[-1][:shape]

    monkeypatch.setattr(delta, '_empty', empty)
    first = state.clone()
    y = delta.rule(q, k, v, decay, beta, state, starts=_ints([0, 1600, tokens]), a=a, dt_bias=dt)
    assert len(made) == 1 and (made[0][-behind:] == 0xA5).all()
    # the last tokens again, from a call of their own: the first windows carried the state over
    z = delta.rule(*(t[1600:] for t in (q, k, v, decay, beta)), first[1:], starts=_ints([0, 100]), a=a, dt_bias=dt)
    torch.testing.assert_close(z.float(), y[1600:].float(), rtol=1e-4 + 2 * HALF[dtype], atol=1e-5)
    sizes = np.zeros((1600, heads[1]))
    _, want = odelta.rule(_np(first[0]), *(_np(t[:1600]) for t in (q, k, v, decay, beta)), _np(a), _np(dt), sizes=sizes)
    for h in range(heads[1]):
        # (a token's (2 sqrt(128) + 16) u, over the 1600 that may last)
        assert np.linalg.norm(_np(state[0, h]) - want[h]) <= 2.4e-6 * 40 * sizes[:, h].max()


def test_states_past_32_bits():
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(12)
    rows = 4300                                            # x 32 x 128 x 128 values of 4 bytes: 9 GB
    state = torch.empty((rows, 32, 128, 128), device='cuda')
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, 70, (16, 32, 128, 128), 'float32', True)
    small = torch.zeros((1, 32, 128, 128), device='cuda')
    for starts, n in ((_ints([0, 70]), 70), (None, 1)):
        state[rows - 1] = 0
        small.zero_()
        args = [t[:n] for t in (q, k, v, decay, beta)]
        y = delta.rule(*args, state, _ints([rows - 1]), starts, a=a, dt_bias=dt)
        z = delta.rule(*args, small, None, starts, a=a, dt_bias=dt)
        assert torch.equal(y, z) and torch.equal(state[rows - 1], small[0])


def test_starts_that_do_not_fit_are_cut():
    """Nothing outside the call's rows is read or written, whatever starts holds."""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(13)
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, 40, (1, 2, 64, 32), 'float32', True)
    state, sv = _random(rng, (3, 2, 64, 32), 'float32')
    out = torch.full((60, 2, 32), 7.0, device='cuda')
    delta.rule(q, k, v, decay, beta, state, None, _ints([-5, 20, 20, 1000]), a=a, dt_bias=dt, out=out[10:50])
    assert (out[:10] == 7).all() and (out[50:] == 7).all() and torch.isfinite(out).all()
    want, after = odelta.rule(sv[0], *(_np(t)[:20] for t in (q, k, v, decay, beta)), _np(a), _np(dt))
    np.testing.assert_allclose(_np(out)[10:30], want, atol=1e-4)
    np.testing.assert_array_equal(_np(state)[1], sv[1])
    x, _ = _random(rng, (40, 64), 'float32')
    w, _ = _random(rng, (64, 4), 'float32')
    cs, _ = _random(rng, (3, 3, 64), 'float32')
    out = torch.full((60, 64), 7.0, device='cuda')
    delta.conv(x, w, cs, None, _ints([-5, 20, 20, 1000]), out=out[10:50])
    assert (out[:10] == 7).all() and (out[50:] == 7).all()


def test_refusals_on_the_device():
    import torch
    from localai_amd import delta, layer
    from localai_amd._lib import HipError
    rng = np.random.default_rng(14)
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, 6, (1, 2, 64, 32), 'float32', True)
    state, _ = _random(rng, (6, 2, 64, 32), 'float32')
    call = lambda **c: delta.rule(**{**dict(q=q, k=k, v=v, decay=decay, beta=beta, state=state), **c})
    for change, error in [(dict(q=q.double()), TypeError), (dict(q=q.half()), TypeError), (dict(k=k[:5]), ValueError),
                          (dict(v=v[..., ::2]), ValueError), (dict(beta=beta[:, :1]), ValueError),
                          (dict(state=state.half()), TypeError), (dict(state=state[:, :, :, :16]), ValueError),
                          (dict(state=state[:2]), ValueError), (dict(a=a), ValueError), (dict(order='other'), ValueError),
                          (dict(norm_eps=-1.0), ValueError), (dict(scale=float('inf')), HipError),
                          (dict(slots=_ints([0] * 5)), ValueError), (dict(starts=_ints([0, 6]), lengths=_ints([1, 2])), ValueError),
                          (dict(starts=_ints(range(9))), ValueError), (dict(out=v[:, :, ::2]), ValueError),
                          (dict(slots=_ints([0] * 6).long()), TypeError), (dict(q=q[..., :63], k=k[..., :63]), (ValueError, HipError))]:
        with pytest.raises(error):
            call(**change)
    call()
    x, w = torch.ones(4, 64, device='cuda'), torch.ones(64, 4, device='cuda')
    cs = torch.zeros(4, 3, 64, device='cuda')
    for change, error in [(dict(x=x.double()), TypeError), (dict(x=x.t()), ValueError), (dict(weight=w[:, :3].contiguous()), ValueError),
                          (dict(state=cs[:, :2]), (TypeError, ValueError)), (dict(bias=w), ValueError),
                          (dict(out=x.half()), TypeError), (dict(weight=torch.ones(64, 9, device='cuda'),
                                                                 state=torch.ones(4, 8, 64, device='cuda')), HipError)]:
        with pytest.raises(error):
            delta.conv(**{**dict(x=x, weight=w, state=cs), **change})
    for change, error in [(dict(x=x.double()), TypeError), (dict(weight=w), ValueError), (dict(residual=x.half()), TypeError),
                          (dict(gate=x[:2]), ValueError), (dict(dtype=torch.int8), TypeError), (dict(dtype='q4_0'), TypeError),
                          (dict(x=x[:, :40], weight=w.reshape(-1)[:40], dtype='q8_0'), ValueError),
                          (dict(x=x.reshape(2, 2, 4, 16)), ValueError), (dict(out=x.half()), TypeError)]:
        with pytest.raises(error):
            layer.rms_norm(**{**dict(x=x, weight=w.reshape(-1)[:64]), **change})


# ---------------------------------------------------------------- steps of many requests, with starts

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [25, 64, 65, 200])
def test_rule_one_token_each_with_starts(n, dtype):
    """A decoding step as paged.extend's tables have it, some requests without a token."""
    counts = [1] * n
    counts[3], counts[n - 2] = 0, 0
    _check_rule((2, 4, 128, 32), counts, dtype, True, 'grouped')


@pytest.mark.parametrize('dtype', TYPES)
def test_rule_many_requests_with_prompts_among_them(dtype):
    """Pieces numbered by rows alone: prompts of every length beside single tokens, at the ends of 64 requests too."""
    rng = np.random.default_rng(5)
    counts = [1] * 260
    for b in (0, 63, 64, 65, 127, 128, 200, 259):
        counts[b] = int(rng.choice([24, 25, 26, 49, 50, 63, 64, 65, 100, 129, 200]))
    counts[30:50] = [0] * 20
    _check_rule((1, 4, 64, 64), counts, dtype, True, 'grouped')
    _check_rule((1, 4, 64, 64), [25] * 70, dtype, True, 'grouped')
    _check_rule((1, 4, 64, 64), [64] * 3 + [24] * 100 + [65, 64, 25, 128], dtype, True, 'tiled')


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('counts', [[1] * 60 + [30] * 20 + [100] * 10 + [400] + [1] * 9, [90] * 28 + [400, 1], [2500] + [1] * 40],
                         ids=['by rows', 'by rows and requests', 'one long'])
def test_rule_more_requests_than_a_window_has_pieces(counts, dtype):
    """Windows of 20 pieces and more (128 heads); requests that begin, go on and end in any of them."""
    _check_rule((8, 128, 128, 16), counts, dtype, True, 'grouped')


def test_captured_step_takes_any_lengths():
    """One graph of 100 requests and 256 tokens, replayed with other tables: single tokens, a prompt among them, all prompts."""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(15)
    n, tokens = 100, 256
    q, k, v, decay, beta, a, dt = _rule_inputs(rng, tokens, (2, 4, 128, 64), 'bfloat16', True)
    first, _ = _random(rng, (n, 4, 128, 64), 'float32')
    starts, lengths, state = _ints([0] * (n + 1)), _ints([500] * n), first.clone()
    out = torch.zeros((tokens, 4, 64), dtype=v.dtype, device='cuda')
    run = lambda: delta.rule(q, k, v, decay, beta, state, None, starts, lengths, a, dt, out=out)
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for counts in ([1] * n, [1] * 50 + [157] + [1] * 49, [25] * 10 + [0] * 89 + [6], [0] * 99 + [256], [24, 0] * 10 + [0] * 80, [1] * n):
        starts.copy_(_ints(np.concatenate([[0], np.cumsum(counts)])))
        results = []
        for call in (g.replay, run):
            state.copy_(first)
            out.fill_(7)
            call()
            torch.cuda.synchronize()
            results.append((out.clone(), state.clone()))
        for got, expected in zip(*results):
            assert torch.equal(got, expected)
        assert (results[0][0][sum(counts):] == 7).all() and torch.isfinite(results[0][0]).all()
        at = 0
        for b, c in enumerate(counts):
            if c > 1:
                rows = slice(at, at + c)
                alone = first[b:b + 1].clone()
                y = delta.rule(q[rows], k[rows], v[rows], decay[rows], beta[rows], alone, starts=_ints([0, c]), a=a, dt_bias=dt)
                torch.testing.assert_close(results[0][0][rows].float(), y.float(), rtol=4 * HALF['bfloat16'], atol=1e-4)
                torch.testing.assert_close(results[0][1][b:b + 1], alone, rtol=1e-4, atol=1e-4)
            at += c
