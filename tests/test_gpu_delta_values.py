"""The linear-attention layers' operators on the GPU where values are far from a unit normal's, and at sizes of their own
forms; u = 2^-24, a result of 16 bits adds half a step of its type (oracle/delta.py, tests/test_gpu_delta.py).

y / (1 + exp(-y)): 6 u of the result. exp(-y) past 2^126 or so (y below -126 ln 2 = -87.3) may give 0, as it does where
exp(-y) leaves fp32 (below -88.7): less than 87.4 / 2^126 < 2^-119 is lost."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ['float32', 'float16', 'bfloat16']
HALF = {'float32': U, 'float16': 2.0 ** -11, 'bfloat16': 2.0 ** -8}
FLOOR = {'float32': 2.0 ** -119, 'float16': 2.0 ** -25, 'bfloat16': 2.0 ** -119}     # what may be lost of small results


def _np(t):
    return t.detach().double().cpu().numpy()


def _ints(x):
    import torch
    return torch.tensor(np.asarray(x, dtype=np.int32), device='cuda')


def _silu_values(dtype):
    """Every value of a 16-bit type; of fp32 all regions, densely where exp(-y) leaves its range; infinities and a NaN."""
    import torch
    if dtype != 'float32':
        bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
        y = bits.view(getattr(torch, dtype))
        y = torch.cat([y[torch.isfinite(y)], torch.tensor([np.inf, -np.inf, np.nan], dtype=y.dtype)])
    else:
        y = torch.cat([torch.linspace(-120, 120, 100001), torch.linspace(-100, -85, 300001), torch.linspace(-2, 2, 10001),
                       torch.logspace(-30, 38, 2001), -torch.logspace(-30, 38, 2001),
                       torch.tensor([0.0, -0.0, 3.4e38, -3.4e38, np.inf, -np.inf, np.nan])])
    return torch.cat([y, torch.zeros(-len(y) % 1024, dtype=y.dtype)]).cuda()


def _silu(y):
    with np.errstate(over='ignore', invalid='ignore'):
        return y / (1 + np.exp(-y))


def _check_silu(got, y, want, dtype, u):
    finite = np.isfinite(y)
    assert np.isfinite(got[finite]).all()
    off = np.abs(got[finite] - want[finite])
    assert (off <= (u * U + HALF[dtype]) * np.abs(want[finite]) + FLOOR[dtype]).all()
    np.testing.assert_array_equal(got[~finite], want[~finite])     # inf of inf, NaN of -inf and NaN


@pytest.mark.parametrize('dtype', TYPES)
def test_conv_of_every_value(dtype):
    """A convolution that passes its rows on: silu of them, whatever they are."""
    import torch
    from localai_amd import delta
    y = _silu_values(dtype).reshape(1024, -1)
    channels = y.shape[1]
    w = torch.zeros(channels, 4, device='cuda')
    w[:, 3] = 1
    got = delta.conv(y, w, torch.zeros(1024, 3, channels, device='cuda'))     # a row each: none meets another
    yv = _np(y)
    _check_silu(_np(got), yv, _silu(yv), dtype, 6)
    rows = torch.where(torch.isfinite(y), y, 0)     # one request's (0 times infinity would be NaN)
    got = delta.conv(rows, w, torch.zeros(1, 3, channels, device='cuda'), starts=_ints([0, 1024]))
    yv = _np(rows)
    _check_silu(_np(got), yv, _silu(yv), dtype, 6)


@pytest.mark.parametrize('dtype', TYPES)
def test_norm_with_gates_of_every_value(dtype):
    """Rows of ones, whose norm is 1 / sqrt(1 + eps); the gate's factor beside 6 u of a norm of 64 ones."""
    import torch
    from localai_amd import dequant, layer
    z = _silu_values(dtype).reshape(-1, 64)
    x, w = torch.ones_like(z), torch.ones(64, device='cuda')
    zv, one = _np(z), 1 / np.sqrt(1 + 1e-6)
    want = _silu(zv) * one
    _check_silu(_np(layer.rms_norm(x, w, gate=z)), zv, want, dtype, 14)
    if dtype != 'float32':
        _check_silu(_np(layer.rms_norm(x, w, gate=z, dtype=torch.float32)), zv, want, 'float32', 14)
    # in blocks: as far as their scales are finite
    z = torch.where(z.abs() <= 1e4, z, 0)
    got = _np(dequant.dequantize_device(layer.rms_norm(x, w, gate=z, dtype='q8_0'), 8, z.shape))
    want = _silu(_np(z)) * one
    top = np.repeat(np.abs(want).reshape(-1, 32).max(-1), 32).reshape(want.shape)
    # half a step of the scale, its own rounding to f16 (normal, or by 2^-25) at 127 steps of it
    assert (np.abs(got - want) <= top / 127 * (0.5 + 127 * 2.0 ** -11) * (1 + 2.0 ** -9) + 128 * 2.0 ** -25 + 14 * U * top).all()


# ---------------------------------------------------------------- values of mixed sizes in the rule

def _columns(state, q, k, v, g, b, scale):
    """One head in 64 bits, token after token: results [tokens, value dim], the state after, and how far fp32 may be off
    in each, column by column.

    A column of the state is a recurrence of its own: s <- e^g s; d = b (v - k^ . s); s <- s + k^ d. With |k^| = 1 and
    0 <= b <= 1 its step is e^g times a contraction, so what a token rounds is not enlarged behind it: with s_t the larger of
    the column's norms after the decay and after the update, r_t = (2 sqrt(key dim) + 16) u s_t is rounded (three
    roundings a value, two sums of key dim products), E_t^2 = (e^g E)^2 + r_t^2, and E_t + r_t, times q^'s scale, bounds the
    result. Operands of 22 bits (4 u each) are fewer roundings than these."""
    S, E, c = state.copy(), np.zeros(v.shape[1]), (2 * k.shape[1] ** 0.5 + 16) * U
    out, off = np.zeros(v.shape), np.zeros(v.shape)
    for t in range(len(v)):
        S *= np.exp(g[t])
        size = np.linalg.norm(S, axis=0)
        S += np.outer(k[t], b[t] * (v[t] - k[t] @ S))
        r = c * np.maximum(size, np.linalg.norm(S, axis=0))
        E = np.hypot(np.exp(g[t]) * E, r)
        out[t], off[t] = scale * (q[t] @ S), scale * (E + r)
    return out, S, off, E


def _mixed(case, rng, q, k, v, g, b, state, big):
    """Puts values `big` times the others into one or more columns of v [tokens, heads, value dim] or of the state."""
    if case == 'one':              # behind and ahead of tokens of 1
        v[40, 0, 5], v[100, -1, 7] = big, -big
    elif case == 'rows':           # whole tokens
        v[[20, 75]] *= big
    elif case == 'forgotten':      # large, then everything forgotten within the same 64
        v[10] *= big
        g[15] = -200
        v[80, -1, 3] = big
        g[81] = -np.inf
    elif case == 'faint':          # large v that a small beta takes down to the others' size
        v[[3, 70]] *= big
        b[[3, 70]] = 1 / big
    elif case == 'state':          # a state that is forgotten in time
        state *= big
        g[5] = -np.log(big) - 3
    elif case == 'zeros':          # ahead of the first value, and between
        v[:30], v[50:60] = 0, 0
        state[:] = 0
        v[33] *= big
    else:                          # of every size, column by column
        v *= big ** rng.uniform(-0.5, 0.5, v.shape)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('big', [1e4, 1e6, 1e8, 1e10, 1e12])
@pytest.mark.parametrize('case', ['one', 'rows', 'forgotten', 'faint', 'state', 'zeros', 'any'])
@pytest.mark.parametrize('heads', [(2, 4, 128, 32), (1, 2, 64, 16), (1, 1, 256, 48)], ids=str)
def test_rule_mixed_sizes_in_64_tokens(heads, case, big, dtype):
    """A value beside one that is far larger, in the same column and the same 64 tokens, keeps its bits."""
    import torch
    from localai_amd import delta
    if dtype == 'float16':
        big = min(big, 1e4)       # (f16 holds none larger beside 1)
    rng = np.random.default_rng(sum(heads) + len(case))
    hk, hv, kd, vd = heads
    n = 150
    q, k, v = (rng.standard_normal((n, h, d)) for h, d in ((hk, kd), (hk, kd), (hv, vd)))
    g, b, state = -rng.exponential(0.05, (n, hv)), rng.random((n, hv)), rng.standard_normal((hv, kd, vd)) * 0.1
    with np.errstate(divide='ignore'):
        _mixed(case, rng, q, k, v, g, b, state, big)
    q, k, v = (torch.tensor(x, dtype=torch.float32).to(getattr(torch, dtype)).cuda() for x in (q, k, v))
    assert torch.isfinite(v).all()
    g, b, state = (torch.tensor(x, dtype=torch.float32, device='cuda') for x in (g, b, state[None]))
    qv, kv, vv, gv, bv, sv = (_np(x) for x in (q, k, v, g, b, state[0]))
    got = _np(delta.rule(q, k, v, g, b, state, starts=_ints([0, n])))
    qv, kv = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (qv, kv))
    for h in range(hv):
        key = h // (hv // hk)
        want, after, off, off_state = _columns(sv[h], qv[:, key], kv[:, key], vv[:, h], gv[:, h], bv[:, h], kd ** -0.5)
        assert (np.abs(got[:, h] - want) <= off + (HALF[dtype] * np.abs(want) if dtype != 'float32' else 0) + 2.0 ** -25 * (dtype == 'float16')).all(), ('out', h)
        assert (np.linalg.norm(_np(state[0, h]) - after, axis=0) <= off_state).all(), ('state', h)


# ---------------------------------------------------------------- long pieces of the convolution

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [2, 4, 8])
@pytest.mark.parametrize('channels', [1 << 20, (1 << 20) - 3])
@pytest.mark.parametrize('counts', [[13, 0, 17], [0, 3, 16, 1, 7, 2], [31, 0, 33, 1], [2, 64, 32, 5]], ids=str)
def test_conv_of_many_values(counts, channels, width, dtype):
    """Pieces of 16 rows (past 2^24 values) and of 32 (past 2^25), with requests on both sides of their ends. (width + 1) u of
    the terms' sizes, passed on by silu with a slope below 1.1, and 6 u of the result."""
    import torch
    from localai_amd import delta
    gen = torch.Generator('cuda').manual_seed(sum(counts) + width)
    normal = lambda *shape: torch.randn(shape, generator=gen, device='cuda')
    n, starts = len(counts), np.concatenate([[0], np.cumsum(counts)])
    x, w, state = normal(sum(counts) + 2, channels).to(getattr(torch, dtype)), normal(channels, width), normal(n + 1, width - 1, channels)
    assert (len(x) * channels > 1 << 25) == (counts[0] not in (0, 13)) and len(x) * channels > 1 << 24
    before, out, slots = state.clone(), torch.full_like(x, 7.0), [(b + 1) % (n + 1) for b in range(n)]
    lengths = [c + b % 2 for b, c in enumerate(counts)]      # every other request starts from zeros
    delta.conv(x, w, state, _ints(slots), _ints(starts), _ints(lengths), out=out)
    assert (out[sum(counts):] == 7).all()
    busy = {s for s, c in zip(slots, counts) if c}
    for s in set(range(n + 1)) - busy:
        assert torch.equal(state[s], before[s])
    for b, c in enumerate(counts):
        if not c:
            continue
        old = before[slots[b]].double() * (b % 2)
        line = torch.cat([old, x[starts[b]:starts[b + 1]].double()])
        want, size = torch.zeros(2, c, channels, dtype=torch.float64, device='cuda')
        for j in range(width):
            term = line[j:j + c] * w[:, j].double()
            want += term
            size += term.abs()
        want = want / (1 + torch.exp(-want))
        off = (out[starts[b]:starts[b + 1]].double() - want).abs()
        assert (off <= 1.1 * (width + 1) * U * size + (6 * U + HALF[dtype]) * want.abs() + FLOOR[dtype]).all(), b
        assert torch.equal(state[slots[b]].double(), line[c:]), b


# ---------------------------------------------------------------- long rows of the norm

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ['equal', 'random', 'first'])
@pytest.mark.parametrize('dim', [4095, 4096, 32768, 100001, (1 << 20) - 1, 1 << 20])
def test_norm_of_long_rows(dim, kind, dtype):
    """Rows whose squares' roundings all go one way, or are lost behind a large one. A lane's squares (u each) are summed
    in runs of at most 16 and 8 of those (23 u), or in 64 bits; lanes and waves in a tree (10 u): half of 34 u reaches the
    root, root and products are 4 u; in all below 24 u of the result."""
    import torch
    from localai_amd import layer
    gen = torch.Generator('cuda').manual_seed(dim)
    for value in ([1.1, 0.77, 3.3e-5] if kind == 'equal' else [1.0]):
        x = torch.full((3, dim), value, device='cuda')
        if kind != 'equal':
            x = torch.randn((3, dim), generator=gen, device='cuda')
        if kind == 'first':
            x[:, :16] *= 1e4
        x = x.to(getattr(torch, dtype))
        w = torch.rand(dim, generator=gen, device='cuda') + 0.5
        h = x.double()
        want = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-10) * w.double()
        got = layer.rms_norm(x, w, eps=1e-10, dtype=torch.float32)
        off = ((got.double() - want).abs() / want.abs().clamp(min=2.0 ** -100)).max().item()
        assert off <= 24 * U, (value, off / U)
        residual = torch.zeros(3, dim, device='cuda')
        got = layer.rms_norm(x, w, eps=1e-10, residual=residual, dtype=torch.float32)     # (four values a lane)
        off = ((got.double() - want).abs() / want.abs().clamp(min=2.0 ** -100)).max().item()
        assert off <= 24 * U, ('residual', value, off / U)


def test_norm_rounds_its_inverse_root_once():
    """Values of 2^-70, whose squares are nothing beside eps: the result is the inverse root of eps, 2^-70 of it. One rounding,
    and 2^-6 of one for what is left of the approximation; past fp32's middle range, 1e-37 and 1e37, a quotient's too where it is
    computed so and, as their square 2^-140 is 2^-17 of 1e-37, half of the sum's: 2.5 u; 2^-70 / sqrt(1e37) = 2.7e-40 is subnormal, rounded to
    steps of 2^-149: half of one, 2^70 times, besides."""
    import torch
    from localai_amd import layer
    rng = np.random.default_rng(0)
    x, w = torch.full((1, 64), 2.0 ** -70, device='cuda'), torch.ones(64, device='cuda')
    eps = np.concatenate([np.float32(10.0) ** rng.uniform(-30, 30, 300).astype(np.float32), np.float32([1, 2, 3, 0.25, 1e-37, 1e37])])
    got = torch.stack([layer.rms_norm(x, w, eps=float(e))[0, 0] for e in eps])
    want = 1 / np.sqrt(eps.astype(np.float64) + 2.0 ** -140)
    off = np.where((eps >= 1e-30) & (eps <= 1e30), 1 + 2.0 ** -6, 2.5) * U * want + 2.0 ** (70 - 150) * (want < 2.0 ** (70 - 126))
    assert (np.abs(_np(got) * 2.0 ** 70 - want) <= off).all()
    x[:] = 0
    for e in (0.0, 1e-45, 3e38):
        y = _np(layer.rms_norm(x, w, eps=e))
        assert np.isnan(y).all() if e == 0 else not y.any()      # 0 / 0
    x[:] = 1
    np.testing.assert_allclose(_np(layer.rms_norm(x, w, eps=3e38)), 1 / np.sqrt(3e38), rtol=3 * U)
    assert not _np(layer.rms_norm(x * 1e30, w)).any()             # squares past fp32: 1 / inf


@pytest.mark.parametrize('dtype', ['float32', 'bfloat16'])
@pytest.mark.parametrize('q_size,k_size,v_size', [(3e13, 3e13, 1e28), (1e14, 3e15, 1), (3e15, 1e14, 1), (1e17, 1e17, 1e29),
                                                  (1, 1, 3e31), (1, 1, 1e34), (1e-12, 1e14, 1e-30)])
@pytest.mark.parametrize('n', [150, 7])     # in pieces, token by token
def test_rule_on_both_sides_of_its_largest_values(n, q_size, k_size, v_size, dtype):
    """Lengths of q and k around 1e15, v around 1e30; the rule is the same but for v's factor."""
    import torch
    from localai_amd import delta
    rng = np.random.default_rng(1)
    q, k, v = (torch.tensor(rng.standard_normal((n, h, d)) * s, dtype=torch.float32).to(getattr(torch, dtype)).cuda()
               for h, d, s in ((1, 128, q_size), (1, 128, k_size), (2, 32, v_size)))
    g, b = (torch.tensor(x, dtype=torch.float32, device='cuda') for x in (-rng.exponential(0.05, (n, 2)), rng.random((n, 2))))
    state = torch.tensor(rng.standard_normal((1, 2, 128, 32)) * 0.1 * v_size, dtype=torch.float32, device='cuda')
    qv, kv, vv, gv, bv, sv = (_np(x) for x in (q, k, v, g, b, state[0]))
    got = _np(delta.rule(q, k, v, g, b, state, starts=_ints([0, n]), norm_eps=0))
    qv, kv = (x / np.sqrt((x * x).sum(-1, keepdims=True)) for x in (qv, kv))
    for h in range(2):
        want, after, off, off_state = _columns(sv[h], qv[:, 0], kv[:, 0], vv[:, h], gv[:, h], bv[:, h], 128 ** -0.5)
        assert (np.abs(got[:, h] - want) <= off + (HALF[dtype] * np.abs(want) if dtype != 'float32' else 0)).all()
        assert (np.linalg.norm(_np(state[0, h]) - after, axis=0) <= off_state).all()
