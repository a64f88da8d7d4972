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
