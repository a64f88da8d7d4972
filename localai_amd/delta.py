"""The linear-attention layers of a hybrid model (Qwen3.5's gated delta net) for
several requests in one step, on the GPU.

    DeltaCache   the states of every layer, a row per request
    conv         the short causal convolution ahead of q, k and v
    rule         the gated delta rule: one token per request, or prompts and
                 pieces of prompts

A step of a server, beside paged.PagedKVCache for the full-attention layers:

    step = cache.extend(new, tokens)
    for each linear-attention layer:
        x = states.conv(layer, x, weight, step)
        q, k, v = views of x
        y = states.rule(layer, q, k, v, decay, beta, step, a=a, dt_bias=dt_bias)
        y = layer.rms_norm(y, weight, gate=z)

The reference serves one token of one request (engine/qwen35.py:224-252,
engine/numba_kernels.py:11-45); attention.delta_net_step is that form, in its
order of operations. Arguments are device tensors, the work runs in the HIP
library, and nothing is read back by the host. Every call may be captured in a
graph; workspaces come from PyTorch's allocator call by call, so graphs and
streams share none. A call with `stream` runs there, allocates there, and holds
the memory of its arguments until that stream has passed it; the streams' own
order is the caller's.
"""
from __future__ import annotations

import functools
import struct

from . import _lib, device
from .paged import _device_tensor, _empty, _hold, _ptr, _r, _refuse, _stream

_REQUESTS = struct.Struct('=QqQQQq')      # localai_delta_requests
_STRIDES = struct.Struct('=10q')


class _Calls:
    """The library's entry points and types, looked up once."""

    def __init__(self):
        t = device.torch()
        lib = _lib.load()
        self.types = {t.float32: 0, t.float16: 1, t.bfloat16: 30}     # of activations -> GGML numbers
        self.conv, self.rule = lib.localai_hip_delta_conv, lib.localai_hip_delta_rule
        self.workspace = functools.lru_cache(4096)(lib.localai_hip_delta_rule_workspace_size)


_calls = None


def _c():
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


def _rows(t, name, dtype, shape):
    """(address, token stride, head stride) of t [tokens, heads, dim]."""
    r = _r()
    if not (isinstance(t, r.Tensor) and t.dtype is dtype and t.get_device() == r.index and t.shape == shape):
        _refuse(t, name, dtype, shape)
    ts, hs, step = t.stride()
    if step != 1 and shape[2] > 1:
        raise ValueError(f'{name} must have adjacent head values')
    # (the stride of a dimension of one says nothing)
    return t.data_ptr(), ts if shape[0] > 1 else 0, hs if shape[1] > 1 else 0


def _gate_rows(t, name, tokens, heads):
    """(address, token stride) of t [tokens, heads] fp32."""
    r = _r()
    if not (isinstance(t, r.Tensor) and t.dtype is r.f32 and t.get_device() == r.index and t.shape == (tokens, heads)):
        _refuse(t, name, r.f32, (tokens, heads))
    ts, step = t.stride()
    if step != 1 and heads > 1:
        raise ValueError(f'{name} must have adjacent heads')
    return t.data_ptr(), ts if tokens > 1 else 0


def _activations(t, name, dims):
    """GGML number of the type of t, a device tensor of this many dimensions."""
    _device_tensor(t, name)
    kind = _c().types.get(t.dtype)
    if kind is None:
        raise TypeError(f'{name} must be float32, float16 or bfloat16')
    if t.dim() != dims:
        raise ValueError(f'{name} must have {dims} dimensions')
    return kind


def _requests(tokens, state, slots, starts, lengths):
    """localai_delta_requests of a state pool and a step's int32 tensors."""
    i32 = _r().i32
    n = tokens
    for t, extra in ((slots, 0), (lengths, 0), (starts, 1)):
        if t is not None:
            _device_tensor(t, 'starts' if extra else 'slots and lengths')
            n = t.numel() - extra
            break
    if starts is None and n != tokens:
        raise ValueError('without starts there is one token per request')
    if slots is None and n > state.shape[0]:
        raise ValueError('more requests than rows of the state')
    return _REQUESTS.pack(state.data_ptr(), state.shape[0], _ptr(slots, 'slots', i32, (n,)) if slots is not None else 0,
                          _ptr(starts, 'starts', i32, (n + 1,)) if starts is not None else 0,
                          _ptr(lengths, 'lengths', i32, (n,)) if lengths is not None else 0, n), n


def conv(x, weight, state, slots=None, starts=None, lengths=None, bias=None, silu=True, out=None, stream=None):
    """The causal convolution of each request's new rows (localai_hip_delta_conv).

    x [tokens, channels]: fp32, f16 or bf16, any row stride; weight [channels,
    width] and bias [channels] fp32, the last tap on the row itself; state [rows,
    width - 1, channels] fp32, updated in place; slots [requests]: the requests'
    rows of it (None: row b), one outside it marking an empty place; starts
    [requests + 1] (None: one token per request) and lengths [requests] (None: no
    request is new) as paged.extend() leaves them: a request whose tokens are all
    new starts from zeros. silu: y / (1 + exp(-y)) of each sum. Returns
    [tokens, channels] of x's type, in `out` if given (memory of its own); rows
    behind starts[-1] and of empty places are left as they were, in a new
    result whatever its memory held."""
    kind = _activations(x, 'x', 2)
    r = _r()
    f32 = r.f32
    tokens, channels = x.shape
    if x.get_device() != r.index:
        _refuse(x, 'x', x.dtype, None)
    if x.stride(1) != 1 and channels > 1:
        raise ValueError('x must have adjacent channels')
    _device_tensor(weight, 'weight')
    if weight.dim() != 2:
        raise ValueError('weight must be [channels, width]')
    width = weight.shape[1]
    wp = _ptr(weight, 'weight', f32, (channels, width))
    bp = _ptr(bias, 'bias', f32, (channels,)) if bias is not None else None
    _device_tensor(state, 'state')
    if state.dim() != 3:
        raise ValueError('state must be [rows, width - 1, channels]')
    _ptr(state, 'state', f32, (state.shape[0], width - 1, channels))
    requests, _ = _requests(tokens, state, slots, starts, lengths)
    if out is None:
        out = _empty(stream, (tokens, channels), x.dtype)
    elif not (isinstance(out, r.Tensor) and out.dtype is x.dtype and out.get_device() == r.index
              and out.shape == x.shape):
        _refuse(out, 'out', x.dtype, x.shape)
    elif out.stride(1) != 1 and channels > 1:
        raise ValueError('out must have adjacent channels')
    status = _c().conv(x.data_ptr(), kind, tokens, channels, x.stride(0), wp, bp, width, bool(silu), requests,
                       out.data_ptr(), out.stride(0), _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, x, weight, bias, state, slots, starts, lengths, out)
    return out


def rule(q, k, v, decay, beta, state, slots=None, starts=None, lengths=None, a=None, dt_bias=None, order='grouped',
         norm_eps=1e-6, scale=None, out=None, stream=None):
    """The gated delta rule over each request's new tokens (localai_hip_delta_rule).

    q, k [tokens, key heads, key dim], v [tokens, value heads, value dim]: fp32,
    f16 or bf16, token and head strides multiples of 4 values (views of the
    convolution's result); decay, beta [tokens, value heads] fp32: the state's
    logarithmic decay and the step's size, or with a, dt_bias [value heads] their
    projections: a softplus(decay + dt_bias) and sigmoid(beta). state [rows, value
    heads, key dim, value dim] fp32, updated in place; slots, starts, lengths:
    as in conv(). order: value head h reads key head h // (value heads / key
    heads) ('grouped') or h % key heads ('tiled', as GGUF files have them).
    norm_eps: q and k go through x / sqrt(|x|^2 + norm_eps), None: as they are;
    scale: q's factor, 1 / sqrt(key dim) by default. Returns [tokens, value heads,
    value dim] of q's type, in `out` if given (memory of its own); rows behind
    starts[-1] and of empty places are left as they were."""
    kind = _activations(q, 'q', 3)
    _device_tensor(v, 'v')
    _device_tensor(state, 'state')
    r, c = _r(), _c()
    f32, dtype = r.f32, q.dtype
    if order not in ('grouped', 'tiled'):
        raise ValueError("order must be 'grouped' or 'tiled'")
    if v.dim() != 3:
        raise ValueError('v must be [tokens, value heads, value dim]')
    tokens, hk, kd = q.shape
    hv, vd = v.shape[1:]
    qp, *qs = _rows(q, 'q', dtype, (tokens, hk, kd))
    kp, *ks = _rows(k, 'k', dtype, (tokens, hk, kd))
    vp, *vs = _rows(v, 'v', dtype, (tokens, hv, vd))
    dp, ds = _gate_rows(decay, 'decay', tokens, hv)
    bp, bs = _gate_rows(beta, 'beta', tokens, hv)
    if (a is None) != (dt_bias is None):
        raise ValueError('a and dt_bias go together')
    ap, tp = (_ptr(a, 'a', f32, (hv,)), _ptr(dt_bias, 'dt_bias', f32, (hv,))) if a is not None else (None, None)
    if state.dim() != 4:
        raise ValueError('state must be [rows, value heads, key dim, value dim]')
    _ptr(state, 'state', f32, (state.shape[0], hv, kd, vd))
    requests, n = _requests(tokens, state, slots, starts, lengths)
    if norm_eps is not None and not norm_eps >= 0:
        raise ValueError('norm_eps must not be negative')
    need = c.workspace(tokens, n, starts is not None, hk, hv, kd, vd)
    ws = _empty(stream, need, r.u8) if need > 0 else None
    if out is None:
        out = _empty(stream, (tokens, hv, vd), dtype)
        op, os = out.data_ptr(), (hv * vd, vd)
    else:
        op, *os = _rows(out, 'out', dtype, (tokens, hv, vd))
    status = c.rule(qp, kp, vp, kind, _STRIDES.pack(*qs, *ks, *vs, *os, ds, bs), tokens, hk, hv, kd, vd, dp, bp, ap, tp,
                    order == 'tiled', -1.0 if norm_eps is None else norm_eps, kd ** -0.5 if scale is None else scale,
                    requests, op, ws.data_ptr() if need > 0 else None, need if need > 0 else 0, _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, q, k, v, decay, beta, state, slots, starts, lengths, a, dt_bias, out)
    return out


class DeltaCache:
    """The linear-attention layers' states (zero-filled): conv [n_layers, rows,
    width - 1, channels] and rule [n_layers, rows, value heads, key dim, value
    dim], fp32, row b a request's; channels: 2 key heads key dim + value heads
    value dim. A request's tokens cannot be taken back: to go on from an earlier
    place, keep a copy of its row."""

    def __init__(self, n_layers, key_heads, value_heads, key_dim, value_dim, rows=1, width=4):
        torch = device.torch()
        dev = device.device()
        self.key_heads, self.value_heads = int(key_heads), int(value_heads)
        self.key_dim, self.value_dim = int(key_dim), int(value_dim)
        channels = 2 * self.key_heads * self.key_dim + self.value_heads * self.value_dim
        self.conv_state = torch.zeros((n_layers, rows, width - 1, channels), dtype=torch.float32, device=dev)
        self.rule_state = torch.zeros((n_layers, rows, self.value_heads, self.key_dim, self.value_dim),
                                      dtype=torch.float32, device=dev)

    def reset(self):
        """Every request starts from zeros."""
        self.conv_state.zero_()
        self.rule_state.zero_()

    def conv(self, layer, x, weight, step, slots=None, bias=None, silu=True, out=None, stream=None):
        """conv() of one layer for the new tokens of a paged.Step."""
        return conv(x, weight, self.conv_state[layer], slots, step.starts, step.lengths, bias, silu, out, stream)

    def split(self, x):
        """Views q, k, v of a convolution's result [tokens, channels]."""
        n = self.key_heads * self.key_dim
        q, k, v = x.split([n, n, x.shape[1] - 2 * n], dim=1)
        return (q.unflatten(-1, (self.key_heads, self.key_dim)), k.unflatten(-1, (self.key_heads, self.key_dim)),
                v.unflatten(-1, (self.value_heads, self.value_dim)))

    def rule(self, layer, q, k, v, decay, beta, step, slots=None, a=None, dt_bias=None, order='grouped', norm_eps=1e-6,
             scale=None, out=None, stream=None):
        """rule() of one layer for the new tokens of a paged.Step."""
        return rule(q, k, v, decay, beta, self.rule_state[layer], slots, step.starts, step.lengths, a, dt_bias, order,
                    norm_eps, scale, out, stream)
