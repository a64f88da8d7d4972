"""The matvec chain of one decode layer (localai_hip_layer_chain), and the norm
between layers for several rows.

DecodeLayerChain holds the seven weight handles of the chain -- attn_output,
ffn_gate, ffn_up, ffn_down of layer L and attn_q, attn_k, attn_v of layer
L+1 -- and the two norm weights, and runs, from the attention output of layer
L, the part of the reference's decode step up to the attention inputs of
layer L+1 (engine/model.py:229-233, then :181-185 and :203-210):

    x1 = pre + W_o att;  u = norm(x1) * w_ffn;  act = silu(W_gate u) * (W_up u)
    x_out = x1 + W_down act;  v' = norm(x_out) * w_attn
    q, k, v = W_q v', W_k v', W_v v'   (+ adjacent-pair RoPE of q and k)

All of it stays on the device; nothing here computes on the host. By default
the chain runs as four launches with the glue fused into the matvec kernels;
set_mode(one_launch=True) selects the single launch with device-side waits
between its stages.

rms_norm is the norm of many tokens at once (localai_hip_rms_norm): with the
residual's addition, with a gate, to any activation type or to Q8_0 blocks.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from . import _lib, device
from .paged import _device_tensor, _empty, _hold, _ptr, _r, _refuse, _stream

ORDER = ('attn_output', 'ffn_gate', 'ffn_up', 'ffn_down', 'attn_q', 'attn_k', 'attn_v')


def set_mode(one_launch):
    """Process-wide: how every DecodeLayerChain runs (False: four launches)."""
    _lib.check(_lib.load().localai_hip_layer_chain_mode(1 if one_launch else 0))


class DecodeLayerChain:
    def __init__(self, mats, w_ffn, w_attn, eps, head_dim=None):
        """mats: name -> device.QMat for the names in ORDER (Q4_K / Q6_K);
        w_ffn: ffn_norm of layer L, w_attn: attn_norm of layer L+1 ([dim] each)."""
        t = device.torch()
        self.mats = [mats[n] for n in ORDER]
        self.dim, self.ffn = self.mats[0].rows, self.mats[1].rows
        self.eps = float(eps)
        self.head_dim = int(head_dim) if head_dim else 0
        dev = device.device()
        self.w_ffn = device.to_device_f32(np.asarray(w_ffn, np.float32).reshape(-1))
        self.w_attn = device.to_device_f32(np.asarray(w_attn, np.float32).reshape(-1))
        if self.w_ffn.numel() != self.dim or self.w_attn.numel() != self.dim:
            raise ValueError(f'norm weights must have {self.dim} values')
        lib = _lib.load()
        n = int(lib.localai_hip_layer_workspace_size(self.dim, self.ffn))
        if n < 0:
            raise ValueError('invalid layer sizes')
        self.ws = t.zeros(n, dtype=t.uint8, device=dev)      # zero-filled once; every launch leaves it so
        self._handles = (ctypes.c_void_p * 7)(*[m.handle.value for m in self.mats])

    def forward_device(self, pre, att, rope=None, out=None, stream=None):
        """pre, att: [dim] fp32 device tensors; rope: (cos, sin) [rope_half]
        fp32 device tensors or None. Returns (x_out [dim], q, k, v)."""
        t = device.torch()
        dev = pre.device
        if out is None:
            out = (t.empty(self.dim, dtype=t.float32, device=dev),
                   t.empty(self.mats[4].rows, dtype=t.float32, device=dev),
                   t.empty(self.mats[5].rows, dtype=t.float32, device=dev),
                   t.empty(self.mats[6].rows, dtype=t.float32, device=dev))
        x_out, q, k, v = out
        p = device.ptr
        cos, sin = rope if rope is not None else (None, None)
        if rope is not None and not self.head_dim:
            raise ValueError('RoPE needs head_dim')
        _lib.check(_lib.load().localai_hip_layer_chain(
            self._handles, p(pre), p(att), p(self.w_ffn), p(self.w_attn), ctypes.c_float(self.eps),
            p(cos) if cos is not None else None, p(sin) if sin is not None else None, self.head_dim,
            int(cos.numel()) if cos is not None else 0, p(x_out), p(q), p(k), p(v), p(self.ws), self.ws.numel(),
            ctypes.c_void_p(device.stream_ptr(stream))))
        return x_out, q, k, v

    def check(self, stream=None):
        """Wait for `stream`; raise if a wait between stages ran out."""
        _lib.check(_lib.load().localai_hip_layer_error(device.ptr(self.ws),
                                                       ctypes.c_void_p(device.stream_ptr(stream))))


_STRIDES = struct.Struct('=8q')


class _Norm:
    """What rms_norm() needs, looked up once."""

    def __init__(self):
        t = device.torch()
        self.types = {t.float32: 0, t.float16: 1, t.bfloat16: 30, 'q8_0': 8}     # GGML numbers
        self.call = _lib.load().localai_hip_rms_norm


_norm = None


def _norm_rows(t, name, dtype, shape):
    """(address, row stride, head stride) of t [rows, dim] or [rows, heads, dim]."""
    r = _r()
    if not (isinstance(t, r.Tensor) and t.dtype is dtype and t.get_device() == r.index and t.shape == shape):
        _refuse(t, name, dtype, shape)
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f'{name} must have adjacent values')
    # (the stride of a dimension of one says nothing)
    return (t.data_ptr(), stride[0] if shape[0] > 1 else 0,
            stride[1] if len(shape) == 3 and shape[1] > 1 else 0)


def rms_norm(x, weight, eps=1e-6, residual=None, gate=None, dtype=None, out=None, stream=None):
    """Root-mean-square norm of rows (localai_hip_rms_norm).

    x [rows, dim] or [rows, heads, dim]: fp32, f16 or bf16, any strides with
    adjacent values, each row (of each head) normed by itself; weight [dim] fp32.
    residual: fp32 of x's shape; x is added to it in place, and the sum is normed.
    gate: of x's type and shape; the result is multiplied by gate / (1 + exp(-gate)).
    dtype: the result's type, x's by default, or 'q8_0': uint8 [.., dim / 32 * 34],
    GGML Q8_0 blocks (dequant.dequantize_device reads them; then dim is a multiple of 32,
    and strides of 4 values). Returns the result, in `out` if given: x itself where the types are
    the same, or memory of its own."""
    global _norm
    _device_tensor(x, 'x')
    r = _r()
    if _norm is None:
        _norm = _Norm()
    given = x.dtype
    if dtype is None:
        dtype = given
    types = _norm.types
    kind, out_type = types.get(given), types.get(dtype)
    if kind is None:
        raise TypeError('x must be float32, float16 or bfloat16')
    if out_type is None:
        raise TypeError("dtype must be float32, float16, bfloat16 or 'q8_0'")
    shape = x.shape
    if len(shape) == 2:
        rows, dim = shape
        heads = 1
    elif len(shape) == 3:
        rows, heads, dim = shape
    else:
        raise ValueError('x must be [rows, dim] or [rows, heads, dim]')
    xp, *xs = _norm_rows(x, 'x', given, shape)
    wp = _ptr(weight, 'weight', r.f32, (dim,))
    rp, *rs = _norm_rows(residual, 'residual', r.f32, shape) if residual is not None else (None, 0, 0)
    gp, *gs = _norm_rows(gate, 'gate', given, shape) if gate is not None else (None, 0, 0)
    if out_type == 8:
        if dim % 32:
            raise ValueError("'q8_0' needs dim to be a multiple of 32")
        width, dtype = dim // 32 * 34, r.u8
        shape = (*shape[:-1], width)
    else:
        width = dim
    if out is None:
        out = _empty(stream, shape, dtype)
        op, os = out.data_ptr(), (heads * width, width)
    else:
        op, *os = _norm_rows(out, 'out', dtype, shape)
    status = _norm.call(xp, kind, _STRIDES.pack(*xs, *rs, *gs, *os), rows, heads, dim, wp, eps, rp, gp, op, out_type,
                        _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, x, weight, residual, gate, out)
    return out
