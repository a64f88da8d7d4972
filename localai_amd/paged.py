"""A paged key / value cache: several requests in one step, on the GPU.

    PagedKVCache      k and v of every layer in pages of `page_size` positions,
                      each request's page table and length, and the pool
    extend / shrink   page tables and slots of a step's new tokens from request
                      lengths, and pages given back
    norm_rope_store   q / k norms per head, the position rotation, and k / v
                      written to their slots, in one pass
    attention         the new tokens' grouped-query attention over the pages,
                      one token per request or several

A step of a server:

    step = cache.extend(new, tokens)             # once per step
    for each layer:
        q = cache.store(layer, q, k, v, step, freq, q_weight, k_weight)
        y = cache.attention(layer, q, step)
    step.check()                                 # waits; raises if the pool ran out

The reference serves one request from one contiguous cache
(engine/model.py:6-9, :203-227; engine/qwen35.py:158-182);
attention.attention_decode is that form. Arguments are device tensors, the
work runs in the HIP library, and nothing is read back by the host but by
check(). Every call may be captured in a graph; workspaces come from PyTorch's
allocator call by call, so graphs and streams share none. A call with `stream`
runs there, allocates there, and holds the memory of its arguments (a Step made
on another stream among them) until that stream has passed it; the streams' own
order is the caller's.
"""
from __future__ import annotations

import collections
import contextlib
import functools
import struct

from . import _lib, device

_STATUS = ((1, 'the pool has too few pages left'),
           (2, 'a length or count is negative, or a request is longer than its page table'),
           (4, 'more new tokens than the step has places for'))

_CACHE = struct.Struct('=QQiiiiqqqq')     # localai_paged_cache
_STRIDES = struct.Struct('=8q')


class _Run:
    """What every call needs, looked up once: a step makes several calls per
    layer, and looking the device up anew took half of their host time."""
    lib = None

    def __init__(self):
        t = device.torch()
        self.Tensor, self.empty, self.split = t.Tensor, t.empty, t.unsafe_split_with_sizes
        self.u8, self.i32, self.f32, self.f64 = t.uint8, t.int32, t.float32, t.float64
        self.types = {t.float32: 0, t.float16: 1, t.bfloat16: 30}     # of a cache -> its GGML number
        self.device = device.device()
        self.index = self.device.index
        self.raw_stream = getattr(t._C, '_cuda_getCurrentRawStream', None)
        lib = _lib.load()
        self.extend, self.shrink = lib.localai_hip_paged_extend, lib.localai_hip_paged_shrink
        self.store, self.attention = lib.localai_hip_norm_rope_store, lib.localai_hip_paged_attention
        self.workspace = functools.lru_cache(4096)(lib.localai_hip_paged_attention_workspace_size)


_run = None


def _r():
    global _run
    if _run is None:
        _run = _Run()
    return _run


class Step(collections.namedtuple('Step', 'lengths used starts slots positions status')):
    """What extend() made (int32 device tensors): lengths [requests] with the
    new tokens, used [1], starts [requests + 1], and per token its slot and
    position (-1 behind the last token); status [1], 0 where all fitted."""
    __slots__ = ()

    def check(self, stream=None):
        check(self.status, stream)


def check(status, stream=None):
    """Wait for `status` (of extend or shrink on `stream`, or on the current
    stream) and raise if it is not 0."""
    with _on(stream):
        bits = int(status.item())
    if bits:
        raise RuntimeError('paged cache: ' + '; '.join(text for bit, text in _STATUS if bits & bit)
                           + ' (nothing was changed)')


def _refuse(t, name, dtype, shape):
    torch = device.torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f'{name} must be a device tensor')
    if t.device.index != _r().index:
        raise ValueError(f'{name} is on {t.device}, the library on {_r().device}')
    if t.dtype != dtype:
        raise TypeError(f'{name} must be a {dtype} tensor')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must be {list(shape)}, got {list(t.shape)}')
    raise TypeError(f'{name} must be contiguous')


def _device_tensor(t, name):
    if not isinstance(t, device.torch().Tensor) or not t.is_cuda:
        raise TypeError(f'{name} must be a device tensor')
    return t


def _ptr(t, name, dtype, shape=None):
    """Address of a contiguous tensor of this type and shape on the library's device."""
    r = _run
    if (isinstance(t, r.Tensor) and t.dtype is dtype and t.get_device() == r.index and t.is_contiguous()
            and (shape is None or t.shape == shape)):
        return t.data_ptr()
    _refuse(t, name, dtype, shape)


def _stream(stream):
    """hipStream_t of `stream`, or of the library device's current stream."""
    r = _run
    if stream is None:
        if r.raw_stream:
            return r.raw_stream(r.index)
        return int(device.torch().cuda.current_stream(r.index).cuda_stream)
    if stream.device.index != r.index:
        raise ValueError(f'the stream is on {stream.device}, the library on {r.device}')
    return int(stream.cuda_stream)


def _on(stream):
    """Allocations inside belong to `stream`."""
    return contextlib.nullcontext() if stream is None else device.torch().cuda.stream(stream)


def _hold(stream, *tensors):
    """Memory of tensors freed before `stream` has passed this point is not given out again until it has."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def _empty(stream, shape, dtype):
    r = _run
    if stream is None:
        return r.empty(shape, dtype=dtype, device=r.device)
    with _on(stream):
        return r.empty(shape, dtype=dtype, device=r.device)


def _table(table):
    """(address, requests, pages, row stride) of a page table."""
    r = _run
    if not (isinstance(table, r.Tensor) and table.dtype is r.i32 and table.get_device() == r.index):
        _refuse(table, 'table', r.i32, None)
    if table.dim() != 2:
        raise ValueError('table must be [requests, pages]')
    n, width = table.shape
    stride, step = table.stride()
    if step != 1 and width > 1:
        raise ValueError('a request\'s pages must be adjacent in table')
    if stride < width:
        if n > 1:
            raise ValueError('rows of table overlap')
        stride = width
    return table.data_ptr(), n, width, stride


def _step_buffers(r, stream, n, tokens, lengths=None, used=None):
    """A Step of new tensors (but for lengths and used, if given), views of one allocation."""
    own = lengths is None
    buf = _empty(stream, n + 2 + 2 * tokens + (n + 1 if own else 0), r.i32)
    if own:
        starts, status, slots, positions, lengths, used = r.split(buf, (n + 1, 1, tokens, tokens, n, 1))
    else:
        starts, status, slots, positions = r.split(buf, (n + 1, 1, tokens, tokens))
    return Step(lengths, used, starts, slots, positions, status)


def extend(lengths, new, table, free, used, page_size, tokens, out=None, stream=None):
    """Give each request its new tokens' pages and slots (localai_hip_paged_extend).

    lengths, new [requests]: cached and new positions; table [requests, pages]
    is updated in place; free [n_pages] lists the pool's pages, the first
    used[0] of them in use; tokens: places for new tokens, at least as many as
    there are. Returns a Step; lengths and used change only if `out`, a Step
    to write to, holds them. All int32."""
    _device_tensor(table, 'table')
    r = _r()
    i32 = r.i32
    at, n, width, stride = _table(table)
    tokens = int(tokens)
    if not 0 < page_size < 1 << 31:
        raise ValueError('page_size must be a power of two, at least 16')
    args = (_ptr(lengths, 'lengths', i32, (n,)), _ptr(new, 'new', i32, (n,)), n, at, stride, width,
            _ptr(free, 'free', i32), free.numel(), _ptr(used, 'used', i32, (1,)), int(page_size), tokens)
    if tokens < 0:
        raise ValueError('tokens must not be negative')
    if out is None:
        out = _step_buffers(r, stream, n, tokens)
        ptrs = [t.data_ptr() for t in out]
    else:
        ptrs = [_ptr(t, name, i32, (size,)) for t, name, size in zip(out, Step._fields, (n, 1, n + 1, tokens, tokens, 1))]
    status = r.extend(*args, *ptrs, _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, lengths, new, table, free, used, *out)
    return out


def shrink(lengths, keep, table, free, used, page_size, stream=None):
    """Cut each request to its first keep positions (localai_hip_paged_shrink):
    lengths, table, free and used are updated in place. Returns the status [1]."""
    _device_tensor(table, 'table')
    r = _r()
    i32 = r.i32
    at, n, width, stride = _table(table)
    if not 0 < page_size < 1 << 31:
        raise ValueError('page_size must be a power of two, at least 16')
    args = (_ptr(lengths, 'lengths', i32, (n,)), _ptr(keep, 'keep', i32, (n,)), n, at, stride, width,
            _ptr(free, 'free', i32), free.numel(), _ptr(used, 'used', i32, (1,)), int(page_size))
    status = _empty(stream, 1, i32)
    _lib.check(r.shrink(*args, status.data_ptr(), _stream(stream)))
    if stream is not None:
        _hold(stream, lengths, keep, table, free, used)
    return status


def _cache(k, v):
    """(localai_paged_cache, kv heads, head dim) of k, v [pages, kv heads, page size, head dim] (any strides with
    adjacent head values)."""
    _device_tensor(k, 'k_cache')
    r = _r()
    kind = r.types.get(k.dtype)
    if kind is None:
        raise TypeError('the cache must be float32, float16 or bfloat16')
    if k.get_device() != r.index:
        _refuse(k, 'k_cache', k.dtype, None)
    if not (isinstance(v, r.Tensor) and v.dtype is k.dtype and v.get_device() == r.index and v.shape == k.shape):
        _refuse(v, 'v_cache', k.dtype, k.shape)
    strides = k.stride()
    if len(strides) != 4 or strides[3] != 1 or v.stride() != strides:
        raise ValueError('k_cache and v_cache must be [pages, kv heads, page size, head dim] with the same strides '
                         'and adjacent head values')
    pages, nkv, page, hd = k.shape
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), kind, nkv, hd, page, pages, *strides[:3]), nkv, hd


def _rows(t, name, tokens, heads, hd):
    """(address, token stride, head stride) of t [tokens, heads, hd] fp32."""
    r = _run
    if not (isinstance(t, r.Tensor) and t.dtype is r.f32 and t.get_device() == r.index and t.shape == (tokens, heads, hd)):
        _refuse(t, name, r.f32, (tokens, heads, hd))
    ts, hs, step = t.stride()
    if step != 1:
        raise ValueError(f'{name} must have adjacent head values')
    return t.data_ptr(), ts, hs


def norm_rope_store(q, k, v, positions, slots, k_cache, v_cache, freq=None, q_weight=None, k_weight=None, eps=1e-6,
                    rope='halves', out=None, stream=None):
    """Norm and rotate q and k, store k and v (localai_hip_norm_rope_store).

    q [tokens, heads, head_dim], k, v [tokens, kv heads, head_dim]: fp32, any
    token and head strides that are multiples of 4 values (views of one fused
    projection); positions, slots [tokens] as extend() makes them, a slot
    outside the cache marking padding; k_cache, v_cache [pages, kv heads, page
    size, head_dim] of one layer. freq: fp64 radians per position and rotated
    pair, or None; rope: 'halves' (j, j + n) or 'pairs' (2j, 2j + 1).
    q_weight, k_weight [head_dim]: the norms' weights, None for no norm.
    Returns q [tokens, heads, head_dim], in `out` if given (q itself, or rows
    that share no memory with each other or the rest); rows of padding are left
    as they were, in a new result whatever its memory held."""
    cache, nkv, hd = _cache(k_cache, v_cache)
    r = _r()
    f32 = r.f32
    if rope not in ('halves', 'pairs'):
        raise ValueError("rope must be 'halves' or 'pairs'")
    _device_tensor(q, 'q')
    if q.dim() != 3:
        raise ValueError('q must be [tokens, heads, head_dim]')
    tokens, heads, _ = q.shape
    qp, *qs = _rows(q, 'q', tokens, heads, hd)
    kp, *ks = _rows(k, 'k', tokens, nkv, hd)
    vp, *vs = _rows(v, 'v', tokens, nkv, hd)
    at = _ptr(positions, 'positions', r.i32, (tokens,)), _ptr(slots, 'slots', r.i32, (tokens,))
    fp, n = (_ptr(freq, 'freq', r.f64), freq.numel()) if freq is not None else (None, 0)
    qw = _ptr(q_weight, 'q_weight', f32, (hd,)) if q_weight is not None else None
    kw = _ptr(k_weight, 'k_weight', f32, (hd,)) if k_weight is not None else None
    if out is None:
        out = _empty(stream, (tokens, heads, hd), f32)
        op, os = out.data_ptr(), (heads * hd, hd)
    else:
        op, *os = _rows(out, 'out', tokens, heads, hd)
    status = r.store(qp, kp, vp, _STRIDES.pack(*qs, *ks, *vs, *os), tokens, heads, *at, fp, n, rope == 'halves', qw, kw,
                     eps, op, cache, _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, q, k, v, positions, slots, k_cache, v_cache, freq, q_weight, k_weight, out)
    return out


def attention(q, k_cache, v_cache, table, lengths, starts=None, window=0, scale=None, gate=None, out=None,
              stream=None):
    """Attention of the new tokens over their requests' pages (localai_hip_paged_attention).

    q [tokens, heads, head_dim] fp32; table [requests, pages], lengths
    [requests] (the new tokens, already stored, counted) and starts
    [requests + 1] (None: one token per request) as extend() leaves them;
    window: the last positions a token sees, 0 for all; scale: 1 /
    sqrt(head_dim) by default; gate: Qwen3.5's output gate, like q. Returns
    [tokens, heads, head_dim]; rows behind starts[-1] stay as they were in
    `out`, and hold whatever was in the memory of a new result. `out` may be q;
    it shares memory with nothing else."""
    cache, nkv, hd = _cache(k_cache, v_cache)
    r = _r()
    f32 = r.f32
    _device_tensor(q, 'q')
    if q.dim() != 3:
        raise ValueError('q must be [tokens, heads, head_dim]')
    shape = tokens, heads, _ = q.shape
    qp = _ptr(q, 'q', f32, (tokens, heads, hd))
    tp, n, width, stride = _table(table)
    lp = _ptr(lengths, 'lengths', r.i32, (n,))
    sp = _ptr(starts, 'starts', r.i32, (n + 1,)) if starts is not None else None
    gp = _ptr(gate, 'gate', f32, shape) if gate is not None else None
    need = r.workspace(tokens, n, heads, nkv, hd)
    ws = _empty(stream, need, r.u8) if need > 0 else None
    if out is None:
        out = _empty(stream, shape, f32)
        op = out.data_ptr()
    else:
        op = _ptr(out, 'out', f32, shape)
    status = r.attention(qp, tokens, heads, cache, tp, stride, width, lp, sp, n, min(int(window), 1 << 31) if window > 0 else 0,
                         hd ** -0.5 if scale is None else scale, gp, op, ws.data_ptr() if need > 0 else None,
                         need if need > 0 else 0, _stream(stream))
    if status:
        _lib.check(status)
    if stream is not None:
        _hold(stream, q, k_cache, v_cache, table, lengths, starts, gate, out)
    return out


class PagedKVCache:
    """k, v [n_layers, n_pages, n_kv_heads, page_size, head_dim] (zero-filled)
    and the requests that share the pages: table [requests, max_pages] (-1: no
    page), lengths [requests], free [n_pages] and used [1]."""

    def __init__(self, n_layers, n_kv_heads, head_dim, n_pages, page_size=64, requests=1, max_pages=None, dtype=None):
        torch = device.torch()
        dev, i32 = device.device(), torch.int32
        dtype = dtype or torch.float32
        if dtype not in _r().types:
            raise TypeError('the cache must be float32, float16 or bfloat16')
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError('page_size must be a power of two, at least 16')
        self.page_size, self.n_pages = int(page_size), int(n_pages)
        self.k = torch.zeros((n_layers, n_pages, n_kv_heads, page_size, head_dim), dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.table = torch.full((requests, max_pages or n_pages), -1, dtype=i32, device=dev)
        self.lengths = torch.zeros(requests, dtype=i32, device=dev)
        self.free = torch.arange(n_pages, dtype=i32, device=dev)
        self.used = torch.zeros(1, dtype=i32, device=dev)

    def reset(self):
        """Every request ends, every page is free."""
        self.table.fill_(-1)
        self.lengths.zero_()
        self.free.copy_(device.torch().arange(self.n_pages, dtype=self.free.dtype, device=self.free.device))
        self.used.zero_()

    def extend(self, new, tokens, stream=None):
        """Places for new[b] tokens of each request (of `tokens` in all at most);
        the cache's own lengths and used move on."""
        out = _step_buffers(_r(), stream, self.lengths.numel(), int(tokens), self.lengths, self.used)
        return extend(self.lengths, new, self.table, self.free, self.used, self.page_size, tokens, out, stream)

    def shrink(self, keep, stream=None):
        """Each request keeps its first keep[b] positions (0: it ends). Returns the status, for check()."""
        return shrink(self.lengths, keep, self.table, self.free, self.used, self.page_size, stream)

    def store(self, layer, q, k, v, step, freq=None, q_weight=None, k_weight=None, eps=1e-6, rope='halves', out=None,
              stream=None):
        return norm_rope_store(q, k, v, step.positions, step.slots, self.k[layer], self.v[layer], freq, q_weight,
                               k_weight, eps, rope, out, stream)

    def attention(self, layer, q, step, window=0, scale=None, gate=None, out=None, stream=None):
        return attention(q, self.k[layer], self.v[layer], self.table, self.lengths, step.starts, window, scale, gate,
                         out, stream)
