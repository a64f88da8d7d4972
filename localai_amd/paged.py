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
allocator call by call, so graphs and streams share none.
"""
from __future__ import annotations

import collections
import contextlib
import ctypes
import math

from . import _lib, device

# torch dtype name -> the cache's GGML type number
_TYPES = {'torch.float32': 0, 'torch.float16': 1, 'torch.bfloat16': 30}

_STATUS = ((1, 'the pool has too few pages left'),
           (2, 'a length or count is negative, or a request is longer than its page table'),
           (4, 'more new tokens than the step has places for'))


class Step(collections.namedtuple('Step', 'lengths used starts slots positions status')):
    """What extend() made (int32 device tensors): lengths [requests] with the
    new tokens, used [1], starts [requests + 1], and per token its slot and
    position (-1 behind the last token); status [1], 0 where all fitted."""
    __slots__ = ()

    def check(self):
        check(self.status)


def check(status):
    """Wait for `status` (of extend or shrink) and raise if it is not 0."""
    bits = int(status.item())
    if bits:
        raise RuntimeError('paged cache: ' + '; '.join(text for bit, text in _STATUS if bits & bit)
                           + ' (nothing was changed)')


def _tensor(t, name, dtype, shape=None, contiguous=True):
    torch = device.torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f'{name} must be a device tensor')
    if t.device.index != device.device().index:
        raise ValueError(f'{name} is on {t.device}, the library on {device.device()}')
    if t.dtype != dtype or (contiguous and not t.is_contiguous()):
        raise TypeError(f'{name} must be a {"contiguous " if contiguous else ""}{dtype} tensor')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must be {list(shape)}, got {list(t.shape)}')
    return t


def _stream(stream):
    """hipStream_t of `stream`, or of the library device's current stream."""
    torch = device.torch()
    if stream is not None:
        if stream.device.index != device.device().index:
            raise ValueError(f'the stream is on {stream.device}, the library on {device.device()}')
        return int(stream.cuda_stream)
    raw = getattr(torch._C, '_cuda_getCurrentRawStream', None)
    index = device.device().index
    return raw(index) if raw else int(torch.cuda.current_stream(index).cuda_stream)


def _on(stream):
    """Allocations inside belong to `stream`."""
    return contextlib.nullcontext() if stream is None else device.torch().cuda.stream(stream)


def _table(table):
    _tensor(table, 'table', device.torch().int32, contiguous=False)
    if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError('table must be [requests, pages] with adjacent pages')
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        raise ValueError('rows of table overlap')
    return max(table.stride(0), table.shape[1])


def extend(lengths, new, table, free, used, page_size, tokens, out=None, stream=None):
    """Give each request its new tokens' pages and slots (localai_hip_paged_extend).

    lengths, new [requests]: cached and new positions; table [requests, pages]
    is updated in place; free [n_pages] lists the pool's pages, the first
    used[0] of them in use; tokens: places for new tokens, at least as many as
    there are. Returns a Step; lengths and used change only if `out`, a Step
    to write to, holds them. All int32."""
    torch = device.torch()
    i32 = torch.int32
    stride = _table(table)
    n, width = table.shape
    _tensor(lengths, 'lengths', i32, (n,))
    _tensor(new, 'new', i32, (n,))
    _tensor(free, 'free', i32)
    _tensor(used, 'used', i32, (1,))
    tokens = int(tokens)
    if out is None:
        with _on(stream):
            new_lengths, rest = torch.empty(n, dtype=i32, device=table.device), torch.empty(
                n + 3, dtype=i32, device=table.device)
            places = torch.empty((2, tokens), dtype=i32, device=table.device)
        out = Step(new_lengths, rest[n + 1:n + 2], rest[:n + 1], places[0], places[1], rest[n + 2:])
    else:
        for t, name, shape in zip(out, Step._fields, ((n,), (1,), (n + 1,), (tokens,), (tokens,), (1,))):
            _tensor(t, name, i32, shape)
    _lib.check(_lib.load().localai_hip_paged_extend(
        lengths.data_ptr(), new.data_ptr(), n, table.data_ptr(), stride, width, free.data_ptr(), free.numel(),
        used.data_ptr(), int(page_size), tokens, out.lengths.data_ptr(), out.used.data_ptr(), out.starts.data_ptr(),
        out.slots.data_ptr(), out.positions.data_ptr(), out.status.data_ptr(), _stream(stream)))
    return out


def shrink(lengths, keep, table, free, used, page_size, stream=None):
    """Cut each request to its first keep positions (localai_hip_paged_shrink):
    lengths, table, free and used are updated in place. Returns the status [1]."""
    torch = device.torch()
    i32 = torch.int32
    stride = _table(table)
    n, width = table.shape
    _tensor(lengths, 'lengths', i32, (n,))
    _tensor(keep, 'keep', i32, (n,))
    _tensor(free, 'free', i32)
    _tensor(used, 'used', i32, (1,))
    with _on(stream):
        status = torch.empty(1, dtype=i32, device=table.device)
    _lib.check(_lib.load().localai_hip_paged_shrink(
        lengths.data_ptr(), keep.data_ptr(), n, table.data_ptr(), stride, width, free.data_ptr(), free.numel(),
        used.data_ptr(), int(page_size), status.data_ptr(), _stream(stream)))
    return status


def _cache(k, v):
    """localai_paged_cache of k, v [pages, kv heads, page size, head dim] (any strides with adjacent head values)."""
    torch = device.torch()
    _tensor(k, 'k_cache', k.dtype if isinstance(k, torch.Tensor) else None, contiguous=False)
    _tensor(v, 'v_cache', k.dtype, k.shape, contiguous=False)
    kind = _TYPES.get(str(k.dtype))
    if kind is None:
        raise TypeError('the cache must be float32, float16 or bfloat16')
    if k.dim() != 4 or k.stride(3) != 1 or k.stride() != v.stride():
        raise ValueError('k_cache and v_cache must be [pages, kv heads, page size, head dim] with the same strides '
                         'and adjacent head values')
    pages, nkv, page, hd = k.shape
    return _lib.PagedCacheArg(k.data_ptr(), v.data_ptr(), kind, nkv, hd, page, pages, k.stride(0), k.stride(1),
                              k.stride(2))


def _rows(t, name, tokens, heads, hd):
    """(pointer, token stride, head stride) of t [tokens, heads, hd] fp32."""
    _tensor(t, name, device.torch().float32, contiguous=False)
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != hd or (heads is not None and t.shape[1] != heads):
        raise ValueError(f'{name} must be [{tokens}, {heads if heads is not None else "heads"}, {hd}], '
                         f'got {list(t.shape)}')
    if hd > 1 and t.stride(2) != 1:
        raise ValueError(f'{name} must have adjacent head values')
    return t.data_ptr(), t.stride(0), t.stride(1)


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
    Returns q [tokens, heads, head_dim], in `out` if given (may be q); rows of
    padding are left as they were."""
    torch = device.torch()
    cache = _cache(k_cache, v_cache)
    tokens, hd = q.shape[0], cache.head_dim
    if rope not in ('halves', 'pairs'):
        raise ValueError("rope must be 'halves' or 'pairs'")
    qs = _rows(q, 'q', tokens, None, hd)
    ks, vs = _rows(k, 'k', tokens, cache.n_kv_heads, hd), _rows(v, 'v', tokens, cache.n_kv_heads, hd)
    heads = q.shape[1]
    _tensor(positions, 'positions', torch.int32, (tokens,))
    _tensor(slots, 'slots', torch.int32, (tokens,))
    n = 0
    if freq is not None:
        _tensor(freq, 'freq', torch.float64)
        n = freq.numel()
    for w, name in ((q_weight, 'q_weight'), (k_weight, 'k_weight')):
        if w is not None:
            _tensor(w, name, torch.float32, (hd,))
    if out is None:
        with _on(stream):
            out = torch.empty((tokens, heads, hd), dtype=torch.float32, device=q.device)
    os = _rows(out, 'out', tokens, heads, hd)
    strides = (ctypes.c_int64 * 8)(*qs[1:], *ks[1:], *vs[1:], *os[1:])
    p = lambda t: t.data_ptr() if t is not None else None
    _lib.check(_lib.load().localai_hip_norm_rope_store(
        qs[0], ks[0], vs[0], strides, tokens, heads, positions.data_ptr(), slots.data_ptr(), p(freq), n,
        1 if rope == 'halves' else 0, p(q_weight), p(k_weight), float(eps), os[0], ctypes.byref(cache),
        _stream(stream)))
    return out


def attention(q, k_cache, v_cache, table, lengths, starts=None, window=0, scale=None, gate=None, out=None,
              stream=None):
    """Attention of the new tokens over their requests' pages (localai_hip_paged_attention).

    q [tokens, heads, head_dim] fp32; table [requests, pages], lengths
    [requests] (the new tokens, already stored, counted) and starts
    [requests + 1] (None: one token per request) as extend() leaves them;
    window: the last positions a token sees, 0 for all; scale: 1 /
    sqrt(head_dim) by default; gate: Qwen3.5's output gate, like q. Returns
    [tokens, heads, head_dim]; rows behind starts[-1] of a given `out` stay as
    they were."""
    torch = device.torch()
    cache = _cache(k_cache, v_cache)
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError('q must be a tensor [tokens, heads, head_dim]')
    tokens, heads, hd = q.shape
    f32 = torch.float32
    _tensor(q, 'q', f32, (tokens, heads, cache.head_dim))
    stride = _table(table)
    n, width = table.shape
    _tensor(lengths, 'lengths', torch.int32, (n,))
    if starts is not None:
        _tensor(starts, 'starts', torch.int32, (n + 1,))
    if gate is not None:
        _tensor(gate, 'gate', f32, q.shape)
    lib = _lib.load()
    need = int(lib.localai_hip_paged_attention_workspace_size(tokens, n, heads, cache.n_kv_heads, hd))
    with _on(stream):
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        if out is None:
            out = torch.empty_like(q)
    _tensor(out, 'out', f32, q.shape)
    _lib.check(lib.localai_hip_paged_attention(
        q.data_ptr(), tokens, heads, ctypes.byref(cache), table.data_ptr(), stride, width, lengths.data_ptr(),
        starts.data_ptr() if starts is not None else None, n, int(max(window, 0)),
        1.0 / math.sqrt(hd) if scale is None else float(scale), gate.data_ptr() if gate is not None else None,
        out.data_ptr(), ws.data_ptr() if ws is not None else None, max(need, 0), _stream(stream)))
    return out


class PagedKVCache:
    """k, v [n_layers, n_pages, n_kv_heads, page_size, head_dim] (zero-filled)
    and the requests that share the pages: table [requests, max_pages] (-1: no
    page), lengths [requests], free [n_pages] and used [1]."""

    def __init__(self, n_layers, n_kv_heads, head_dim, n_pages, page_size=64, requests=1, max_pages=None, dtype=None):
        torch = device.torch()
        dev, i32 = device.device(), torch.int32
        dtype = dtype or torch.float32
        if str(dtype) not in _TYPES:
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

    def extend(self, new, tokens, out=None, stream=None):
        """Places for new[b] tokens of each request (of `tokens` in all at most);
        the cache's own lengths and used move on."""
        torch = device.torch()
        n, dev = self.lengths.numel(), self.lengths.device
        if out is None:
            with _on(stream):
                rest = torch.empty(n + 2, dtype=torch.int32, device=dev)
                places = torch.empty((2, int(tokens)), dtype=torch.int32, device=dev)
            out = Step(self.lengths, self.used, rest[:n + 1], places[0], places[1], rest[n + 1:])
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
