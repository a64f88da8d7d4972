"""The paged cache without a GPU: its oracle's pins, the C ABI's refusals
before any device use, and the Python checks that need no device."""
import ctypes

import numpy as np
import pytest

from localai_amd import _lib
from oracle import attention as oatt
from oracle import paged as opaged

ONE = ctypes.c_void_p(16)


def test_tables_pages_and_shrink_is_the_inverse():
    t = opaged.Tables([0, 0], [[-1] * 3, [-1] * 3], [4, 2, 0, 1, 3, 5], 0, 16)
    status, starts, slots, positions = t.extend([17, 3], 24)
    assert (status, starts, t.used, t.lengths) == (0, [0, 17, 20], 3, [17, 3])
    assert positions == list(range(17)) + [0, 1, 2] + [-1] * 4
    assert slots == list(range(64, 80)) + [32] + [0, 1, 2] + [-1] * 4
    before = ([list(r) for r in t.table], t.used, list(t.lengths))
    t.extend([15, 14], 40)
    assert t.used == 4 and t.table[0][:2] == [4, 2] and t.table[1][:2] == [0, 1]
    t.shrink([17, 3])
    assert (t.table, t.used, t.lengths) == before and t.free == [4, 2, 0, 1, 3, 5]
    assert t.extend([40, 0], 64)[0] == 2 and t.extend([16, 16], 31)[0] == 4


def test_rotation_is_complex_multiplication():
    rng = np.random.default_rng(0)
    x, freq = rng.standard_normal((3, 16)), rng.uniform(0, 2, 5)
    turn = np.exp(1j * 7 * freq)
    pairs = opaged.norm_rope(x, 7, freq, None, 0, 'pairs')
    z = (x[:, 0:10:2] + 1j * x[:, 1:10:2]) * turn
    np.testing.assert_allclose(pairs[:, 0:10:2] + 1j * pairs[:, 1:10:2], z, atol=1e-12)
    halves = opaged.norm_rope(x, 7, freq, None, 0, 'halves')
    z = (x[:, :5] + 1j * x[:, 5:10]) * turn
    np.testing.assert_allclose(halves[:, :5] + 1j * halves[:, 5:10], z, atol=1e-12)
    np.testing.assert_array_equal(pairs[:, 10:], x[:, 10:])
    unit = opaged.norm_rope(x, 0, freq, np.ones(16), 0, 'pairs')
    np.testing.assert_allclose(np.mean(unit * unit, axis=1), 1)


@pytest.mark.parametrize('window', [0, 5])
def test_attention_oracle_is_gqa_decode(window):
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((20, 2, 64)).astype(np.float32) for _ in range(2))
    q, gate = rng.standard_normal((3, 6, 64)), rng.standard_normal((3, 6, 64))
    out, _, _ = opaged.attention(q, k, v, 3, opaged.default_scale(64), window, gate)
    for i in range(3):
        want, _, _ = oatt.gqa_decode(q[i], k, v, 17 + i, 6, 2, 64, window=window, gate=gate[i])
        np.testing.assert_allclose(out[i].reshape(-1), want, rtol=1e-10)


def cache_arg(**change):
    a = dict(k_dev=16, v_dev=16, type=1, n_kv_heads=2, head_dim=128, page_size=16, n_pages=8,
             page_stride=2 * 16 * 128, head_stride=16 * 128, pos_stride=128)
    a.update(change)
    return _lib.PagedCacheArg(**a)


BAD_CACHES = [
    (dict(k_dev=None), 1), (dict(v_dev=None), 1), (dict(k_dev=24), 1), (dict(v_dev=8), 1),
    (dict(type=2), 2), (dict(head_dim=96), 2), (dict(head_dim=0), 2), (dict(n_kv_heads=0), 1),
    (dict(page_size=8), 1), (dict(page_size=24), 1), (dict(page_size=0), 1), (dict(page_size=-16), 1),
    (dict(n_pages=0), 1), (dict(n_pages=1 << 28), 1), (dict(pos_stride=64), 1), (dict(pos_stride=132), 1),
    (dict(head_stride=0), 1), (dict(page_stride=0), 1), (dict(pos_stride=-128), 1), (dict(pos_stride=1 << 40), 1),
]


@pytest.mark.parametrize('change,status', BAD_CACHES)
def test_bad_caches_are_refused(change, status):
    lib, c = _lib.load(), cache_arg(**change)
    strides = (ctypes.c_int64 * 8)(*[512] * 8)
    assert lib.localai_hip_paged_attention(ONE, 2, 4, ctypes.byref(c), ONE, 8, 8, ONE, None, 2, 0, 1.0, None, ONE,
                                           ONE, 1 << 40, None) == status
    assert lib.localai_hip_norm_rope_store(ONE, ONE, ONE, strides, 2, 4, ONE, ONE, ONE, 64, 0, None, None, 1e-6, ONE,
                                           ctypes.byref(c), None) == status
    assert lib.localai_hip_last_error()


def test_attention_arguments_are_refused():
    lib, c = _lib.load(), cache_arg()

    def call(q=ONE, tokens=2, heads=4, cache=ctypes.byref(c), table=ONE, stride=8, pages=8, lengths=ONE, starts=None,
             requests=2, window=0, scale=1.0, gate=None, out=ONE, ws=ONE, ws_bytes=1 << 40):
        return lib.localai_hip_paged_attention(q, tokens, heads, cache, table, stride, pages, lengths, starts,
                                               requests, window, scale, gate, out, ws, ws_bytes, None)

    odd = ctypes.c_void_p(20)
    for change in (dict(q=None), dict(q=odd), dict(tokens=-1), dict(tokens=1 << 31), dict(heads=0), dict(heads=3),
                   dict(heads=65536), dict(cache=None), dict(table=None), dict(stride=7), dict(pages=0),
                   dict(pages=1 << 28, stride=1 << 28), dict(lengths=None), dict(requests=0), dict(requests=4097),
                   dict(tokens=3), dict(window=-1), dict(scale=float('nan')), dict(scale=float('inf')),
                   dict(tokens=1 << 24, starts=ONE), dict(gate=odd), dict(out=None), dict(out=odd), dict(ws=odd)):
        assert call(**change) == 1, change
    need = lib.localai_hip_paged_attention_workspace_size(2, 2, 4, 2, 128)
    if need > 0:
        assert call(ws=None) == 1 and call(ws_bytes=need - 1) == 1
    assert call(tokens=0, starts=ONE) == 0           # nothing to do, nothing touched
    size = lib.localai_hip_paged_attention_workspace_size
    assert size(-1, 1, 4, 2, 128) == size(1, 0, 4, 2, 128) == size(1, 1, 4, 3, 128) == size(1, 1, 4, 2, 96) == -1


@pytest.mark.parametrize('tokens,requests,heads,kv_heads,head_dim', [
    (8192, 1, 32, 8, 128), (131072, 1, 32, 8, 128), (131072, 64, 64, 8, 128), (1 << 20, 4096, 16, 4, 256),
    (4096, 4096, 32, 8, 128), (8192, 4096, 8, 8, 64), (1, 1, 32, 8, 128), (3, 2, 8, 2, 64)])
def test_attention_workspace_holds_cut_blocks_only(tokens, requests, heads, kv_heads, head_dim):
    """8 bytes a token, and partial results of at most twice the chunks that a call may cut (four rounds of two
    workgroups for each of 256 CUs) of 32 columns: not of every block of a prompt."""
    size = _lib.load().localai_hip_paged_attention_workspace_size(tokens, requests, heads, kv_heads, head_dim)
    assert 0 < size <= 8 * tokens + 2 * 4 * 512 * 32 * (head_dim * 4 + 8) + 3 * 256


def test_store_arguments_are_refused():
    lib, c = _lib.load(), cache_arg()

    def call(q=ONE, k=ONE, v=ONE, strides=(512,) * 8, tokens=2, heads=4, positions=ONE, slots=ONE, freq=ONE, n=64,
             halves=0, out=ONE, cache=ctypes.byref(c)):
        return lib.localai_hip_norm_rope_store(q, k, v, (ctypes.c_int64 * 8)(*strides), tokens, heads, positions,
                                               slots, freq, n, halves, None, None, 1e-6, out, cache, None)

    odd = ctypes.c_void_p(20)
    for change in (dict(q=None), dict(k=None), dict(v=None), dict(q=odd), dict(k=odd), dict(v=odd), dict(out=odd),
                   dict(out=None), dict(strides=(512,) * 7 + (510,)), dict(strides=(-512,) + (512,) * 7),
                   dict(tokens=-1), dict(tokens=1 << 24), dict(heads=0), dict(positions=None), dict(slots=None), dict(freq=None),
                   dict(n=65), dict(n=-1), dict(halves=2), dict(cache=None)):
        assert call(**change) == 1, change
    assert call(tokens=0) == 0


@pytest.mark.parametrize('tokens,heads,ts,hs,overlap', [
    (2, 4, 512, 128, False), (2, 4, 128, 256, False), (1, 4, 0, 128, False), (3, 1, 128, 0, False), (1, 1, 0, 0, False),
    (2, 4, 512, 512, True), (2, 4, 0, 128, True), (2, 4, 512, 0, True), (2, 4, 384, 128, True), (5, 4, 128, 512, True),
    (4, 3, 384, 512, False), (5, 4, 384, 512, True), (5, 4, 384, 516, True), (2, 4, 64, 1024, True),
    (1 << 20, 65536, 128, 1 << 27, False), (1 << 20, 65536, 128, (1 << 27) - 128, True)])
def test_store_outputs_that_overlap_are_refused(tokens, heads, ts, hs, overlap):
    """Every row writes its own memory: rows that share some would be written by two workgroups."""
    import itertools
    hd, lib = 128, _lib.load()
    if tokens * heads < 100:
        taken = [t * ts + h * hs for t, h in itertools.product(range(tokens), range(heads))]
        assert overlap == any(abs(a - b) < hd for i, a in enumerate(taken) for b in taken[:i])
    strides = (ctypes.c_int64 * 8)(512, 128, 512, 128, 512, 128, ts, hs)
    c = cache_arg(n_kv_heads=1)
    status = lib.localai_hip_norm_rope_store(ONE, ONE, ONE, strides, tokens, heads, ONE, ONE, None, 0, 0, None, None,
                                             1e-6, ctypes.c_void_p(20), ctypes.byref(c), None)     # q_out: misaligned
    assert status == 1
    assert (b'overlap' in lib.localai_hip_last_error()) == overlap


def test_table_arguments_are_refused():
    lib = _lib.load()

    def extend(ptrs=(ONE,) * 11, requests=2, stride=8, pages=8, pool=8, page=16, tokens=4):
        a = iter(ptrs)
        return lib.localai_hip_paged_extend(next(a), next(a), requests, next(a), stride, pages, next(a), pool, next(a),
                                            page, tokens, *a, None)

    def shrink(ptrs=(ONE,) * 6, requests=2, stride=8, pages=8, pool=8, page=16):
        a = iter(ptrs)
        return lib.localai_hip_paged_shrink(next(a), next(a), requests, next(a), stride, pages, next(a), pool, next(a),
                                            page, next(a), None)

    for f, n in ((extend, 11), (shrink, 6)):
        for i in range(n):
            assert f(ptrs=tuple(None if j == i else ONE for j in range(n))) == 1, (f, i)
        for change in (dict(requests=0), dict(requests=4097), dict(stride=7), dict(pages=0), dict(pool=0),
                       dict(pool=1 << 28), dict(page=8), dict(page=48), dict(pages=1 << 28, stride=1 << 28)):
            assert f(**change) == 1, change
    assert extend(tokens=-1) == extend(tokens=1 << 31) == 1


def test_python_checks_without_a_device():
    import torch
    from localai_amd import paged
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match='device tensor'):
        paged.extend(z, z, z.reshape(1, 2), z, z, 16, 4)
    x = torch.zeros(1, 2, 64)
    with pytest.raises(TypeError, match='device tensor'):
        paged.attention(x, x[None], x[None], z.reshape(1, 2), z)
    with pytest.raises(TypeError, match='device tensor'):
        paged.norm_rope_store(x, x, x, z, z, x[None], x[None])
    with pytest.raises(RuntimeError, match='too few pages.*places'):
        paged.check(torch.tensor([5]))


def test_packed_cache_argument_is_the_c_structure():
    from localai_amd import paged
    c = cache_arg(k_dev=0x1234567890, v_dev=0x987654320, type=30, page_stride=1 << 40)
    fields = [getattr(c, n) for n, _ in c._fields_]
    assert paged._CACHE.pack(*fields) == bytes(c)
    assert paged._STRIDES.pack(*range(8)) == bytes((ctypes.c_int64 * 8)(*range(8)))
