"""The linear-attention layers' operators without a GPU: their oracle's pins, the
C ABI's refusals before any device use, and the Python checks that need no device."""
import ctypes

import numpy as np
import pytest

from localai_amd import _lib
from oracle import attention as oatt
from oracle import delta as odelta
from oracle import quant

ONE = ctypes.c_void_p(16)


@pytest.mark.parametrize('order', ['grouped', 'tiled'])
def test_rule_is_the_step_token_by_token(order):
    rng = np.random.default_rng(0)
    q, k = rng.standard_normal((2, 5, 2, 8))
    v, S = rng.standard_normal((5, 6, 4)), rng.standard_normal((6, 8, 4))
    g, b = -rng.random((5, 6)), rng.random((5, 6))
    out, after = odelta.rule(S, q, k, v, g, b, order=order, norm_eps=None, scale=1.0)
    for t in range(5):
        heads = [h // 3 if order == 'grouped' else h % 2 for h in range(6)]
        S, core = oatt.delta_net_step_f64(S, q[t, heads], k[t, heads], v[t], g[t], b[t])
        np.testing.assert_allclose(out[t], core, rtol=1e-12)
    np.testing.assert_allclose(after, S, rtol=1e-12)


def test_rule_norms_and_gates():
    from scipy import special
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((2, 3, 1, 16))
    v, S = rng.standard_normal((3, 2, 4)), np.zeros((2, 16, 4))
    x, y, a, dt = rng.standard_normal((3, 2)), rng.standard_normal((3, 2)), -rng.random(2), rng.standard_normal(2)
    g, b = odelta.gates(x, y, a, dt)
    np.testing.assert_allclose(g, a * -special.log_expit(-(x + dt)), rtol=1e-12)
    np.testing.assert_allclose(b, special.expit(y), rtol=1e-12)
    # a unit key read back at once gives beta v, whatever the key's length
    out, _ = odelta.rule(S, 5 * k, 0.1 * k, v, x, y, a, dt, norm_eps=0.0, scale=1.0)
    np.testing.assert_allclose(out[0], b[0][:, None] * v[0], rtol=1e-12)


def test_conv_is_a_convolution_and_keeps_rows():
    rng = np.random.default_rng(2)
    x, w, before = rng.standard_normal((9, 3)), rng.standard_normal((3, 4)), rng.standard_normal((3, 3))
    y, after, _ = odelta.conv(before, x, w, silu=False)
    for c in range(3):
        line = np.concatenate([before[:, c], x[:, c]])
        np.testing.assert_allclose(y[:, c], np.convolve(line, w[c, ::-1], 'valid'), rtol=1e-12)
    np.testing.assert_array_equal(after, x[-3:])
    first, middle, _ = odelta.conv(before, x[:2], w)
    np.testing.assert_array_equal(middle, [before[2], x[0], x[1]])
    rest, _, _ = odelta.conv(middle, x[2:], w)
    np.testing.assert_allclose(np.concatenate([first, rest]), odelta.conv(before, x, w)[0], rtol=1e-12)


def test_rms_norm_and_blocks():
    rng = np.random.default_rng(3)
    x, r, z = rng.standard_normal((3, 4, 64))
    y, h = odelta.rms_norm(x, np.ones(64), 0.0, r)
    np.testing.assert_allclose((y * y).mean(-1), 1, rtol=1e-12)
    np.testing.assert_allclose(h, x + r)
    np.testing.assert_allclose(odelta.rms_norm(x, np.ones(64), 0.0, r, z)[0], y * z / (1 + np.exp(-z)))
    d, q = odelta.q8_0(y)
    raw = np.concatenate([d[..., None].view(np.uint8), q.view(np.uint8)], -1).tobytes()
    back = np.asarray(quant.dequantize(raw, 8, (4, 64)), np.float64)
    assert (np.abs(back - y) <= np.repeat(d.astype(np.float64), 32, -1) * 0.5 * (1 + 2.0 ** -10)).all()


def requests(**change):
    a = dict(state_dev=16, n_slots=4, slots_dev=16, starts_dev=16, lengths_dev=16, requests=3)
    a.update(change)
    return _lib.DeltaRequestsArg(**a)


def refused(status):
    message = _lib.load().localai_hip_last_error().decode()
    assert status and message
    return {1: 'EARG', 2: 'ETYPE'}[status]


def conv(r=None, **change):
    a = dict(x=ONE, type=0, tokens=5, channels=64, x_stride=64, weight=ONE, bias=None, width=4, silu=1,
             requests=ctypes.byref(r or requests()), out=ONE, out_stride=64, stream=None)
    a.update(change)
    return _lib.load().localai_hip_delta_conv(*a.values())


@pytest.mark.parametrize('change,status', [
    (dict(x=None), 'EARG'), (dict(weight=None), 'EARG'), (dict(out=None), 'EARG'), (dict(requests=None), 'EARG'),
    (dict(type=8), 'ETYPE'), (dict(width=1), 'ETYPE'), (dict(width=9), 'ETYPE'), (dict(channels=0), 'EARG'),
    (dict(channels=(1 << 20) + 1), 'EARG'), (dict(tokens=-1), 'EARG'), (dict(tokens=1 << 24), 'EARG'),
    (dict(out_stride=63), 'EARG'), (dict(x_stride=-1), 'EARG'), (dict(silu=2), 'EARG')])
def test_conv_refusals(change, status):
    assert refused(conv(**change)) == status


@pytest.mark.parametrize('change', [dict(state_dev=None), dict(requests=0), dict(requests=4097), dict(n_slots=0),
                                    dict(starts_dev=None), dict(n_slots=1 << 62)])
def test_request_refusals(change):
    assert refused(conv(requests(**change))) == 'EARG'
    assert refused(rule(requests(**change))) == 'EARG'


def rule(r=None, strides=(256, 128, 256, 128, 512, 128, 512, 128, 4, 4), **change):
    a = dict(q=ONE, k=ONE, v=ONE, type=0, strides=(ctypes.c_int64 * 10)(*strides), tokens=5, key_heads=2, value_heads=4,
             key_dim=128, value_dim=128, decay=ONE, beta=ONE, a=None, dt_bias=None, tiled=0,
             norm_eps=ctypes.c_float(1e-6), scale=ctypes.c_float(0.1), requests=ctypes.byref(r or requests()), out=ONE,
             ws=ONE, ws_bytes=1 << 40, stream=None)
    a.update(change)
    return _lib.load().localai_hip_delta_rule(*a.values())


@pytest.mark.parametrize('change,status', [
    (dict(q=None), 'EARG'), (dict(k=None), 'EARG'), (dict(v=None), 'EARG'), (dict(strides=None), 'EARG'),
    (dict(decay=None), 'EARG'), (dict(beta=None), 'EARG'), (dict(out=None), 'EARG'), (dict(a=ONE), 'EARG'),
    (dict(dt_bias=ONE), 'EARG'), (dict(type=1 << 20), 'ETYPE'), (dict(key_dim=96), 'ETYPE'),
    (dict(value_dim=100), 'ETYPE'), (dict(value_dim=1040), 'ETYPE'), (dict(value_dim=0), 'ETYPE'),
    (dict(key_heads=3), 'EARG'), (dict(key_heads=0), 'EARG'), (dict(value_heads=0), 'EARG'),
    (dict(value_heads=4098), 'EARG'), (dict(tiled=2), 'EARG'), (dict(tokens=-1), 'EARG'), (dict(tokens=1 << 24), 'EARG'),
    (dict(scale=ctypes.c_float(np.inf)), 'EARG'), (dict(norm_eps=ctypes.c_float(np.nan)), 'EARG'),
    (dict(q=ctypes.c_void_p(20)), 'EARG'), (dict(out=ctypes.c_void_p(24)), 'EARG'), (dict(ws=ctypes.c_void_p(24)), 'EARG')])
def test_rule_refusals(change, status):
    if 'strides' in change:
        args = dict(change)
        args.pop('strides')
        r = requests()
        f = _lib.load().localai_hip_delta_rule
        assert refused(f(ONE, ONE, ONE, 0, None, 5, 2, 4, 128, 128, ONE, ONE, None, None, 0, ctypes.c_float(1e-6),
                         ctypes.c_float(1), ctypes.byref(r), ONE, ONE, 1 << 40, None)) == status
        return
    assert refused(rule(**change)) == status


def test_rule_refuses_strides_and_overlaps():
    good = (256, 128, 256, 128, 512, 128, 512, 128, 4, 4)
    for i, value in [(0, 258), (1, -128), (5, 130), (8, -1), (6, 384), (7, 64)]:
        s = list(good)
        s[i] = value
        assert refused(rule(strides=s)) == 'EARG', (i, value)
    assert refused(rule(requests(requests=4096), value_heads=4096, key_heads=1, value_dim=1024,
                        strides=(128, 0, 128, 0, 1 << 22, 1024, 1 << 22, 1024, 4096, 4096))) == 'EARG'


def test_rule_workspace_size():
    size = _lib.load().localai_hip_delta_rule_workspace_size
    assert size(7, 7, 0, 2, 4, 128, 128) == 0
    for bad in [(-1, 1, 1, 2, 4, 128, 128), (1 << 24, 1, 1, 2, 4, 128, 128), (1, 0, 1, 2, 4, 128, 128),
                (1, 4097, 1, 2, 4, 128, 128), (1, 1, 1, 3, 4, 128, 128), (1, 1, 1, 2, 4, 32, 128),
                (1, 1, 1, 2, 4, 128, 8)]:
        assert size(*bad) == -1, bad


def test_rule_sizes_that_no_launch_holds():
    """Workgroups of 512 threads for prompts, 256 for a step: fewer than 2^32 threads; refused before anything is queued."""
    size = _lib.load().localai_hip_delta_rule_workspace_size
    for n, starts, hk, hv, vd, fits in [
            (4096, 1, 64, 64, 512, False), (4095, 1, 64, 64, 512, True), (4096, 0, 64, 64, 512, True),
            (4096, 0, 64, 64, 1024, False), (4095, 0, 64, 64, 1024, True), (4096, 1, 4, 64, 512, False),
            (4095, 1, 1, 64, 512, False), (4088, 1, 1, 64, 512, True),      # (4095 key heads are launched as 4096)
            (2048, 1, 128, 128, 512, False), (2047, 1, 128, 128, 512, True)]:
        case = n, starts, hk, hv, vd
        assert (size(n, n, starts, hk, hv, 64, vd) >= 0) == fits, case
        r = requests(requests=n, **({} if starts else {'starts_dev': None}))
        s = (hk * 64, 64, hk * 64, 64, hv * vd, vd, hv * vd, vd, hv, hv)
        # (what fits goes on to the next check: an address that is not aligned)
        assert refused(rule(r, s, tokens=n, key_heads=hk, value_heads=hv, key_dim=64, value_dim=vd,
                            q=ctypes.c_void_p(20))) == 'EARG'
        message = _lib.load().localai_hip_last_error().decode()
        assert ('aligned' if fits else 'too many') in message, (case, message)


def norm(strides=(64, 0, 64, 0, 64, 0, 64, 0), **change):
    a = dict(x=ONE, type=0, strides=(ctypes.c_int64 * 8)(*strides), rows=3, heads=1, dim=64, weight=ONE,
             eps=ctypes.c_float(1e-6), residual=None, gate=None, out=ONE, out_type=0, stream=None)
    a.update(change)
    return _lib.load().localai_hip_rms_norm(*a.values())


@pytest.mark.parametrize('change,status', [
    (dict(x=None), 'EARG'), (dict(weight=None), 'EARG'), (dict(out=None), 'EARG'), (dict(type=8), 'ETYPE'),
    (dict(out_type=2), 'ETYPE'), (dict(dim=0), 'EARG'), (dict(dim=(1 << 20) + 1), 'EARG'), (dict(heads=0), 'EARG'),
    (dict(rows=-1), 'EARG'), (dict(rows=1 << 31), 'EARG'), (dict(eps=ctypes.c_float(-1)), 'EARG'),
    (dict(eps=ctypes.c_float(np.nan)), 'EARG'), (dict(out_type=8, dim=48), 'ETYPE'),
    (dict(out_type=8, out=ctypes.c_void_p(17), strides=(64, 0, 64, 0, 64, 0, 68, 0)), 'EARG'),
    (dict(out_type=8, x=ctypes.c_void_p(20), strides=(64, 0, 64, 0, 64, 0, 68, 0)), 'EARG'),
    (dict(out_type=8, strides=(66, 0, 64, 0, 64, 0, 68, 0)), 'EARG'),
    (dict(out_type=8, strides=(64, 0, 64, 0, 64, 0, 66, 0)), 'EARG'),
    (dict(strides=(64, 0, 64, 0, 64, 0, 63, 0)), 'EARG'), (dict(strides=(-64, 0, 64, 0, 64, 0, 64, 0)), 'EARG'),
    (dict(residual=ONE, strides=(64, 0, 32, 0, 64, 0, 64, 0)), 'EARG')])
def test_norm_refusals(change, status):
    assert refused(norm(**change)) == status


def test_packed_requests_are_the_c_structure():
    from localai_amd import delta
    fields = (1, 2, 3, 4, 5, 6)
    assert delta._REQUESTS.pack(*fields) == bytes(_lib.DeltaRequestsArg(*fields))
    assert delta._STRIDES.pack(*range(10)) == bytes((ctypes.c_int64 * 10)(*range(10)))


def test_python_refuses_host_tensors():
    import torch
    from localai_amd import delta, layer
    x = torch.zeros(4, 64)
    with pytest.raises(TypeError, match='device tensor'):
        delta.conv(x, x, x)
    with pytest.raises(TypeError, match='device tensor'):
        delta.rule(x, x, x, x, x, x)
    with pytest.raises(TypeError, match='device tensor'):
        layer.rms_norm(x, x)
