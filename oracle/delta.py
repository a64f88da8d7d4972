"""Oracle of the linear-attention layers' operators. TEST INFRASTRUCTURE ONLY.

rule restates the gated delta rule in fp64, token after token, as
oracle.attention.delta_net_step_f64 does for one token (engine/qwen35.py:248-252),
with the norms of q and k, the gates' projections and the heads' order ahead of
it. conv is the causal convolution of one request's rows, rms_norm the norm of
engine/model.py:82 with the residual, the gate, and Q8_0 blocks.

Pins (tests/test_delta.py): rule against delta_net_step_f64 token by token, the
gates against SciPy's softplus and logistic forms, both head orders; conv against
numpy.convolve, and its state as the rows before; rms_norm against unit root mean
squares, Q8_0 blocks against oracle.quant.dequantize.
"""
from __future__ import annotations

import numpy as np

from .attention import delta_net_step_f64


def gates(decay, beta, a=None, dt_bias=None):
    decay, beta = np.asarray(decay, np.float64), np.asarray(beta, np.float64)
    if a is None:
        return decay, beta
    return (np.asarray(a, np.float64) * np.logaddexp(0, decay + np.asarray(dt_bias, np.float64)),
            1 / (1 + np.exp(-beta)))


def rule(state, q, k, v, decay, beta, a=None, dt_bias=None, order='grouped', norm_eps=1e-6, scale=None, sizes=None):
    """One request: state [value heads, key dim, value dim]; q, k [tokens, key heads, key dim]; v [tokens, value
    heads, value dim]; decay, beta [tokens, value heads]. Returns (out, state after); sizes [tokens, value heads] takes the larger norm of
    each head's state after the decay and after the update."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    hk, hv = q.shape[1], v.shape[1]
    key = np.arange(hv) // (hv // hk) if order == 'grouped' else np.arange(hv) % hk
    if norm_eps is not None:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + norm_eps) for x in (q, k))
    q = (q * (q.shape[-1] ** -0.5 if scale is None else scale))[:, key]
    k = k[:, key]
    g, b = gates(decay, beta, a, dt_bias)
    S, out = np.asarray(state, np.float64), np.zeros(v.shape)
    for t in range(len(v)):
        decayed = np.linalg.norm(S, axis=(1, 2)) * np.exp(g[t])
        S, out[t] = delta_net_step_f64(S, q[t], k[t], v[t], g[t], b[t])
        if sizes is not None:
            sizes[t] = np.maximum(decayed, np.linalg.norm(S, axis=(1, 2)))
    return out, S


def conv(state, x, weight, bias=None, silu=True):
    """One request: state [width - 1, channels], x [tokens, channels]. Returns (out, state after, sum of |terms|)."""
    width = np.asarray(weight).shape[1]
    line = np.concatenate([np.asarray(state, np.float64), np.asarray(x, np.float64)])
    w, n = np.asarray(weight, np.float64), len(x)
    terms = np.stack([w[:, j] * line[j:j + n] for j in range(width)])
    b = np.zeros(line.shape[1]) if bias is None else np.asarray(bias, np.float64)
    y = terms.sum(0) + b
    size = np.abs(terms).sum(0) + np.abs(b)
    return y / (1 + np.exp(-y)) if silu else y, line[n:], size


def rms_norm(x, weight, eps=1e-6, residual=None, gate=None):
    """Returns (y, x + residual)."""
    h = np.asarray(x, np.float64)
    if residual is not None:
        h = h + np.asarray(residual, np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if gate is not None:
        z = np.asarray(gate, np.float64)
        y = y * z / (1 + np.exp(-z))
    return y, h


def q8_0(y):
    """(scales as fp16, quants) of rows of whole blocks of 32."""
    blocks = np.asarray(y, np.float64).reshape(*np.shape(y)[:-1], -1, 32)
    d = (np.abs(blocks).max(-1) / 127).astype(np.float16)
    q = np.rint(blocks / np.where(d == 0, 1, d.astype(np.float64))[..., None])
    return d, np.clip(q, -127, 127).astype(np.int8)
