"""Oracle of the paged key / value cache. TEST INFRASTRUCTURE ONLY.

Tables keeps the bookkeeping as Python lists, page by page and token by token.
norm_rope restates the per-head norm (engine/model.py:82 on one head) and the
rotation of pairs (engine/model.py:205-210) or halves in fp64. attention runs
oracle.attention's softmax over one request's positions at a time, in fp64,
and returns beside each output the sum of p |v| and the largest sum of |q k|,
from which the tests bound fp32 errors.

Pins (tests/test_paged.py): a page's positions against arange, shrink as the
inverse of extend; the rotation against complex multiplication; attention of
one token against oracle.attention.gqa_decode.
"""
from __future__ import annotations

import math

import numpy as np

from .attention import sigmoid


class Tables:
    def __init__(self, lengths, table, free, used, page):
        self.lengths, self.table = [int(x) for x in lengths], [list(map(int, row)) for row in table]
        self.free, self.used, self.page = [int(x) for x in free], int(used), page

    def extend(self, new, tokens):
        """(status, starts, slots, positions); the tables move on if status is 0."""
        page = self.page
        need = [-(-(o + n) // page) - -(-o // page) for o, n in zip(self.lengths, new)]
        status = 0
        if any(o < 0 or n < 0 or -(-(o + n) // page) > len(row)
               for o, n, row in zip(self.lengths, new, self.table)):
            status |= 2
        else:
            status |= (self.used + sum(need) > len(self.free)) + 4 * (sum(new) > tokens)
        starts, slots, positions = [0] * (len(new) + 1), [], []
        if status == 0:
            for b, (row, n) in enumerate(zip(self.table, new)):
                for _ in range(n):
                    p = self.lengths[b]
                    if p % page == 0:
                        row[p // page] = self.free[self.used]
                        self.used += 1
                    slots.append(row[p // page] * page + p % page)
                    positions.append(p)
                    self.lengths[b] += 1
                starts[b + 1] = len(slots)
        rest = [-1] * (tokens - len(slots))
        return status, starts, slots + rest, positions + rest

    def shrink(self, keep):
        back = []
        for b, (row, k) in enumerate(zip(self.table, keep)):
            end = min(k, self.lengths[b])
            for j in range(-(-end // self.page), -(-self.lengths[b] // self.page)):
                back.append(row[j])
                row[j] = -1
            self.lengths[b] = end
        self.used -= len(back)
        self.free[self.used:self.used + len(back)] = back


def norm_rope(x, position, freq, weight, eps, rope):
    """x [heads, head_dim] of one token."""
    y = np.array(x, dtype=np.float64)
    if weight is not None:
        y = y / np.sqrt(np.mean(y * y, axis=-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    n = len(freq)
    angle = float(position) * np.asarray(freq, np.float64)
    c, s = np.cos(angle), np.sin(angle)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rope == 'pairs' else (slice(0, n), slice(n, 2 * n))
    a, b = y[:, first].copy(), y[:, second].copy()
    y[:, first], y[:, second] = a * c - b * s, a * s + b * c
    return y


def attention(q, keys, values, count, scale, window=0, gate=None):
    """q [tokens, heads, hd] at the last `count` of keys' positions; keys, values
    [positions, kv heads, hd]. Returns (out, weight = sum p |v|, spread =
    largest scale * sum |q k|, per token and head)."""
    q = np.asarray(q, np.float64)
    keys, values = np.asarray(keys, np.float64), np.asarray(values, np.float64)
    length, nkv, hd = keys.shape
    heads = q.shape[1]
    out, weight, spread = np.zeros_like(q), np.zeros_like(q), np.zeros(q.shape[:2])
    for i in range(count):
        p = length - count + i
        if p < 0:
            continue
        lo = max(0, p + 1 - window) if window else 0
        for h in range(heads):
            k, v = keys[lo:p + 1, h * nkv // heads], values[lo:p + 1, h * nkv // heads]
            score = scale * (k @ q[i, h])
            w = np.exp(score - score.max())
            w /= w.sum()
            out[i, h], weight[i, h] = w @ v, w @ np.abs(v)
            spread[i, h] = abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()
    if gate is not None:
        g = sigmoid(gate)
        out, weight = out * g, weight * g
    return out, weight, spread


def default_scale(hd):
    return 1.0 / math.sqrt(hd)
