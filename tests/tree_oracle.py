"""Plain float64 implementations of the ops of a step of drafted tokens (test infrastructure), and the bounds their results are held to.

u is the largest relative error of one rounding (half a step): fp32 2^-24, bfloat16 2^-8."""
from __future__ import annotations

import math

import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -8
UNIT = {"f32": U32, "bf16": U16}


def round8(n):
    return (n + 7) // 8 * 8


def frequencies(dims, base, scaling="plain", factor=1.0, orig=0.0, low=0.0, high=1.0):
    i = np.arange(dims // 2)
    if scaling == "base":
        base = base * factor ** (dims / (dims - 2))
    f = np.array([base ** (-2.0 * k / dims) for k in i])
    if scaling == "linear":
        return f / factor
    if scaling == "ramp":
        w = np.clip((orig * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * (w + (1 - w) / factor)
    return f


def rotate(x, cos, sin, half):
    """The first 2 * len(cos) elements of x."""
    x, n = x.copy(), len(cos)
    if half:
        a, b = x[:n].copy(), x[n:2 * n].copy()
        x[:n], x[n:2 * n] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[0:2 * n:2].copy(), x[1:2 * n:2].copy()
        x[0:2 * n:2], x[1:2 * n:2] = a * cos - b * sin, b * cos + a * sin
    return x


def norm(x, w, eps):
    return x if w is None else x / math.sqrt(np.mean(x * x) + eps) * w


def tree_mask(parents):
    """seen[i][j]: node j is node i or one of its ancestors."""
    n = len(parents)
    m = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def bits(m, words):
    out = np.zeros((len(m), words), np.uint32)
    for j in range(m.shape[1]):
        out[:, j // 32] |= m[:, j].astype(np.uint32) << np.uint32(j % 32)
    return out


def attend(q, k, v, seen, scale):
    """Outputs of one head [n][dv] for queries q [n][d] over keys k, values v under the mask seen [n][keys], and what bounds their
    error: sum p |v| per output, and per row the size of the terms of its largest score."""
    n, dv = len(q), v.shape[1]
    out, weight, size = np.zeros((n, dv)), np.zeros((n, dv)), np.zeros(n)
    for i in range(n):
        at = np.flatnonzero(seen[i])
        if len(at) == 0:
            continue
        s = scale * (k[at] @ q[i])
        size[i] = scale * (np.abs(k[at]) @ np.abs(q[i])).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i], weight[i] = p @ v[at], p @ np.abs(v[at])
    return out, weight, size


def attention_bound(out, weight, size, d, keys, dtype):
    """A score is a sum of d products in fp32, in any order: off by (d + 3) u of its terms' size.  That moves every weight by a factor
    of 1 +- 2 delta (numerator and denominator); a weight's exponential adds 2^-21, running maxima that move add 4 u a tile, sums of
    `keys` terms in fp32 keys * u.  bfloat16: a weight is rounded before its product, and the result once."""
    delta = (d + 3) * U32 * size[:, None]
    f = 2 * delta + 2.0 ** -20 + (keys / 16 + keys + 40) * U32
    bound = weight * f
    if dtype == "bf16":
        bound = bound + U16 * weight + U16 * (np.abs(out) + U16 * weight)
    return bound + U32 * np.abs(out) + 1e-37
