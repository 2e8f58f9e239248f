"""Rotary variants, the 8-bit K/V cache and packed-batch attention in 64 bits
on the host (test infrastructure)."""
import math

import numpy as np

BLOCK = 32


def rope_frequencies(layout, rot, scaling, theta, factor=1.0, low=0.0, high=0.0, orig=0, magnitude=0.0):
    w = []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if scaling == 1:
            f /= factor
        elif scaling == 2:
            t = orig * f / (2 * math.pi)
            if t <= low:
                f /= factor
            elif t < high:
                keep = (t - low) / (high - low)
                f = keep * f + (1 - keep) * f / factor
        elif scaling == 3:
            a, b = (rot * math.log(orig / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (high, low))
            a, b = max(0, math.floor(a)), min(rot - 1, math.ceil(b))
            slow = min(1.0, max(0.0, (i - a) / (b - a if b > a else 0.001)))
            f = slow * f / factor + (1 - slow) * f
        w.append(f)
    if magnitude == 0.0:
        magnitude = 0.1 * math.log(factor) + 1.0 if scaling == 3 and factor > 1 else 1.0
    return np.array(w), magnitude


def rope(x, pos, layout, rot, w, magnitude):
    """x [rows, heads, hd] float64."""
    y = x.copy()
    a = pos.astype(np.float64)[:, None] * w
    c, s = np.cos(a)[:, None] * magnitude, np.sin(a)[:, None] * magnitude
    j = slice(0, rot // 2) if layout == 0 else slice(0, rot, 2)
    k = slice(rot // 2, rot) if layout == 0 else slice(1, rot, 2)
    y[..., j] = x[..., j] * c - x[..., k] * s
    y[..., k] = x[..., k] * c + x[..., j] * s
    return y


def quantise(x):
    """x [..., n % 32 == 0] float32 -> int8 codes and f16 steps of each 32."""
    b = np.where(np.isnan(x), np.float32(0), x).reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    top = np.abs(b).max(-1)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        d = np.minimum(top / np.float32(127), np.float32(65504)).astype(np.float16)
        q = np.rint(b.astype(np.float64) / d.astype(np.float64)[..., None])
    q = np.where(d[..., None] > 0, np.clip(q, -127, 127), 0).astype(np.int8)
    return q.reshape(x.shape), d


def values(q, d):
    return (q.reshape(*d.shape, BLOCK).astype(np.float64) * d.astype(np.float64)[..., None]).reshape(q.shape)


def ancestors(parent):
    """[n, n] bool: whether draft i sees draft j; a parent that is not an earlier draft counts as none."""
    n = len(parent)
    sees = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while True:
            sees[i, j] = True
            up = int(parent[j])
            if up < 0 or up >= j:
                break
            j = up
    return sees


def attend(q, K, V, sees, hd):
    """One kv head: q [n, G, hd], K, V [keys, hd] float64, sees [n, keys].  Returns out, and the largest
    sum |q_i k_i| / sqrt(hd) and |score| of a seen key."""
    s = np.einsum("ngd,kd->ngk", q, K) / math.sqrt(hd)
    mag = np.einsum("ngd,kd->ngk", np.abs(q), np.abs(K)) / math.sqrt(hd)
    s = np.where(sees[:, None], s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    out = np.einsum("ngk,kd->ngd", p, V) / p.sum(-1, keepdims=True)
    return out, float(np.where(sees[:, None], mag, 0).max()), float(np.abs(np.where(sees[:, None], s, 0)).max())
