"""CPU restatement (numpy) of the serving-step operators: norm + rotation + cache append, the 4-bit KV cache, attention
over it, sampling.

TEST INFRASTRUCTURE ONLY.  Written from the definitions in include/kore_b200.h.  The append's f32 roundings are part of
its definition (they decide codes) and are made one by one here; attention and sampling are in 64 bits.
"""
from __future__ import annotations

import numpy as np

f32 = np.float32


def normed(x, gamma, eps):
    """x [..., hd] f32 -> (x * inv) * gamma, inv = f32(1 / sqrt(mean(x^2) + eps)) with the mean in f64"""
    if gamma is None:
        return x
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        ms = (x.astype(np.float64) ** 2).mean(-1, keepdims=True)
        inv = (1.0 / np.sqrt(ms + np.float64(f32(eps)))).astype(f32)
        return (x * inv) * np.asarray(gamma, f32)


def rotated(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    with np.errstate(invalid="ignore", over="ignore"):
        return np.concatenate([a * c - b * s, a * s + b * c], -1)


def append(qkv, positions, cos, sin, heads, n_kv, hd, q_gamma=None, k_gamma=None, eps=1e-5):
    """rows [q | k | v] -> rotated q [n, heads, hd], rotated k and v [n, n_kv, hd], all f32"""
    rows = np.asarray(qkv, f32).reshape(len(positions), heads + 2 * n_kv, hd)
    c, s = cos[positions][:, None], sin[positions][:, None]
    q = rotated(normed(rows[:, :heads], q_gamma, eps), c, s)
    k = rotated(normed(rows[:, heads:heads + n_kv], k_gamma, eps), c, s)
    return q, k, rows[:, heads + n_kv:]


def bf16_below(x):
    """largest bfloat16 <= x (finite f32)"""
    i = np.asarray(x, f32).view(np.uint32)
    cut = i & np.uint32(0xFFFF0000)
    return np.where((x < 0) & (cut != i), cut + np.uint32(0x10000), cut).astype(np.uint32).view(f32)


def quantise(x):
    """x [..., hd] f32 -> (code words uint32 [..., ceil(hd / 8)], step words uint32 [...])"""
    x = np.asarray(x, f32)
    hd = x.shape[-1]
    with np.errstate(all="ignore"):
        lo = bf16_below(x.min(-1))
        want = np.maximum((x.max(-1) - lo) / f32(15.0), f32(2.0 ** -100))
        step = -bf16_below(-want)
        ok = np.isfinite(x).all(-1) & np.isfinite(lo) & np.isfinite(step)
        code = np.rint((x - lo[..., None]) * (f32(1.0) / step)[..., None])
    code = np.where(ok[..., None], np.clip(np.nan_to_num(code), 0, 15), 0).astype(np.uint32)
    code = np.concatenate([code, np.zeros((*x.shape[:-1], -hd % 8), np.uint32)], -1).reshape(*x.shape[:-1], -1, 8)
    words = (code << (4 * np.arange(8, dtype=np.uint32))).sum(-1, dtype=np.uint32)
    pair = (step.view(np.uint32) >> np.uint32(16)) | lo.view(np.uint32)
    return words, np.where(ok, pair, np.uint32(0x7FC07FC0)).astype(np.uint32)


def pair_of(steps):
    steps = np.asarray(steps).view(np.uint32)
    return (steps << np.uint32(16)).view(f32), (steps & np.uint32(0xFFFF0000)).view(f32)


def values(words, steps, hd):
    """planes -> the f32 values they stand for (code * step is exact in f32, one rounding in the sum)"""
    words = np.asarray(words).view(np.uint32)
    nib = (words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & np.uint32(15)
    step, lo = pair_of(steps)
    with np.errstate(invalid="ignore"):
        return nib.reshape(*words.shape[:-1], -1)[..., :hd].astype(f32) * step[..., None] + lo[..., None]


def attention(q, words_k, steps_k, words_v, steps_v, lens, scale=0.0):
    """q [batch, t, heads, hd] over planes [batch, n_kv, lmax, ...], in f64 on the values in 64 bits"""
    b, t, heads, hd = q.shape
    n_kv = words_k.shape[1]
    out = np.zeros(q.shape, np.float64)
    scale = float(f32(scale)) if scale else 1.0 / np.sqrt(hd)

    def wide(words, steps):
        nib = (np.asarray(words).view(np.uint32)[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & np.uint32(15)
        step, lo = (a.astype(np.float64)[..., None] for a in pair_of(steps))
        return nib.reshape(*words.shape[:-1], -1)[..., :hd] * step + lo

    for i in range(b):
        n = int(np.clip(lens[i], 0, words_k.shape[2]))
        for h in range(heads):
            g = h // (heads // n_kv)
            for j in range(t):
                m = n - (t - 1 - j)
                if m <= 0:
                    continue
                k, v = wide(words_k[i, g, :m], steps_k[i, g, :m]), wide(words_v[i, g, :m], steps_v[i, g, :m])
                s = k @ q[i, j, h].astype(np.float64) * scale
                p = np.exp(s - s.max())
                out[i, j, h] = (p / p.sum()) @ v
    return out


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob, margin): margin = distance of u to the nearest border of the drawn token, as a share of the total"""
    l = np.asarray(logits, np.float64).copy()
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return 0, np.nan, np.inf
    order = np.argsort(-l, kind="stable")
    if not temperature > 0:
        return int(order[0]), 0.0, np.inf
    with np.errstate(invalid="ignore", divide="ignore"):
        x = np.where(l == top, 0.0, np.where(np.isinf(l) | np.isinf(top), -np.inf, (l - top) / max(np.float64(temperature), 2.0 ** -100)))
    x = x[order]
    n = len(l) if top_k <= 0 else min(int(top_k), len(l))
    if min_p > 0:
        n = min(n, int((x >= np.log(min(float(min_p), 1.0))).sum()))
    w = np.exp(x[:n])
    if top_p < 1.0:
        run = np.cumsum(w)
        n = min(n, 1 + int((run[:-1] < max(float(top_p), 0.0) * run[-1]).sum()))
        w = w[:n]
    by_index = np.argsort(order[:n])
    kept, w = order[:n][by_index], w[by_index]
    cdf = np.cumsum(w)
    u = float(u) if u > 0 else 0.0
    target = min(u, 1.0) * cdf[-1]
    i = int((cdf <= target).sum())
    if i >= n:
        i = int(np.flatnonzero(w > 0)[-1])
    below = cdf[i] - w[i]
    margin = min(abs(target - below) if i else np.inf, abs(cdf[i] - target)) / cdf[-1]
    return int(kept[i]), float(np.log(w[i] / cdf[-1])), margin
