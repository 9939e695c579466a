"""Plain 64-bit forms of the latent-attention operators, on the CPU."""
from __future__ import annotations

import numpy as np

LATENT, ROPE, WIDTH = 512, 64, 576


def as64(t):
    return t.detach().double().cpu().numpy()


def _attend(q, k, v, seen, scale):
    """One query of h heads: q [h, d] over the keys k [m, d] and values v [m, e] in `seen` [m].

    Returns the output, the LSE, sum p |v| / sum p per element and the largest
    sum |q k| scale of a head's keys (what the scores' rounding goes by).
    """
    h, e = q.shape[0], v.shape[-1]
    k, v = k[seen], v[seen]
    if not len(k):
        return np.zeros((h, e)), np.full(h, -np.inf), np.zeros((h, e)), np.zeros(h)
    with np.errstate(invalid="ignore", over="ignore"):
        x = q @ k.T * scale
        top = x.max(1, keepdims=True)
        p = np.exp(x - top)
        total = p.sum(1)
        out, weight = p @ v / total[:, None], p @ np.abs(v) / total[:, None]
        size = (np.abs(q) @ np.abs(k).T).max(1) * scale
        lse = top[:, 0] + np.log(total)
    return out, lse, weight, size


def _results(rows, heads, width):
    return [np.full((rows, heads, width), np.nan), np.full((rows, heads), np.nan),
            np.zeros((rows, heads, width)), np.zeros((rows, heads))]


def absorbed(q, cache, cu_q, kv_lens, table, scale):
    """(out, lse, weight, size) for the rows of cu_q; cache [blocks, page, 576], all 64-bit."""
    blocks, page = cache.shape[:2]
    res = _results(int(cu_q[-1]), q.shape[1], LATENT)
    flat = cache.reshape(-1, WIDTH)
    for b, length in enumerate(kv_lens):
        n = int(cu_q[b + 1] - cu_q[b])
        if length < 0 or length > table.shape[1] * page:
            length, keys, ok = 0, np.zeros((0, WIDTH)), np.zeros(0, bool)
            n_base = -10 ** 9
        else:
            j = np.arange(length)
            pages = table[b, j // page] if length else np.zeros(0, int)
            ok = (pages >= 0) & (pages < blocks)
            keys = flat[np.where(ok, pages, 0) * page + j % page]
            n_base = length - n
        for i in range(n):
            seen = ok & (np.arange(len(ok)) <= n_base + i)
            for r, x in zip(res, _attend(q[cu_q[b] + i], keys, keys[..., :LATENT], seen, scale)):
                r[cu_q[b] + i] = x
    return res


def expanded(q, kv, rope, cu_q, cu_k, scale):
    """As absorbed; kv [keys, heads, 256], rope [keys, 64]. A key that is not finite counts where it is seen only."""
    res = _results(int(cu_q[-1]), q.shape[1], 128)
    for b in range(len(cu_q) - 1):
        n, m = int(cu_q[b + 1] - cu_q[b]), int(cu_k[b + 1] - cu_k[b])
        seen = np.arange(m)[None, :] <= m - n + np.arange(n)[:, None]
        some = seen.any(1)
        for h in range(q.shape[1]):
            one = kv[cu_k[b]:cu_k[b + 1], h]
            k, v = np.concatenate([one[:, :128], rope[cu_k[b]:cu_k[b + 1]]], 1), one[:, 128:]
            x = q[cu_q[b]:cu_q[b + 1], h]
            fine = np.isfinite(v)
            with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                s = np.where(seen, x @ k.T * scale, -np.inf)
                top = np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None]
                p = np.where(seen, np.exp(s - top), 0.0)
                total = p.sum(1)
                inv = np.where(some, 1.0 / total, 0.0)[:, None]
                out, weight = p @ np.where(fine, v, 0.0) * inv, p @ np.where(fine, np.abs(v), 0.0) * inv
                for key in np.nonzero(~fine.all(1))[0]:
                    rows = seen[:, key]
                    out[rows] += np.where(fine[key], 0.0, p[rows, key, None] * v[key])
                size = np.where(seen, np.abs(x) @ np.abs(k).T * scale, 0.0).max(1, initial=0.0)
                lse = np.where(some, top[:, 0] + np.log(total), -np.inf)
            for r, y in zip(res, (out, lse, weight, size)):
                r[cu_q[b]:cu_q[b + 1], h] = y
    return res


def rotate(x, cos, sin, interleaved):
    """x [..., 64], cos and sin [..., 32]."""
    out = np.empty_like(x)
    if interleaved:
        a, z = x[..., 0::2], x[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * cos - z * sin, z * cos + a * sin
    else:
        a, z = x[..., :32], x[..., 32:]
        out[..., :32], out[..., 32:] = a * cos - z * sin, z * cos + a * sin
    return out


def normalise(x, weight, eps):
    return x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * weight
