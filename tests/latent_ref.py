"""Plain 64-bit forms of the latent-attention operators, on the CPU."""
from __future__ import annotations

import numpy as np

LATENT, ROPE, WIDTH = 512, 64, 576


def as64(t):
    return t.detach().double().cpu().numpy()


def _attend(q, k, v, seen, scale):
    """One query: q [h, d] over the keys k [m, h or 1, d] and values v [m, h or 1, e] in `seen` [m].

    Returns the output, the LSE, sum p |v| / sum p per element and the largest
    sum |q k| scale of a head's keys (what the scores' rounding goes by).
    """
    h, e = q.shape[0], v.shape[-1]
    k, v = k[seen], v[seen]
    if not len(k):
        return np.zeros((h, e)), np.full(h, -np.inf), np.zeros((h, e)), np.zeros(h)
    # [h, m, d]: products a head; keys that all heads share are one matrix
    k, v = (np.moveaxis(x, 1, 0) if x.shape[1] > 1 else x[None, :, 0] for x in (k, v))
    with np.errstate(invalid="ignore", over="ignore"):
        x = (k @ q[:, :, None])[..., 0] * scale if len(k) > 1 else q @ k[0].T * scale
        top = x.max(1, keepdims=True)
        p = np.exp(x - top)
        total = p.sum(1)
        if len(k) > 1:
            sums = lambda w: (p[:, None, :] @ w)[:, 0]  # noqa: E731
            size = (np.abs(k) @ np.abs(q)[:, :, None])[..., 0].max(1) * scale
        else:
            sums = lambda w: p @ w[0]  # noqa: E731
            size = (np.abs(q) @ np.abs(k[0]).T).max(1) * scale
        out, weight = sums(v) / total[:, None], sums(np.abs(v)) / total[:, None]
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
            length, keys, ok = 0, np.zeros((0, 1, WIDTH)), np.zeros(0, bool)
            n_base = -10 ** 9
        else:
            j = np.arange(length)
            pages = table[b, j // page] if length else np.zeros(0, int)
            ok = (pages >= 0) & (pages < blocks)
            keys = flat[np.where(ok, pages, 0) * page + j % page][:, None]
            n_base = length - n
        for i in range(n):
            seen = ok & (np.arange(len(ok)) <= n_base + i)
            for r, x in zip(res, _attend(q[cu_q[b] + i], keys, keys[..., :LATENT], seen, scale)):
                r[cu_q[b] + i] = x
    return res


def expanded(q, kv, rope, cu_q, cu_k, scale):
    res = _results(int(cu_q[-1]), q.shape[1], 128)
    heads = q.shape[1]
    for b in range(len(cu_q) - 1):
        n, m = int(cu_q[b + 1] - cu_q[b]), int(cu_k[b + 1] - cu_k[b])
        one, r = kv[cu_k[b]:cu_k[b + 1]], rope[cu_k[b]:cu_k[b + 1]]
        k = np.concatenate([one[..., :128], np.broadcast_to(r[:, None], (m, heads, ROPE))], -1)
        for i in range(n):
            seen = np.arange(m) <= m - n + i
            for x, y in zip(res, _attend(q[cu_q[b] + i], k, one[..., 128:], seen, scale)):
                x[cu_q[b] + i] = y
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
