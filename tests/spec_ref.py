"""Plain 64-bit forms of the speculative-decoding operators, for their tests.
NumPy on the host; BF16 tensors come in as their values."""
from __future__ import annotations

import math

import numpy as np

MASK64 = (1 << 64) - 1


def as64(t):
    return t.detach().cpu().double().numpy()


def ancestors(parents):
    """[n, n] bool: node i sees itself and its ancestors."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def pack_bits(seen, words):
    """[rows, n] bool -> [rows, words] int64 masks."""
    out = np.zeros((seen.shape[0], words), np.uint64)
    for i, j in zip(*np.nonzero(seen)):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def tree_attention(q, k, v, cu, lens, table, seens, block_size):
    """(out, lse, weight, size) in 64 bits; seens[b] [n, n] bool. weight
    [rows, qh, 128] is sum p |v| and size [rows, qh] the largest sum |q k| /
    sqrt(dim) of a seen key: what rounding errors scale with. Rows behind
    cu[-1] are NaN (nobody writes them). Keys nobody sees are left out of the
    sums, as the formula has them."""
    rows, qh, dim = q.shape
    blocks, _, kvh, _ = k.shape
    group = qh // kvh
    out, lse = np.full((rows, qh, dim), np.nan), np.full((rows, qh), np.nan)
    weight, size = np.zeros((rows, qh, dim)), np.zeros((rows, qh))
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        ctx = lens[b] - n
        fits = ctx >= 0 and lens[b] <= len(table[b]) * block_size
        for i in range(n):
            r = cu[b] + i
            keys = [*range(ctx), *(ctx + t for t in range(n) if seens[b][i, t])] if fits else []
            keys = [x for x in keys if 0 <= table[b][x // block_size] < blocks]
            if not keys:
                out[r], lse[r] = 0.0, -math.inf
                continue
            page = np.array([table[b][x // block_size] for x in keys], int)
            slot = np.array([x % block_size for x in keys], int)
            kk, vv = k[page, slot], v[page, slot]  # [keys, kvh, dim]
            with np.errstate(all="ignore"):
                for g in range(kvh):
                    h = slice(g * group, (g + 1) * group)
                    x = q[r, h] @ kk[:, g].T / math.sqrt(dim)  # [group, keys]
                    size[r, h] = (np.abs(q[r, h]) @ np.abs(kk[:, g]).T / math.sqrt(dim)).max(1)
                    m = x.max(1, keepdims=True)
                    e = np.exp(x - m)
                    lse[r, h] = m[:, 0] + np.log(e.sum(1))
                    e = e / e.sum(1, keepdims=True)
                    out[r, h] = (e[:, :, None] * vv[None, :, g]).sum(1)
                    weight[r, h] = (e[:, :, None] * np.abs(vv[None, :, g])).sum(1)
    return out, lse, weight, size


def splitmix(x):
    x = (x + 0x9e3779b97f4a7c15) & MASK64
    x = ((x ^ (x >> 30)) * 0xbf58476d1ce4e5b9) & MASK64
    x = ((x ^ (x >> 27)) * 0x94d049bb133111eb) & MASK64
    return x ^ (x >> 31)


def gumbel(seed, vocab):
    """The sampler's noise of every token, in 64 bits (wrapping 64-bit products in NumPy)."""
    with np.errstate(over="ignore"):
        x = np.uint64(seed & MASK64) ^ (np.arange(vocab, dtype=np.uint64) * np.uint64(0xd2b74407b1ce6e93))
        x = x + np.uint64(0x9e3779b97f4a7c15)
        x = (x ^ (x >> np.uint64(30))) * np.uint64(0xbf58476d1ce4e5b9)
        x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94d049bb133111eb)
        x = x ^ (x >> np.uint64(31))
    return -np.log(-np.log(((x >> np.uint64(41)).astype(np.float64) + 0.5) / 2.0 ** 23))


def softmax(l, temperature):
    l = np.where(np.isnan(l), -np.inf, l)
    m = l.max()
    if m == -np.inf:
        return np.zeros_like(l)
    if m == np.inf:
        e = (l == np.inf).astype(np.float64)
    else:
        e = np.exp((l - m) / temperature)
    return e / e.sum()


def argmax(l):
    """The sampler's choice at temperature 0: NaN is never it, 0 if there is no other."""
    l = np.where(np.isnan(l), -np.inf, l)
    return int(np.argmax(l))


def verify(logits, draft, tokens, parents, uniforms, seeds, temps, cu, max_q, eps=3e-5):
    """(out_tokens, path, counts, accept_prob, bound, margin, drawable): bound is
    how far accept_prob may be off where every probability is eps off (relative),
    and margin how near the nearest decision was to falling the other way (so that
    the tests know that their inputs are not borderline).

    drawable[b]: the next tokens that such probabilities may draw where something
    was rejected. What is left of P, p = max(P - Q, 0) / sum, is off by e = eps
    (P + Q) / sum and more with each level, so a token's score lies between
    log(p - e) and log(p + e) plus its noise, and may be the highest where its
    upper end reaches the best lower end. That is one token, unless P and Q agree
    so far that their difference is below the rounding of either: where they put
    all but 1e-28 on the same few tokens, 32-bit differences of those tokens are
    rounding (1e-8), and outweigh what the others have left."""
    rows, vocab = logits.shape
    batch = len(temps)
    out, path = np.full((batch, max_q), -1), np.full((batch, max_q), -1)
    counts, prob, bound = np.zeros(batch, int), np.zeros(rows), np.zeros(rows)
    margin, drawable = math.inf, [set() for _ in range(batch)]
    for b in range(batch):
        n, first = cu[b + 1] - cu[b], cu[b]
        if n <= 0:
            continue
        winner, left = [-1] * n, [None] * n
        for node in range(n):
            r = first + node
            kids = [i for i in range(node + 1, n) if parents[first + i] == node]
            if not temps[b] > 0:
                best = argmax(logits[r])
                for i in kids:
                    if winner[node] < 0 and tokens[first + i] == best:
                        winner[node], prob[first + i] = i, 1.0
                continue
            if not kids:
                continue
            p = softmax(logits[r], temps[b])
            q = softmax(draft[r], temps[b]) if draft is not None else None
            ep, eq = eps * p, eps * q if q is not None else None
            for i in kids:
                t = tokens[first + i]
                inside = 0 <= t < vocab
                have = p[t] if inside else 0.0
                asked = (q[t] if inside else 0.0) if q is not None else 1.0
                a = 0.0 if have <= 0 else (min(1.0, have / asked) if asked > 0 else 1.0)
                prob[first + i] = a
                if have > 0 and asked > 0:
                    off = ep[t] / asked + (have * eq[t] / asked ** 2 if q is not None else 0.0)
                    bound[first + i] = off if have / asked < 1 + off else 0.0
                u = uniforms[first + i]
                if 0 < a < 1:
                    margin = min(margin, abs(u - a))
                if u < a:
                    winner[node] = i
                    break
                if q is None:
                    rest = p.copy()
                    if inside:
                        rest[t] = 0
                    erest = ep
                else:
                    rest, erest = np.maximum(p - q, 0), ep + eq
                    q, eq = q.copy(), eq.copy()
                    if inside:
                        q[t] = eq[t] = 0
                    if q.sum() > 0:
                        eq = eq / q.sum() + q * eq.sum() / q.sum() ** 2
                        q = q / q.sum()
                total = rest.sum()
                if total > 0:
                    p, ep = rest / total, erest / total + rest * erest.sum() / total ** 2
                left[node] = p, ep
        at, seq = 0, [0]
        while winner[at] >= 0:
            at = winner[at]
            seq.append(at)
        counts[b] = len(seq)
        path[b, :len(seq)] = seq
        out[b, :len(seq) - 1] = [tokens[first + i] for i in seq[1:]]
        r = first + at
        if not temps[b] > 0:
            out[b, len(seq) - 1] = argmax(logits[r])
            continue
        with np.errstate(divide="ignore"):
            noise = gumbel(int(seeds[r]), vocab)
            if left[at] is not None:
                (p, ep), score = left[at], np.log(left[at][0]) + noise
                drawable[b] = set(np.nonzero(np.log(p + ep) + noise >= (np.log(np.maximum(p - ep, 0)) + noise).max())[0])
            else:
                score = np.where(np.isnan(logits[r]), -np.inf, logits[r]) / temps[b] + noise
        out[b, len(seq) - 1] = int(np.argmax(score))
        top = np.sort(score)[-2:]
        if len(top) == 2 and np.isfinite(top).all():
            margin = min(margin, top[1] - top[0])
    return out, path, counts, prob, bound, margin, drawable


def drawn_from(logits, draft, tokens, parents, seeds, temps, cu, path, counts, eps=3e-5):
    """For each sequence the next tokens that may be drawn behind its path where every probability is eps off
    (relative), or None where nothing was rejected there (then verify's token is the one). As verify's `drawable`, but a
    factor that all tokens share is no error of a score: the sum that P is divided by counts only where Q is taken from
    P after it."""
    out = []
    for b in range(len(temps)):
        n, first, last = cu[b + 1] - cu[b], cu[b], path[b][counts[b] - 1]
        kids = [i for i in range(last + 1, n) if parents[first + i] == last] if counts[b] else []
        if not kids or not temps[b] > 0:
            out.append(None)
            continue
        p, vocab = softmax(logits[first + last], temps[b]), logits.shape[1]
        q = softmax(draft[first + last], temps[b]) if draft is not None else None
        ep, shared = eps * p, 0.0
        eq = eps * q if q is not None else None
        for i in kids:
            t, inside = tokens[first + i], 0 <= tokens[first + i] < vocab
            if q is None:
                rest = p.copy()
                if inside:
                    rest[t] = 0
                erest = np.where(rest > 0, ep, 0)
            else:
                rest, erest, shared = np.maximum(p - q, 0), ep + shared * p + eq, 0.0
                q, eq = q.copy(), eq.copy()
                if inside:
                    q[t] = eq[t] = 0
                if q.sum() > 0:
                    eq, q = eq / q.sum() + q * eq.sum() / q.sum() ** 2, q / q.sum()
            total = rest.sum()
            if total > 0:
                p, ep, shared = rest / total, erest / total, shared + erest.sum() / total
        with np.errstate(divide="ignore"):
            noise = gumbel(int(seeds[first + last]), vocab)
            low, high = np.log(np.maximum(p - ep, 0)) + noise, np.log(p + ep) + noise
        # a score of log 0 is nobody's
        out.append({int(t) for t in np.nonzero((high >= low.max()) & (high > -math.inf))[0]})
    return out
