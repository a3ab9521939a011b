"""Plain implementations, in 64 bits and on the CPU, of the serving operators: a paged
cache's tables, rotary positions, attention of drafted tokens and logits' adjustment."""
from __future__ import annotations

import math

import numpy as np

# Half a unit in the last place, relative, of each type's rounding.
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}  # below the normal range


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def ceil_div(a, b):
    return -(-a // b)


def grow(table, lens, new, free, count, block, tokens):
    """(table, slots, positions, cu, after, left) by walking the requests and their tokens."""
    table = table.copy()
    slots, positions = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int64)
    cu, after = [0], []
    wanted = used = 0
    count = max(0, min(count, len(free)))
    for b, (n, a) in enumerate(zip(lens, new)):
        n, a = max(0, int(n)), max(0, int(a))
        had, need = ceil_div(n, block), ceil_div(n + a, block)
        fits = need <= table.shape[1]
        want = need - had if fits else 0
        ok = fits and (want == 0 or wanted + want <= count) and (a == 0 or cu[-1] + a <= tokens)
        if ok:
            for j in range(want):
                table[b, had + j] = free[count - 1 - (wanted + j)]
            if want:
                used = wanted + want
        for i in range(a):
            t = cu[-1] + i
            if t < tokens:
                positions[t] = n + i
                if ok and table[b, (n + i) // block] >= 0:
                    slots[t] = int(table[b, (n + i) // block]) * block + (n + i) % block
        wanted += want
        cu.append(cu[-1] + a)
        after.append(n + a if ok else n)
    return table, slots, positions, np.array(cu), np.array(after, np.int64), count - used


def release(table, lens, keep, free, count, block):
    """(free, left)"""
    free, top = free.copy(), count
    for b, (n, k) in enumerate(zip(lens, keep)):
        last = min(ceil_div(max(0, int(n)), block), table.shape[1])
        for j in range(ceil_div(max(0, int(k)), block), last):
            if top < len(free):
                free[top] = table[b, j]
            top += 1
    return free, min(top, len(free))


def rope(x, cos_sin, positions, axis, paired, inverse):
    """(y, size): the turned x [T, heads, dim] and, for each element, the sum of the absolute
    values of its terms."""
    y, size = x.copy(), np.abs(x)
    pairs = cos_sin.shape[1] // 2
    pos = positions.reshape(-1, x.shape[0])
    for i in range(pairs):
        p = pos[axis[i]]
        good = (p >= 0) & (p < cos_sin.shape[0])
        row = cos_sin[np.where(good, p, 0)]
        c, s = row[:, i], row[:, pairs + i] * (-1 if inverse else 1)
        c, s = np.where(good, c, np.nan)[:, None], np.where(good, s, np.nan)[:, None]
        ia, ib = (2 * i, 2 * i + 1) if paired else (i, pairs + i)
        a, b = x[:, :, ia], x[:, :, ib]
        y[:, :, ia], y[:, :, ib] = a * c - b * s, b * c + a * s
        size[:, :, ia], size[:, :, ib] = abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)
    return y, size


def attention(q, k_cache, v_cache, table, cu, kv_lens, mask, scale, weight_ulp):
    """(o, lse, o_tol, lse_tol) for f64 q [T, H, D], caches [NB, block, HK, D]. The tolerances
    follow from the arithmetic: scores are dot products of D terms in f32, weights and their sum
    f32 with a weight rounded to `weight_ulp` for the product with the values."""
    T, H, D = q.shape
    nb, block, hk, _ = k_cache.shape
    group = H // hk
    o, lse = np.zeros((T, H, D)), np.full((T, H), -np.inf)
    o_tol, lse_tol = np.zeros((T, H)), np.zeros((T, H))
    eps = 2.0 ** -24
    for b in range(len(kv_lens)):
        n, kv = int(cu[b + 1] - cu[b]), max(0, int(kv_lens[b]))
        prefix = kv - n
        pos = np.arange(min(kv, table.shape[1] * block))
        blk = table[b, pos // block]
        good = (blk >= 0) & (blk < nb)
        for i in range(n):
            t = int(cu[b]) + i
            j = pos - prefix
            if mask is None:
                see = j <= i
            else:
                word = mask[t, np.clip(j >> 5, 0, mask.shape[1] - 1)].astype(np.int64)
                see = (j < 0) | ((j >> 5 < mask.shape[1]) & ((word >> (j & 31)) & 1 == 1))
            at = pos[good & see]
            if len(at) == 0:
                continue
            rows, off = table[b, at // block], at % block
            for h in range(H):
                k, v = k_cache[rows, off, h // group], v_cache[rows, off, h // group]
                s = k @ q[t, h] * scale
                m = s.max()
                p = np.exp(s - m)
                o[t, h] = p @ v / p.sum()
                lse[t, h] = m + math.log(p.sum())
                size = np.max(np.abs(k) @ np.abs(q[t, h])) * abs(scale)
                ds = (D + 4) * eps * size            # a score's error
                # a weight's relative error: both of its scores', the argument's rounding,
                # the exponential's own (2^-21), and the sums' (one rounding a term)
                rho = 2 * ds + 4 * eps * (size + abs(m)) + 2.0 ** -21 + (len(at) + 8) * eps
                # f16 weights below 2^-14 are rounded on a fixed grid of 2^-24
                grid = len(at) * 2.0 ** -25 if weight_ulp == HALF_ULP["f16"] else 0.0
                o_tol[t, h] = 2 * (weight_ulp + rho + grid) * np.max(np.abs(v))
                lse_tol[t, h] = rho + 4 * eps * abs(lse[t, h]) + 2 * eps
    return o, lse, o_tol, lse_tol


def logits(x, ids, cu, prompt, rep, pre, fre, bias_ids, bias_values, bias_cu, allowed):
    """(y, size): the adjusted logits and the sum of the absolute values of each one's terms."""
    y, size = x.copy(), np.abs(x)
    V = x.shape[1]
    for r in range(x.shape[0]):
        history = ids[max(0, cu[r]):cu[r + 1]]
        inside = (history >= 0) & (history < V)
        for v in np.unique(history[inside]):
            n = int(np.sum(history[prompt[r]:] == v))
            if rep is not None:
                y[r, v] = y[r, v] / rep[r] if y[r, v] > 0 else y[r, v] * rep[r]
                size[r, v] = max(size[r, v], abs(y[r, v]))
            if n:
                f, p = (0.0 if z is None else z[r] for z in (fre, pre))
                y[r, v] -= f * n + p
                size[r, v] += abs(f * n) + abs(p)
        if bias_ids is not None:
            for v, w in dict(zip(bias_ids[bias_cu[r]:bias_cu[r + 1]],
                                 bias_values[bias_cu[r]:bias_cu[r + 1]])).items():
                if 0 <= v < V:
                    y[r, v] += w
                    size[r, v] += abs(w)
        if allowed is not None:
            bits = (allowed[r].astype(np.int64)[:, None] >> np.arange(32)) & 1
            y[r, bits.reshape(-1)[:V] == 0] = -np.inf
    return y, size
