"""The 8-bit key/value cache in 64 bits on the CPU (numpy), from its definition: what the GPU tests compare with.

A cache is a dict: k, v float64 (pages, H, 64, D), the values that the stored bytes stand for in units of their scale; k_scale, v_scale float64 (pages, H);
desc int64 (pages, H, 64) or None.
"""
import numpy as np

PAGE = 64


def e4m3(x):
    """x rounded to the numbers of e4m3: sign, 4 significant bits, steps of 2**-9 at the bottom, 448 at most, nearest even; NaN for what is not finite."""
    x = np.asarray(x, np.float64)
    fin = np.isfinite(x)
    y = np.where(fin, x, 0.0)
    _, e = np.frexp(y)
    step = np.exp2(np.maximum(e - 4, -9).astype(np.float64))
    r = np.clip(np.round(y / step) * step, -448.0, 448.0)   # numpy rounds halves to even
    return np.where(fin, r, np.nan)


def exponent(x):
    """The smallest e with max |finite x| <= 448 * 2**e, from -32 to 31."""
    a = np.abs(x[np.isfinite(x)])
    if a.size == 0 or a.max() == 0:
        return -32
    e = -32
    while e < 31 and a.max() > 448.0 * 2.0 ** e:
        e += 1
    return e


def descriptors(in_span, span_id, is_prefix):
    in_span, is_prefix = np.asarray(in_span, bool), np.asarray(is_prefix, bool)
    span_id = np.asarray(span_id, np.int64)
    mq = span_id == -1
    ctx = ~in_span & ~is_prefix & ~mq
    d = is_prefix * 1 + ctx * 2 + in_span * 4 + mq * 8 + (in_span & (span_id > 0)) * 16
    sees = (is_prefix | ctx | mq) * 1 + in_span * 2 + mq * 4
    return d + sees * 32 + (span_id & 0xFFFFFF) * 256


def append(cache, k, v, table, lens, n_new, desc=None):
    """k, v float64 (B, H, T, D). Changes the cache."""
    B, H = k.shape[:2]
    for b in range(B):
        n, ln = int(n_new[b]), int(lens[b])
        if n == 0:
            continue
        for block in range(ln // PAGE, -(-(ln + n) // PAGE)):
            page, base = table[b][block], block * PAGE
            lo, hi = max(ln - base, 0), min(ln + n - base, PAGE)
            for h in range(H):
                for x, name in ((k, "k"), (v, "v")):
                    new = x[b, h, base + lo - ln:base + hi - ln]
                    old = int(np.log2(cache[name + "_scale"][page, h])) if lo > 0 else -32
                    e = max(exponent(new), old)
                    stored = cache[name][page, h]
                    if lo == 0:
                        stored[:] = 0.0
                    elif e > old:
                        stored[:lo] = e4m3(stored[:lo] * 2.0 ** (old - e))
                    stored[lo:hi] = e4m3(new / 2.0 ** e)
                    cache[name + "_scale"][page, h] = 2.0 ** e
                if desc is not None and cache["desc"] is not None:
                    cache["desc"][page, h, lo:hi] = desc[b, base + lo - ln:base + hi - ln]


def values(cache, table_row, n, h, name):
    """(n, D): what a sequence's head holds."""
    pages = [table_row[i] for i in range(-(-n // PAGE))]
    if not pages:
        return np.zeros((0, cache[name].shape[3]))
    return np.concatenate([cache[name][p, h] * cache[name + "_scale"][p, h] for p in pages])[:n]


def rule(dq, i, dk, j):
    """(queries, keys): the 4-section rule on descriptors dq (queries,), dk (keys,) at indices i, j."""
    dq, i = dq[:, None], i[:, None]
    sees = ((dq >> 5) & dk & 7) != 0
    causal = ((dq & dk & 2) != 0) & (i >= j)
    span = ((dq & 16) != 0) & ((dk & 4) != 0) & ((dq >> 8) == (dk >> 8))
    return sees | causal | span


def attention(cache, q, table, lens, q_lens, scale, causal=True):
    """q float64 (B, H, T, D). Returns O, LSE (base 2), weights (B, Hkv, max len), A = sum p |v|, and the largest sum of |q k| of a row, in score units."""
    B, H, T, D = q.shape
    Hkv = cache["k"].shape[1]
    G = H // Hkv
    o, a = np.zeros(q.shape), np.zeros(q.shape)
    lse, mag = np.full((B, H, T), -np.inf), np.zeros((B, H, T))
    weights = np.zeros((B, Hkv, max([int(n) for n in lens] + [1])))
    for b in range(B):
        n, m = int(lens[b]), int(q_lens[b])
        j = np.arange(n)
        for h in range(Hkv):
            k, v = values(cache, table[b], n, h, "k"), values(cache, table[b], n, h, "v")
            rows = np.array([i for i in range(m) if n - m + i >= 0], int)
            at = n - m + rows
            if len(rows) == 0 or n == 0:
                continue
            if cache["desc"] is not None:
                d = np.concatenate([cache["desc"][p, h] for p in table[b][:-(-n // PAGE)]])[:n]
                see = rule(d[at], at, d, j)
            else:
                see = at[:, None] >= j if causal else np.ones((len(rows), n), bool)
            for g in range(G):
                x = q[b, h * G + g, rows]
                for r, row in enumerate(rows):   # a row takes the keys and values that it sees and nothing of the others
                    s = see[r]
                    if not s.any():
                        continue
                    sc = (k[s] @ x[r]) * scale
                    top = sc.max()
                    p = np.exp(sc - top)
                    l = p.sum()
                    p = p / l
                    o[b, h * G + g, row] = p @ v[s]
                    a[b, h * G + g, row] = p @ np.abs(v[s])
                    lse[b, h * G + g, row] = (top + np.log(l)) / np.log(2.0)
                    mag[b, h * G + g, row] = (np.abs(k[s]) @ np.abs(x[r])).max() * scale
                    weights[b, h, :n][s] += p
    return o, lse, weights, a, mag


def evict(weights, lens, keep, recent, first):
    """index (B, H, keep), -1 behind; new lens. weights (B, H, tokens) as numbers of any type; missing tokens weigh 0."""
    B, H, W = weights.shape
    index = np.full((B, H, keep), -1, np.int64)
    for b in range(B):
        n = int(lens[b])
        for h in range(H):
            if n <= keep:
                index[b, h, :n] = np.arange(n)
                continue
            w = np.zeros(n)
            w[:min(n, W)] = weights[b, h, :n]
            w = np.where(np.isnan(w), np.inf, w)
            nan_above = np.zeros(n)
            nan_above[:min(n, W)] = np.isnan(weights[b, h, :n])
            free = np.arange(first, n - recent)
            order = sorted(free, key=lambda t: (-nan_above[t], -w[t], t))[:keep - first - recent]
            index[b, h] = np.sort(np.concatenate([np.arange(first), np.array(order, int), np.arange(n - recent, n)]))
    return index, np.minimum(np.asarray(lens), keep)
