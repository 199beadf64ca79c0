"""The 4-bit key/value cache in 64 bits on the CPU (numpy), from its definition: what the GPU tests compare with.

A cache is a dict: k, v uint8 (pages, H, 64, D / 2), the bytes; k_scale, v_scale uint8 (pages, H, 64, D / 16); desc int64 (pages, H, 64) or None.
"""
import numpy as np

PAGE, GROUP, TOP, NAN = 64, 16, 226, 255
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SCALES = np.array([b * 2.0 ** -17 if b < 8 else (8 + b % 8) * 2.0 ** (b // 8 - 18) for b in range(TOP + 1)])


def _nearest(x, grid):
    """Index of the nearest of an ascending grid; of two equally near ones the even index; x >= 0 beyond the last has the last. Exact: the middles times anything of few bits are."""
    middle = (grid[1:] + grid[:-1]) / 2
    lower, upper = np.searchsorted(middle, x, "left"), np.searchsorted(middle, x, "right")
    return np.where((lower != upper) & (lower % 2 == 1), upper, lower)


def quantise(x):
    """(bytes, scale bytes) of x float64 (..., D)."""
    g = np.asarray(x, np.float64)
    g = g.reshape(g.shape[:-1] + (-1, GROUP))
    bad = ~np.isfinite(g).all(-1)
    a = np.where(bad[..., None], 0.0, np.abs(g))
    byte = _nearest(a.max(-1), 6.0 * SCALES)   # nearest to a sixth
    size = SCALES[byte][..., None]
    code = np.zeros(g.shape, int)
    for i, (lo, hi) in enumerate(zip(LEVELS[:-1], LEVELS[1:])):   # past the middle of two levels, or on it where the upper one is even
        edge = (lo + hi) / 2 * size
        code += (a > edge) | ((a == edge) & (i % 2 == 1) & (size > 0))
    code = np.where(size == 0, 0, code) + 8 * (np.signbit(g) & ~bad[..., None])
    code = code.reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(bad, NAN, byte).astype(np.uint8)


def numbers(codes, scale):
    """What bytes stand for, float64 (..., D)."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (-1,)).astype(int)
    x = np.where(c & 8, -1.0, 1.0) * LEVELS[c & 7]
    size = np.append(SCALES, [np.nan] * (256 - TOP - 1))[scale.astype(int)]
    return x * np.repeat(size, GROUP, -1)


def append(cache, k, v, table, lens, n_new, desc=None):
    """k, v float64 (B, H, T, D). Changes the cache."""
    for b in range(k.shape[0]):
        n, ln = int(n_new[b]), int(lens[b])
        if n == 0:
            continue
        for block in range(ln // PAGE, -(-(ln + n) // PAGE)):
            page, base = table[b][block], block * PAGE
            lo, hi = max(ln - base, 0), min(ln + n - base, PAGE)
            for x, name in ((k, "k"), (v, "v")):
                if lo == 0:
                    cache[name][page], cache[name + "_scale"][page] = 0, 0
                codes, scale = quantise(x[b, :, base + lo - ln:base + hi - ln])
                cache[name][page, :, lo:hi], cache[name + "_scale"][page, :, lo:hi] = codes, scale
            if desc is not None and cache["desc"] is not None:
                cache["desc"][page, :, lo:hi] = desc[b, base + lo - ln:base + hi - ln]


def as_values(cache):
    """The cache as the attention of kv_cache_oracle takes one: values, and scales of 1."""
    ones = np.ones(cache["k"].shape[:2])
    return {"k": numbers(cache["k"], cache["k_scale"]), "v": numbers(cache["v"], cache["v_scale"]), "k_scale": ones, "v_scale": ones, "desc": cache["desc"]}
