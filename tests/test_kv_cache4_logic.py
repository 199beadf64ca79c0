"""CPU tests of the 4-bit cache: its number format, the arithmetic that the kernels form it with, and the entry points' checks of arguments."""
import ctypes

import numpy as np
import torch

from oracle import kv_cache4_oracle as k4


def test_scales_are_the_upper_bits_of_halves():
    halves = (np.arange(256, dtype=np.uint16) << 7).view(np.float16).astype(np.float64)
    assert np.array_equal(halves[:k4.TOP + 1], k4.SCALES) and np.isnan(halves[k4.NAN]) and k4.SCALES[-1] == 10240
    # times any number a half, and a bfloat16, exactly
    every = (k4.SCALES[:, None] * k4.LEVELS).ravel()
    assert np.array_equal(every, every.astype(np.float16).astype(np.float64))
    assert np.array_equal(every, torch.tensor(every).bfloat16().double().numpy())


def test_oracle_takes_the_nearest():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * np.exp(4 * rng.standard_normal((200, 1)))
    x[0], x[1, :16], x[2, 3], x[3, 20], x[4, :16] = 0, 1e6, np.nan, -np.inf, 2.0 ** -20
    codes, scale = k4.quantise(x)
    y = k4.numbers(codes, scale)
    g, s = x.reshape(200, 4, 16), scale.astype(int)
    bad = ~np.isfinite(g).all(-1)
    assert np.array_equal(s == k4.NAN, bad) and np.isnan(y.reshape(g.shape)[bad]).all() and not codes.reshape(200, 4, 8)[bad].any()
    top = np.abs(g).max(-1)
    for other in range(k4.TOP + 1):
        assert (np.abs(top / 6 - k4.SCALES[np.minimum(s, k4.TOP)]) <= np.abs(top / 6 - k4.SCALES[other]))[~bad].all()
    grid = np.concatenate((-k4.LEVELS, k4.LEVELS))
    size = np.where(bad, 1, k4.SCALES[np.minimum(s, k4.TOP)])[..., None]
    best = np.abs(g[..., None] - grid * size[..., None]).min(-1)
    assert (np.abs(g - y.reshape(g.shape)) <= best)[~bad].all()
    assert np.abs(y[1, :16]).max() == 61440 and not y[0].any() and not y[4, :16].any()
    # ties go to even: a quarter of the scale, three quarters, five, seven ...
    x = np.zeros((1, 16))
    x[0, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]
    assert k4.numbers(*k4.quantise(x))[0, :8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4]
    assert k4.quantise(np.full((1, 16), 6 * 17 / 16))[1] == 120 and k4.quantise(np.full((1, 16), 6 * 19 / 16))[1] == 122   # scales of 1 and 1.25: 1.0625 is between 1 and 1.125


def test_product_with_a_rounded_inverse_decides_as_the_quotient_does():
    """What the kernels do with 16-bit numbers: x times a float within 2**-22 of 1 / scale, brought to a grid of 2**-13 by a fused sum with 1536, decides on the same side of each middle of two levels as
    x / scale, for every x of 11 bits (halves, and bfloat16 of 8 bits among them) and every scale of 4 bits. Powers of two apart, that is all of them: quotients are 6.4 at most."""
    x = np.arange(1024, 2048, dtype=np.float64)
    plain = 0
    for m in range(8, 16):
        nearest = np.float32(1) / np.float32(m)   # numpy divides as IEEE says
        for inverse in (nearest, np.nextafter(nearest, np.float32(0)), np.nextafter(nearest, np.float32(1))):   # the hardware's is off by one step at most
            inverse = np.float64(inverse)
            for e in range(-30, -4):
                v = x * 2.0 ** e
                v = v[v <= 6.5 * m]
                q = (v * inverse + 1536.0).astype(np.float32) - np.float32(1536)   # (the sum has 48 bits: exact in 64, rounded once)
                for middle in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
                    exact = np.sign(v - middle * m)
                    assert np.array_equal(np.sign(q.astype(np.float64) - middle), exact)
                    plain += (np.sign((v * inverse).astype(np.float32).astype(np.float64) - middle) != exact).sum()
    assert plain > 0   # the grid is needed


def test_product_with_a_sixth_decides_as_the_quotient_does():
    """What the kernels do with the largest of a group of 16-bit numbers: times the float nearest to 1 / 6, rounded to 17 bits, then to the nearest scale."""
    x = (np.arange(1024, 2048, dtype=np.float64)[:, None] * 2.0 ** np.arange(-40.0, 7.0)).ravel()
    x = x[x <= 65504]
    u = (x.astype(np.float32) * (np.float32(1) / np.float32(6))).view(np.uint32)
    u = (u + np.uint32(0x40)) & ~np.uint32(0x7F)
    sixth = u.view(np.float32)
    byte = np.where(sixth < 2.0 ** -14, np.rint(sixth * np.float32(2.0 ** 17)).astype(np.int64), np.minimum(k4.TOP, ((u + np.uint32(0x7FFFF) + (u >> 20 & 1)) >> 20).astype(np.int64) - 896))
    assert np.array_equal(byte, k4._nearest(x, 6.0 * k4.SCALES))


def test_quotient_by_six_is_not_rounded_onto_the_middle_of_two_scales():
    """In 32 bits, for the floats next to six times each middle: they stay on their side of it."""
    middle = (k4.SCALES[1:] + k4.SCALES[:-1]) / 2
    six = (6 * middle).astype(np.float32)
    assert np.array_equal(six.astype(np.float64), 6 * middle)
    for towards, side in ((0, -1), (np.inf, 1)):
        q = np.nextafter(six, np.float32(towards)) / np.float32(6)
        assert (np.sign(q.astype(np.float64) - middle) == side).all()
    assert np.array_equal((six / np.float32(6)).astype(np.float64), middle)


def test_entry_points_reject_bad_arguments_before_touching_cuda():
    from kerneldev_b200 import _capi as m
    lib, ref = m.load(), ctypes.byref
    c, s, t, q = m.KdCache4(), m.KdCacheSeqs(), m.KdCacheTokens(), m.KdCacheQueries()
    c.k = c.v = c.k_scale = c.v_scale = 0x10000
    c.pages, c.H, c.D = 4, 2, 64
    s.table = s.lens = 0x10000
    s.B, s.blocks, s.table_stride = 1, 2, 2
    t.T, t.dtype = 1, m.KD_BF16

    def refused(rc, code, text):
        assert rc == code and text in lib.kd_last_error(), lib.kd_last_error()

    refused(lib.kd_cache4_append(None, ref(s), ref(t), None), -1, b"null")
    refused(lib.kd_cache4_append(ref(c), ref(s), ref(t), None), -1, b"k is null")
    for field, value, code, text in (("D", 72, -1, b"head dim"), ("k", 0x10008, -2, b"aligned"), ("k_scale", 0x10004, -2, b"k_scale"), ("v_scale", 0x10008, -2, b"v_scale"), ("v_scale", 0, -1, b"null"),
                                     ("pages", 0, -1, b"shape")):
        old = getattr(c, field)
        setattr(c, field, value)
        refused(lib.kd_cache4_append(ref(c), ref(s), ref(t), None), code, text)
        setattr(c, field, old)
    q.H, q.T, q.dtype, q.sm_scale = 3, 1, m.KD_F16, 1.0
    refused(lib.kd_cache4_attention(ref(c), ref(s), ref(q), None), -1, b"H=3 for 2 heads")
    q.H = 4
    refused(lib.kd_cache4_attention(ref(c), ref(s), ref(q), None), -1, b"q is null")
    refused(lib.kd_cache4_attention_workspace(ref(c), ref(s), ref(q), None), -1, b"null")
    e = m.KdCacheEviction()
    refused(lib.kd_cache4_evict(ref(c), ref(s), ref(e), None), -1, b"eviction")
    refused(lib.kd_cache4_read(ref(c), ref(s), None, -1, m.KD_F16, None, None, None), -1, b"count")
    # workspaces go by shapes alone, and are the 8-bit cache's
    n4, n8, c8 = ctypes.c_size_t(1), ctypes.c_size_t(2), m.KdCache()
    for name, _ in m.KdCache._fields_:
        setattr(c8, name, getattr(c, name))
    s.blocks = 40
    assert lib.kd_cache4_attention_workspace(ref(c), ref(s), ref(q), ref(n4)) == 0 and lib.kd_cache_attention_workspace(ref(c8), ref(s), ref(q), ref(n8)) == 0 and n4.value == n8.value > 0


def test_a_cache_has_eight_or_four_bits():
    import pytest
    from kerneldev_b200.kv_cache import KVCache
    with pytest.raises(ValueError, match="8 or 4"):
        KVCache.empty(2, 2, 64, device="cpu", bits=5)
    with pytest.raises(ValueError, match="head_dim"):
        KVCache.empty(2, 2, 40, device="cpu", bits=4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        KVCache.empty(2, 2, 64, device="cpu", bits=4)
