"""CPU tests of the 8-bit cache: the entry points' checks of arguments, and the oracle's number format against torch's."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_cache_oracle as ko


def _cache():
    from kerneldev_b200 import _capi
    c = _capi.KdCache()
    c.k = c.v = c.k_scale = c.v_scale = 0x10000   # never read: every call here is refused first
    c.pages, c.H, c.D = 4, 2, 64
    s = _capi.KdCacheSeqs()
    s.table = s.lens = 0x10000
    s.B, s.blocks, s.table_stride = 1, 2, 2
    return _capi, _capi.load(), c, s


def test_entry_points_reject_bad_arguments_before_touching_cuda():
    m, lib, c, s = _cache()
    t = m.KdCacheTokens()
    t.T, t.dtype = 1, m.KD_BF16
    ref = ctypes.byref

    def refused(rc, code, text):
        assert rc == code and text in lib.kd_last_error(), lib.kd_last_error()

    refused(lib.kd_cache_append(None, ref(s), ref(t), None), -1, b"null")
    refused(lib.kd_cache_append(ref(c), ref(s), None, None), -1, b"null")
    refused(lib.kd_cache_append(ref(c), ref(s), ref(t), None), -1, b"k is null")
    t.k.ptr = t.v.ptr = 0x10000
    t.k.stride_t = 3
    refused(lib.kd_cache_append(ref(c), ref(s), ref(t), None), -2, b"16")
    t.k.stride_t, t.dtype = 64, 7
    refused(lib.kd_cache_append(ref(c), ref(s), ref(t), None), -1, b"dtype")
    t.dtype, t.T = m.KD_F32, -1
    refused(lib.kd_cache_append(ref(c), ref(s), ref(t), None), -1, b"count")
    t.T = 0
    assert lib.kd_cache_append(ref(c), ref(s), ref(t), None) == 0   # nothing to do
    for field, value, text in (("D", 72, b"head dim"), ("D", 144, b"head dim"), ("pages", 0, b"shape"), ("H", 0, b"shape"), ("k", 0, b"null"), ("v", 0x10008, b"aligned")):
        old = getattr(c, field)
        setattr(c, field, value)
        refused(lib.kd_cache_append(ref(c), ref(s), ref(t), None), -2 if text == b"aligned" else -1, text)
        setattr(c, field, old)
    for field, value, code in (("B", -1, -1), ("blocks", -1, -1), ("blocks", (1 << 24) + 1, -4), ("lens", None, -1), ("table", None, -1)):
        old = getattr(s, field)
        setattr(s, field, value)
        assert lib.kd_cache_append(ref(c), ref(s), ref(t), None) == code
        setattr(s, field, old)
    q = m.KdCacheQueries()
    q.H, q.T, q.dtype, q.sm_scale = 3, 1, m.KD_F16, 1.0
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -1, b"H=3 for 2 heads")
    q.H, q.dtype = 4, m.KD_F32
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -1, b"dtype")
    q.dtype, q.sm_scale = m.KD_F16, float("nan")
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -1, b"sm_scale")
    q.sm_scale = 1.0
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -1, b"q is null")
    q.q.ptr = q.o.ptr = 0x10000
    q.weights, q.w_len = 0x10000, -1
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -1, b"w_len")
    q.T = 1 << 30
    refused(lib.kd_cache_attention(ref(c), ref(s), ref(q), None), -4, b"rows")
    n = ctypes.c_size_t(1)
    q.T = 0
    assert lib.kd_cache_attention_workspace(ref(c), ref(s), ref(q), ref(n)) == 0 and n.value == 0
    refused(lib.kd_cache_attention_workspace(ref(c), ref(s), ref(q), None), -1, b"null")
    e = m.KdCacheEviction()
    for keep, recent, first in ((0, 0, 0), (4, -1, 0), (4, 0, -1), (4, 3, 2), (4, 5, 0)):
        e.keep, e.recent, e.first = keep, recent, first
        refused(lib.kd_cache_evict(ref(c), ref(s), ref(e), None), -1, b"eviction")
    e.keep, e.recent, e.first = 4, 2, 2
    refused(lib.kd_cache_evict(ref(c), ref(s), ref(e), None), -1, b"null")
    refused(lib.kd_cache_read(ref(c), ref(s), None, -1, m.KD_F16, None, None, None), -1, b"count")
    refused(lib.kd_cache_read(ref(c), ref(s), None, 1, 9, None, None, None), -1, b"dtype")
    refused(lib.kd_cache_read(ref(c), ref(s), None, 1, m.KD_F16, None, None, None), -1, b"null")
    s.B = 0
    assert lib.kd_cache_read(ref(c), ref(s), None, 1, m.KD_F16, None, None, None) == 0


def test_entry_points_reject_descriptors_that_16_byte_copies_cannot_read():
    m, lib, c, s = _cache()
    ref = ctypes.byref
    t, q, e, n = m.KdCacheTokens(), m.KdCacheQueries(), m.KdCacheEviction(), ctypes.c_size_t()
    t.T, t.dtype = 0, m.KD_BF16
    q.H, q.T, q.dtype, q.sm_scale = 2, 0, m.KD_F16, 1.0
    e.keep = 1
    s.B = 0   # nothing to do, were it not for desc
    for offset, code in ((0, 0), (4, -2), (8, -2), (12, -2), (16, 0)):
        c.desc = 0x10000 + offset
        for rc in (lib.kd_cache_append(ref(c), ref(s), ref(t), None), lib.kd_cache_attention(ref(c), ref(s), ref(q), None), lib.kd_cache_evict(ref(c), ref(s), ref(e), None),
                   lib.kd_cache_attention_workspace(ref(c), ref(s), ref(q), ref(n)), lib.kd_cache_read(ref(c), ref(s), None, 0, m.KD_F16, None, None, None)):
            assert rc == code and (rc == 0 or b"desc" in lib.kd_last_error())


def test_workspace_of_weights_is_bounded_by_the_cache():
    """However wide the page tables are: 256 MB, or an eighth of the cache's own bytes, and the parts and statistics besides. What is below that keeps its place for the scores."""
    m, lib, c, s = _cache()
    q, n = m.KdCacheQueries(), ctypes.c_size_t()
    q.T, q.dtype, q.sm_scale, q.weights = 1, m.KD_F16, 1.0, 0x10000
    for B, H, rows, blocks, pages, D in ((128, 8, 8, 2048, 4000, 128), (1, 1, 1, 1 << 24, 10, 16), (64, 8, 5, 1 << 16, 100000, 64), (16, 4, 8, 64, 1024, 128), (128, 8, 8, 2048, 128 * 2048, 128)):
        s.B, s.blocks, s.table_stride, c.H, c.D, c.pages, q.H = B, blocks, blocks, H, D, pages, H * rows
        bytes_ = []
        for q.weights in (None, 0x10000):
            assert lib.kd_cache_attention_workspace(ctypes.byref(c), ctypes.byref(s), ctypes.byref(q), ctypes.byref(n)) == 0
            bytes_.append(n.value)
        limit = max(256 << 20, pages * H * 64 * 2 * D // 8)
        scores = B * H * blocks * 64 * {1: 2, 5: 8, 8: 8}[rows] * 4
        stats = B * H * rows * 8
        extra = bytes_[1] - bytes_[0]
        assert extra <= limit + stats + 1024
        assert extra >= scores if scores <= limit else extra <= stats + 1024


def test_cache_has_no_cpu_path():
    from kerneldev_b200 import KVCache
    with pytest.raises(RuntimeError, match="no CPU path"):
        KVCache.empty(2, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        KVCache.empty(2, 2, 60, device="cpu")


def test_oracle_numbers_are_torchs():
    """Every number of e4m3 and every point halfway between two, with their neighbours in 64 bits."""
    grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    grid = np.unique(grid[np.isfinite(grid)])
    mid = (grid[1:] + grid[:-1]) / 2
    x = np.concatenate([grid, mid, np.nextafter(mid, np.inf), np.nextafter(mid, -np.inf)])
    x32 = x.astype(np.float32).astype(np.float64)
    assert np.array_equal(ko.e4m3(x32), torch.tensor(x32).float().to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(ko.e4m3([np.inf, np.nan])).all() and ko.e4m3([1e9])[0] == 448
    assert [ko.exponent(np.array([a])) for a in (0.0, 448.0, 448.0001, 1e30, 1e-30, np.inf)] == [-32, 0, 1, 31, -32, -32]


def test_oracle_rule_is_the_operators():
    """The oracle's descriptors and rule give the mask of the attention oracle."""
    from oracle import attention_oracle as ao
    rng = np.random.default_rng(0)
    B, T = 3, 40
    ins, pre = rng.random((B, T)) < 0.4, rng.random((B, T)) < 0.3
    sid = rng.integers(-1, 4, (B, T))
    mask = np.asarray(ao.dense_mask(T, ins, sid, pre, None, B=B)).reshape(B, T, T).astype(bool)
    d = ko.descriptors(ins, sid, pre)
    for b in range(B):
        assert np.array_equal(ko.rule(d[b], np.arange(T), d[b], np.arange(T)), mask[b])
