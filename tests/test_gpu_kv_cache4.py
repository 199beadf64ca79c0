"""The 4-bit key/value cache on the GPU against its definition in 64 bits (oracle/kv_cache4_oracle.py).

Tolerances. What is stored is equal to the definition (zeros of either sign). The attention has those of the 8-bit cache, derived in test_gpu_kv_cache.py: keys and values are exact as halves there
and here, and probabilities are rounded alike. One term more: most values of a group with a large one are zeros here, so that a column's only number may belong to an unlikely token, whose probability is a
subnormal half. A half is off by 2**-25 at most below 2**-14; in its units the row's largest probability is 2**8 or more (the reference is never above the largest score), so the weight is off by 2**-33
of the largest, which is 1 at most: 2**-33 of the sum of |v| in all. (Halves as outputs are off by 2**-25 below 2**-14 as well: that term was there.)"""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import kv_cache4_oracle as k4
from oracle import kv_cache_oracle as ko
from oracle import rotate_oracle as ro
from tests.test_gpu_kv_cache import APPENDS, ATTENTION, DEV, DT, EVICTIONS, i32, metadata, rand_kv, strided, tables

pytestmark = pytest.mark.gpu


def make_cache(pages, H, D, metadata=False, fill=0xFF):
    """A cache whose pages hold NaN before anything is appended."""
    from kerneldev_b200 import KVCache
    c = KVCache.empty(pages, H, D, device=DEV, metadata=metadata, bits=4)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t.fill_(fill)
    return c


def as_oracle(c):
    raw = lambda t: t.cpu().numpy().copy()  # noqa: E731
    return {"k": raw(c.k), "v": raw(c.v), "k_scale": raw(c.k_scale), "v_scale": raw(c.v_scale), "desc": None if c.desc is None else raw(c.desc).astype(np.int64) & 0xFFFFFFFF}


def assert_cache(c, want):
    got = as_oracle(c)
    for name in ("k", "v"):
        assert np.array_equal(got[name + "_scale"], want[name + "_scale"]), name + "_scale"
        assert np.array_equal(k4.numbers(got[name], got[name + "_scale"]), k4.numbers(want[name], want[name + "_scale"]), equal_nan=True), name
    if want["desc"] is not None:
        assert np.array_equal(got["desc"], want["desc"])


def check_attention(c, q, table, lens, q_lens, got, causal=True, scale=None, weights=None, before=None):
    D = q.shape[3]
    o, lse = (x.double().cpu().numpy() for x in got)
    scale = D ** -0.5 if scale is None else scale
    held = k4.as_values(as_oracle(c))
    ro_, rl, rw, a, mag = ko.attention(held, q.cpu().double().numpy(), table, lens, q_lens, scale, causal)
    n, G = max(int(max(lens)), 1), q.shape[1] // rw.shape[1]
    size = np.stack([[np.abs(np.nan_to_num(ko.values(held, table[b], int(lens[b]), h // G, "v"))).sum(0) for h in range(q.shape[1])] for b in range(q.shape[0])])[:, :, None]
    delta = 2.0 ** -21 * (mag * 1.5 + 2) + n * 2.0 ** -24
    err = np.abs(o - ro_)
    tol = torch.finfo(q.dtype).eps / 2 * (np.abs(ro_) + 0.01 * a) + a * (2.0 ** -11 + 2 * delta[..., None]) + 2.0 ** -25 + 2.0 ** -33 * size
    assert np.isfinite(o).all()
    assert (err <= tol).all(), f"O: {(err / tol).max()} of the tolerance at {np.unravel_index((err / tol).argmax(), err.shape)}"
    assert np.array_equal(np.isinf(lse), np.isinf(rl)) and (lse[np.isinf(lse)] < 0).all()
    fin = np.isfinite(rl)
    assert (np.abs(lse[fin] - rl[fin]) <= (2 * delta)[fin] + 2.0 ** -22 * np.abs(rl[fin])).all(), "LSE"
    if weights is not None:
        w = weights.double().cpu().numpy() - (0 if before is None else before.double().cpu().numpy())
        rw = np.pad(rw, ((0, 0), (0, 0), (0, max(0, w.shape[2] - rw.shape[2]))))[..., :w.shape[2]]
        size = np.abs(rw) + (0 if before is None else np.abs(before.double().cpu().numpy()))
        rows = G * q.shape[2]
        top = delta.reshape(rw.shape[0], rw.shape[1], G, -1).max((2, 3))[..., None]
        assert (np.abs(w - rw) <= rw * 3 * top + size * rows * 2.0 ** -24 + 1e-30).all(), "weights"


def filled(rng, B, H, D, lens, dtype, meta, outliers=True):
    from kerneldev_b200 import cache_append
    blocks = max(-(-int(max(lens)) // 64), 1)
    pages = B * blocks + 2
    c = make_cache(pages, H, D, metadata=meta)
    table = tables(rng, B, blocks, pages)
    T = max(int(max(lens)), 1)
    x = rand_kv(rng, (2, B, H, T, D), dtype, outliers).to(DEV)
    m = metadata(rng, B, T)
    extra = dict(zip(("in_span", "span_id", "is_prefix"), (torch.tensor(t, device=DEV) for t in m))) if meta else {}
    cache_append(c, x[0], x[1], i32(table), i32(np.zeros(B)), i32(lens), **extra)
    return c, table


# ---- appending and reading ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[0]}-{c[2]}-{c[3]}")
def test_append_and_read(case):
    from kerneldev_b200 import cache_append, cache_read
    D, H, dtype, layout, lens, new = case
    rng = np.random.default_rng(D)
    B, T, blocks = len(lens), max(new), -(-max(a + n for a, n in zip(lens, new)) // 64) + 1
    pages = B * blocks + 2
    c = make_cache(pages, H, D, metadata=True)
    table = tables(rng, B, blocks, pages)
    want = as_oracle(c)
    zero = np.zeros(B, int)
    meta = [metadata(rng, B, n) for n in (max(max(lens), 1), T)]
    steps = [(zero, lens, rand_kv(rng, (2, B, H, max(max(lens), 1), D), DT[dtype], False), meta[0]), (lens, new, rand_kv(rng, (2, B, H, T, D), DT[dtype]), meta[1])]
    for start, count, x, m in steps:
        x = x.to(DEV)
        cache_append(c, strided(x[0], layout), strided(x[1], layout), i32(table), i32(start), i32(count),
                     in_span=torch.tensor(m[0], device=DEV), span_id=torch.tensor(m[1], device=DEV), is_prefix=torch.tensor(m[2], device=DEV))
        k4.append(want, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, start, count, ko.descriptors(*m))
        assert_cache(c, want)
    total = np.array(lens) + np.array(new)
    start = np.maximum(total - 70, 0)
    held = k4.as_values(want)
    for out in (torch.bfloat16, torch.float32, torch.float16):
        k, v = cache_read(c, i32(table), i32(total), 75, start=i32(start), dtype=out)
        for b in range(B):
            for h in range(H):
                for got, name in ((k, "k"), (v, "v")):
                    x = np.zeros((75, D))
                    own = ko.values(held, table[b], int(total[b]), h, name)[start[b]:]
                    x[:len(own)] = own
                    assert np.array_equal(got[b, h].double().cpu().numpy(), x)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_magnitude(dtype):
    """Groups of all sizes, from below the smallest scale to beyond the largest, whose numbers lie on and beside the middles of the levels."""
    from kerneldev_b200 import cache_append
    rng = np.random.default_rng(3)
    n, D = 640, 64
    x = np.concatenate([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], rng.uniform(0, 6, 8)])[None, :] * rng.choice([-1.0, 1.0], (n * D // 16, 16))
    x *= np.exp2(rng.integers(-24, 15, (n * D // 16, 1))) * rng.integers(8, 16, (n * D // 16, 1)) / 8
    x = torch.tensor(x.reshape(1, 1, n, D)).clamp(-65000, 65000).to(DT[dtype])
    if dtype == "f32":   # the floats next to the middles
        u = x.view(torch.int32)
        u[..., ::3] += 1
        u[..., 1::3] -= 1
    c = make_cache(11, 1, D)
    want, table = as_oracle(c), np.arange(10)[None]
    cache_append(c, x.to(DEV), -x.to(DEV), i32(table), i32([0]))
    k4.append(want, x.double().numpy(), -x.double().numpy(), table, [0], [n])
    assert_cache(c, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_numbers_without_a_place(dtype):
    """Infinities and NaN make their group NaN, and no other; numbers beyond the largest scale saturate, those below the smallest are zeros."""
    from kerneldev_b200 import cache_append, cache_read
    c = make_cache(2, 1, 64)
    x = torch.randn((1, 1, 66, 64))
    x[0, 0, 3, 5], x[0, 0, 4, 63], x[0, 0, 5, 16] = float("nan"), float("inf"), -float("inf")
    x[0, 0, 64] = 6e4 if dtype == "f16" else 1e38
    x[0, 0, 65] = 2.0 ** -20
    x[0, 0, 6, 0] = 1e-40
    x = x.to(DT[dtype])
    want, table = as_oracle(c), np.array([[1, 0]])
    cache_append(c, x.to(DEV), x.to(DEV), i32(table), i32([0]))
    k4.append(want, x.double().numpy(), x.double().numpy(), table, [0], [66])
    assert_cache(c, want)
    k, _ = cache_read(c, i32(table), i32([66]), 66)
    bad = torch.zeros((66, 64), dtype=torch.bool, device=DEV)
    bad[3, :16] = bad[4, 48:] = bad[5, 16:32] = True
    assert torch.equal(torch.isnan(k[0, 0]), bad) and float(k[0, 0, 64].abs().min()) >= 5.5e4 and not k[0, 0, 65].any()


# ---- attention ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"h{c[1]}-{c[2]}-d{c[3]}-q{c[4]}-{c[5]}-{c[6]}")
@pytest.mark.parametrize("weigh", [False, True], ids=["plain", "weigh"])
def test_attention(case, weigh):
    from kerneldev_b200 import cache_attention
    B, H, Hkv, D, T, dtype, mask, layout, lens, q_lens = case
    rng = np.random.default_rng(D + T)
    c, table = filled(rng, B, Hkv, D, lens, DT[dtype], mask == "hier")
    q = strided((rand_kv(rng, (B, H, T, D), torch.float32, False) * 1.5).to(DT[dtype]).to(DEV), layout)
    kw, before = {}, None
    if weigh:
        before = torch.tensor(rng.random((B, Hkv, max(lens) + 3)), dtype=torch.float32, device=DEV)
        kw["weights"] = before.clone()
    o, lse = cache_attention(q, c, i32(table), i32(lens), None if q_lens is None else i32(q_lens), causal=mask != "full", return_lse=True, **kw)
    check_attention(c, q, table, lens, q_lens or [T] * B, (o, lse), causal=mask != "full", weights=kw.get("weights"), before=before)
    assert o.is_contiguous() and o.dtype == q.dtype
    o2 = cache_attention(q, c, i32(table), i32(lens), None if q_lens is None else i32(q_lens), causal=mask != "full", out_layout="input")
    assert torch.equal(o, o2)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("G,T", [(1, 1), (3, 4), (4, 7), (2, 40)])
def test_attention_at_every_head_dim(D, G, T):
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(D * T)
    lens = [n + T for n in (700, 0, 63, 1)]
    c, table = filled(rng, 4, 2, D, lens, torch.float16, False)
    q = (rand_kv(rng, (4, 2 * G, T, D), torch.float32, False) * 1.5).half().to(DEV)
    w = torch.zeros((4, 2, max(lens)), device=DEV)
    check_attention(c, q, table, lens, [T] * 4, cache_attention(q, c, i32(table), i32(lens), return_lse=True, weights=w), weights=w)


@pytest.mark.parametrize("D", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("T,G", [(1, 4), (6, 3), (80, 2)])
def test_attention_does_not_read_what_is_masked(D, T, G):
    """Groups of NaN in keys and values that a query does not see, and behind the sequences, reach nothing; those that it sees do."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    rng = np.random.default_rng(8)
    B, Hkv, n = 2, 2, 330
    c = make_cache(16, Hkv, D, metadata=True)
    table = tables(rng, B, 6, 16)
    x = rand_kv(rng, (2, B, Hkv, n, D), torch.float32)
    ins, sid, pre = np.zeros((B, n), bool), np.zeros((B, n), np.int64), np.zeros((B, n), bool)
    ins[:, 70:190] = True
    sid[:, 70:190] = 1 + np.arange(120) // 40
    bad = rng.random((2, B, Hkv, n)) < 0.2
    bad[:, :, :, :70] = bad[:, :, :, 190:] = False
    x[torch.tensor(bad)] = float("nan")
    x[0, :, :, 100, 5] = float("inf")
    cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32([0, 0]), i32([n, n - 7]), in_span=torch.tensor(ins, device=DEV), span_id=torch.tensor(sid, device=DEV),
                 is_prefix=torch.tensor(pre, device=DEV))
    q = rand_kv(rng, (B, Hkv * G, T, D), torch.bfloat16, False).to(DEV)
    lens = [n, n - 7]
    w = torch.zeros((B, Hkv, n), device=DEV)
    got = cache_attention(q, c, i32(table), i32(lens), return_lse=True, weights=w)
    check_attention(c, q, table, lens, [T] * B, got, weights=w)
    # what lies behind the last token of its page may be anything, scales that are never written among it
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t[table[1, 5], :, 323 % 64:] = 0xF3
    again = cache_attention(q, c, i32(table), i32(lens), return_lse=True)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    # a group of values that a query does see: NaN in its columns alone
    ks, vs = (torch.where(t == 0xFF, 0, t) for t in (c.k_scale, c.v_scale))
    ks[table[1, 5]], vs[table[1, 5]] = 100, 100
    c2 = KVCache(c.k.clone(), c.v.clone(), ks, vs)   # without metadata, causal: the spans are seen
    vs[table[0, 2], :, 9, 0] = 0xFF
    o, lse = cache_attention(q, c2, i32(table), i32(lens), return_lse=True)
    assert torch.isfinite(lse).all() and torch.isfinite(o[1]).all()
    assert torch.isnan(o[0, ..., :16]).all() and torch.isfinite(o[0, ..., 16:]).all()


@pytest.mark.parametrize("B,Hkv,G,T,D,meta", [(70, 2, 2, 1, 64, True), (300, 1, 8, 1, 32, False), (140, 4, 1, 3, 48, True), (300, 8, 1, 1, 16, False), (40, 8, 5, 8, 64, False),
                                              (7, 1, 12, 3, 128, True), (30, 8, 2, 1, 128, False)])
def test_attention_many_sequences(B, Hkv, G, T, D, meta):
    """More sequences than lanes, shares of few and of many heads, CTAs with several items, empty sequences and sequences without a query among them."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 140, B)
    lens[rng.integers(0, B, 3)] = [700, 641, 0]
    q_lens = rng.integers(0, T + 1, B) if T > 1 else None
    c, table = filled(rng, B, Hkv, D, lens, torch.float16, meta)
    q = rand_kv(rng, (B, Hkv * G, T, D), torch.float16, False).to(DEV)
    w = torch.zeros((B, Hkv, int(lens.max())), device=DEV)
    got = cache_attention(q, c, i32(table), i32(lens), None if q_lens is None else i32(q_lens), return_lse=True, weights=w)
    check_attention(c, q, table, lens, [T] * B if q_lens is None else q_lens, got, weights=w)


@pytest.mark.parametrize("G,T", [(4, 1), (3, 4), (2, 60)])
def test_attention_of_sizes_far_apart(G, T):
    """Values whose groups lie 2**30 apart, keys that make scores of hundreds, groups of zeros."""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(4)
    c = make_cache(6, 1, 32)
    table, n = np.array([[4, 1, 0, 5, 2]]), 300
    x = rand_kv(rng, (2, 1, 1, n, 32), torch.float32, False)
    x[1, :, :, ::3] *= 2.0 ** 12
    x[1, :, :, 1::3, :16] *= 2.0 ** -14
    x[1, :, :, 128:192] = 0
    x[0, :, :, 64:128] *= 100
    cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32([0]))
    q = (rand_kv(rng, (1, G, T, 32), torch.float32, False) * 3).to(torch.float16).to(DEV)
    check_attention(c, q, table, [n], [T], cache_attention(q, c, i32(table), i32([n]), return_lse=True, sm_scale=0.5), scale=0.5)


@pytest.mark.parametrize("G,T", [(2, 1), (2, 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scores_far_from_zero(G, T, dtype):
    """Keys of 2**15 and queries of the largest halves: the row's largest score takes it all (in 64 bits: scores lie thousands apart). Weights are checked for few rows, whose scores are kept; those of many rows
    come from scores that are added up once more in another order, which in such rows says nothing (the 8-bit cache's do, too)."""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(4)
    n, D = 200, 64
    c = make_cache(5, 1, D)
    table = np.arange(4)[None]
    x = torch.tensor(rng.standard_normal((2, 1, 1, n, D)))
    x[0] *= 2.0 ** 13
    cache_append(c, x[0].float().to(DEV), x[1].float().to(DEV), i32(table), i32([0]))
    q = (torch.tensor(rng.standard_normal((1, G, T, D))) * 8000).to(dtype).to(DEV)
    w = torch.zeros((1, 1, n), device=DEV)
    o, lse = cache_attention(q, c, i32(table), i32([n]), return_lse=True, weights=w)
    v = k4.as_values(as_oracle(c))
    ro_, rl, rw, _, _ = ko.attention(v, q.cpu().double().numpy(), table, [n], [T], D ** -0.5)
    # the two largest scores of a row lie at least 2**12 apart here, beside errors of 2**-21 of 2**33: one weight is 1 but where they are nearer
    err = np.abs(o.double().cpu().numpy() - ro_)
    assert (err <= np.abs(ro_) * torch.finfo(dtype).eps + 2.0 ** -10).all()
    assert (np.abs(lse.double().cpu().numpy() - rl) <= np.abs(rl) * 2.0 ** -20).all()
    if G * T <= 8:
        assert np.abs(w.double().cpu().numpy() - rw).max() < 1e-3


def test_attention_long_tail():
    """One key that takes half of the weight and thousands that share the rest."""
    from kerneldev_b200 import cache_append, cache_attention
    n, D = 20000, 64
    rng = np.random.default_rng(6)
    c = make_cache(320, 1, D)
    table = tables(rng, 1, 313, 320)
    k, v = torch.zeros((1, 1, n, D)), rand_kv(rng, (1, 1, n, D), torch.float32, False) + 1.0
    k[0, 0, 777, 0] = 8.0
    q = torch.zeros((1, 2, 1, D))
    q[..., 0] = np.log(n) * D ** 0.5 / 8
    q = q.to(torch.float16).to(DEV)
    cache_append(c, k.to(DEV), v.to(DEV), i32(table), i32([0]))
    check_attention(c, q, table, [n], [1], cache_attention(q, c, i32(table), i32([n]), return_lse=True))


@pytest.mark.parametrize("B,Hkv,G,T", [(2, 2, 3, 1), (2, 1, 8, 3), (40, 8, 1, 1), (2, 2, 2, 40)])
@pytest.mark.parametrize("weigh", [False, True], ids=["plain", "weigh"])
def test_nan_in_a_live_query_row(B, Hkv, G, T, weigh):
    """The row is NaN, its log-sum-exp too, and so is the weight of every token that it sees; all other rows are as without it."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(B + T)
    lens = rng.integers(1200, 1900, B)
    c, table = filled(rng, B, Hkv, 64, lens, torch.bfloat16, False)
    q = rand_kv(rng, (B, Hkv * G, T, 64), torch.bfloat16, False).to(DEV)
    bad = q.clone()
    b, h, i = B - 1, Hkv * G - 1, T // 2
    bad[b, h, i, 7] = float("nan")
    results = []
    for x in (q, bad):
        w = torch.zeros((B, Hkv, 1900), device=DEV) if weigh else None
        results.append((*cache_attention(x, c, i32(table), i32(lens), return_lse=True, weights=w), w))
    (o, lse, w), (bo, bl, bw) = results
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    assert torch.isnan(bo[b, h, i]).all() and torch.isnan(bl[b, h, i])
    live = torch.ones((B, Hkv * G, T), dtype=torch.bool, device=DEV)
    live[b, h, i] = False
    assert torch.equal(bo[live], o[live]) and torch.equal(bl[live], lse[live])
    if weigh:
        seen = torch.zeros_like(w, dtype=torch.bool)
        seen[b, Hkv - 1, :int(lens[b]) - T + i + 1] = True
        assert torch.isnan(bw[seen]).all() and torch.equal(bw[~seen], w[~seen])


# ---- eviction -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("case", EVICTIONS[:9], ids=lambda c: f"d{c[1]}-keep{c[3]}-{c[6]}")
def test_evict(case):
    from kerneldev_b200 import KVCache, cache_evict
    H, D, lens, keep, recent, first, kind = case
    rng = np.random.default_rng(keep)
    B, n = len(lens), max(lens)
    c, table = filled(rng, B, H, D, lens, torch.bfloat16, True)
    out_blocks, pages = -(-keep // 64), c.k.shape[0]
    grow = lambda t: torch.cat([t, torch.full((B * out_blocks + 1,) + t.shape[1:], 0xFF if t.dtype == torch.uint8 else 1, dtype=t.dtype, device=DEV)])  # noqa: E731
    c = KVCache(*(grow(t) for t in (c.k, c.v, c.k_scale, c.v_scale, c.desc)))
    out = pages + rng.permutation(B * out_blocks + 1)[:B * out_blocks].reshape(B, out_blocks)
    w = {"spread": np.exp(2 * rng.standard_normal((B, H, n))), "ties": rng.integers(0, 3, (B, H, n)) * 0.5, "zeros": np.zeros((B, H, n)),
         "odd": np.where(rng.random((B, H, n)) < 0.1, np.nan, rng.standard_normal((B, H, n))), "short": rng.random((B, H, 200))}[kind]
    w = torch.tensor(w, dtype=torch.float32, device=DEV)
    want = as_oracle(c)
    index, new_lens, kept = cache_evict(c, i32(table), i32(lens), w, i32(out), keep, recent=recent, first=first)
    ri, rl = ko.evict(w.cpu().numpy(), lens, keep, recent, first)
    assert np.array_equal(index.cpu().numpy(), ri) and np.array_equal(new_lens.cpu().numpy(), rl)
    wide = np.pad(w.cpu().numpy(), ((0, 0), (0, 0), (0, max(0, n - w.shape[2]))))
    assert np.array_equal(kept.cpu().numpy(), np.where(ri >= 0, np.take_along_axis(wide, np.maximum(ri, 0), 2), 0), equal_nan=True)
    for b in range(B):   # the kept tokens' bytes in the new pages, zeros behind them
        for block in range(-(-int(rl[b]) // 64)):
            page = out[b, block]
            for h in range(H):
                at = ri[b, h, 64 * block:64 * block + 64]
                at = at[at >= 0]
                source, slot = table[b][at // 64], at % 64
                for name in ("k", "v", "k_scale", "v_scale"):
                    rows = want[name][source, h, slot]
                    want[name][page, h] = 0
                    want[name][page, h, :len(at)] = rows
                want["desc"][page, h, :len(at)] = want["desc"][source, h, slot]
    got = as_oracle(c)
    for name in want:
        assert np.array_equal(got[name], want[name]), name


# ---- together -----------------------------------------------------------------------------------------------------

def test_cache_attention_equals_flash_attention_over_the_same_numbers():
    from kerneldev_b200 import cache_append, cache_attention, cache_read, flash_attention, synthetic
    B, H, T, D = 3, 4, 333, 64
    ins, sid, pre, lens = synthetic.batch_metadata(1, B, T, prefix=(8, 40), context=(64, 160), n_spans=(2, 6), span_len=(8, 40))
    rng = np.random.default_rng(0)
    m = dict(in_span=torch.tensor(ins, device=DEV), span_id=torch.tensor(sid, device=DEV), is_prefix=torch.tensor(pre, device=DEV))
    c = make_cache(20, H, D, metadata=True)
    table = tables(rng, B, 6, 20)
    x = rand_kv(rng, (3, B, H, T, D), torch.bfloat16).to(DEV)
    cache_append(c, x[0], x[1], i32(table), i32([0] * B), i32(lens), **m)
    o, lse = cache_attention(x[2], c, i32(table), i32(lens), i32(lens), return_lse=True)
    k, v = cache_read(c, i32(table), i32(lens), T)   # exact in bfloat16
    fo, fl = flash_attention(x[2], k, v, lens=i32(lens), return_lse=True, **m)
    # the bounds of the same test of the 8-bit cache
    a = flash_attention(x[2], k, v.abs(), lens=i32(lens), **m).float()
    floor = 2.0 ** -33 * v.float().abs().sum(2, keepdim=True)
    assert ((o.float() - fo.float()).abs() <= a * (2.0 ** -11 + 2.0 ** -8) + (o.float().abs() + fo.float().abs()) * 2.0 ** -8 + a * 2.0 ** -8 + floor).all()
    live = torch.isfinite(fl)
    assert torch.equal(live, torch.isfinite(lse)) and ((fl - lse)[live].abs() <= 2e-3).all()


@pytest.mark.parametrize("D,sections", [(64, None), (128, (16, 24, 24))])
def test_generation_with_rotation_and_eviction(D, sections):
    """As a model generates: heads normalised and turned behind what the cache holds, appended, attended to; steps that weigh, an eviction, more steps. Turned heads against their definition,
    what is stored against that of the turned keys, every output against 64 bits on what the cache holds."""
    from kerneldev_b200 import KVCache, Rotation, cache_append, cache_attention, cache_evict, rotate_heads
    rng = np.random.default_rng(12)
    B, H, Hkv = 2, 6, 2
    c = KVCache.empty(24, Hkv, D, device=DEV, bits=4)
    want = as_oracle(c)
    rotation, rot = Rotation(D, base=1e5, sections=sections, device=DEV), ro.rotation(D, base=1e5, sections=sections)
    wq, wk = (torch.tensor(1 + 0.2 * rng.standard_normal(D)).bfloat16().to(DEV) for _ in range(2))
    order = rng.permutation(24)
    table, spare = order[:12].reshape(2, 6), order[12:18].reshape(2, 3)
    lens, seen = np.zeros(B, int), np.zeros(B, int)   # held by the cache; positions so far
    weights = torch.zeros((B, Hkv, 400), device=DEV)
    keep = 100

    def step(n):
        nonlocal lens, seen
        T = max(n)
        x = rand_kv(rng, (2, B, T, Hkv, D), torch.bfloat16).to(DEV).transpose(2, 3)
        q = rand_kv(rng, (B, T, H, D), torch.bfloat16, False).to(DEV).transpose(1, 2)
        at = seen[:, None] + np.arange(T)
        if sections:
            pos = np.stack((at, at // 7, at % 7))
            where = {"positions": torch.tensor(pos, device=DEV)}
        else:
            pos = at[None]
            where = {"offsets": i32(seen)}
        q2, k2 = rotate_heads(q, x[0], rotation, q_weight=wq, k_weight=wk, out_layout="input", **where)
        for y, z, w in ((q2, q, wq), (k2, x[0], wk)):
            exact, size = ro.forward(rot, z.double().cpu().numpy(), pos, w.double().cpu().numpy())
            assert (np.abs(y.double().cpu().numpy() - exact) <= size * 2.0 ** -19 + np.abs(exact) * 2.0 ** -8).all()
        cache_append(c, k2, x[1], i32(table), i32(lens), i32(n))
        k4.append(want, k2.double().cpu().numpy(), x[1].double().cpu().numpy(), table, lens, n)
        assert_cache(c, want)
        lens, seen = lens + np.array(n), seen + np.array(n)
        before = weights.clone()
        got = cache_attention(q2, c, i32(table), i32(lens), i32(n), return_lse=True, weights=weights)
        check_attention(c, q2, table, lens, n, got, weights=weights, before=before)

    step([150, 70])
    for _ in range(3):
        step([1, 1])
    index, new, w = cache_evict(c, i32(table), i32(lens), weights, i32(spare), keep, recent=16, first=4)
    ri, rl = ko.evict(weights.cpu().numpy(), lens, keep, 16, 4)
    assert np.array_equal(index.cpu().numpy(), ri) and np.array_equal(new.cpu().numpy(), rl)
    table, lens, want = spare, rl, as_oracle(c)
    weights = torch.cat([w, torch.zeros((B, Hkv, 100), device=DEV)], 2).contiguous()
    step([3, 2])
    for _ in range(3):
        step([1, 1])


def test_captured_step_follows_lengths_and_pages_on_the_device(monkeypatch):
    """Rotation, append and attention captured once serve every later token: lengths and the table are read at replay. Two graphs, another stream."""
    from kerneldev_b200 import KVCache, Rotation, cache_append, cache_attention, rotate_heads
    monkeypatch.delenv("KD_CHECK_STATUS", raising=False)
    rng = np.random.default_rng(2)
    B, H, Hkv, D = 2, 4, 2, 128
    c, rotation = KVCache.empty(16, Hkv, D, device=DEV, bits=4), Rotation(D, device=DEV)
    table = tables(rng, B, 8, 16)
    t, lens = i32(table), i32([60, 3])
    start = rand_kv(rng, (2, B, Hkv, 60, D), torch.float16).to(DEV)
    cache_append(c, start[0], start[1], t, i32([0, 0]), lens)
    x = torch.zeros((2, B, Hkv, 1, D), dtype=torch.float16, device=DEV)
    q = torch.zeros((B, H, 1, D), dtype=torch.float16, device=DEV)
    w = torch.zeros((B, Hkv, 512), device=DEV)

    def step():
        q2, k2 = rotate_heads(q, x[0], rotation, offsets=lens)
        cache_append(c, k2, x[1], t, lens)
        lens.add_(1)
        return q2, cache_attention(q2, c, t, lens, return_lse=True, weights=w)

    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    n = np.array([60, 3])
    side = torch.cuda.Stream()
    rot = ro.rotation(D)
    for i in range(9):
        x.copy_(rand_kv(rng, (2, B, Hkv, 1, D), torch.float16))
        q.copy_(rand_kv(rng, (B, H, 1, D), torch.float16, False))
        before = w.clone()
        g, (q2, out) = graphs[i % 2]
        if i % 3 == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            g.replay()
        torch.cuda.synchronize()
        exact, size = ro.forward(rot, q.double().cpu().numpy(), n[None, :, None])
        assert (np.abs(q2.double().cpu().numpy() - exact) <= size * 2.0 ** -19 + np.abs(exact) * 2.0 ** -11 + 1e-7).all()
        n = n + 1
        assert lens.tolist() == n.tolist()
        check_attention(c, q2, table, n, [1, 1], out, weights=w, before=before)


def test_results_repeat_bit_for_bit():
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(20)
    for B, H, Hkv, D, T, n in ((1, 8, 2, 128, 1, 5000), (3, 4, 4, 64, 7, 700), (1, 4, 2, 128, 150, 900)):
        c, table = filled(rng, B, Hkv, D, [n] * B, torch.bfloat16, False)
        q = rand_kv(rng, (B, H, T, D), torch.bfloat16, False).to(DEV)
        outs = []
        for _ in range(4):
            w = torch.zeros((B, Hkv, n), device=DEV)
            outs.append((*cache_attention(q, c, i32(table), i32([n] * B), return_lse=True, weights=w), w))
        for other in outs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("T", [1, 40])
def test_two_graphs_of_one_cache_replayed_on_two_streams(T):
    """Each has a workspace of its own, though both run at once."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(50 + T)
    lens = [3000, 900]
    c, table = filled(rng, 2, 2, 128, lens, torch.float16, False)
    t, n = i32(table), i32(lens)
    streams, graphs, qs, outs = [torch.cuda.Stream() for _ in range(2)], [], [], []
    for i in range(2):
        q = rand_kv(rng, (2, 8, T, 128), torch.float16, False).to(DEV)
        cache_attention(q, c, t, n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        w = torch.zeros((2, 2, 3000), device=DEV)
        with torch.cuda.graph(g, stream=streams[i]):
            w.zero_()
            outs.append((cache_attention(q, c, t, n, return_lse=True, weights=w), w))
        graphs.append(g)
        qs.append(q)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for q, (got, w) in zip(qs, outs):
        check_attention(c, q, table, lens, [T, T], got, weights=w)


# ---- what is refused ----------------------------------------------------------------------------------------------

def test_refusals():
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    c = KVCache.empty(4, 2, 64, device=DEV, bits=4)
    q, k = torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device=DEV)
    t, n = i32([[0, 1]]), i32([5])
    bad = [
        lambda: cache_attention(q.float(), c, t, n), lambda: cache_attention(q[:, :3], c, t, n), lambda: cache_attention(q[..., :48], c, t, n), lambda: cache_attention(q[..., :32], c, t, n),
        lambda: cache_append(c, k[..., :32], k[..., :32], t, n), lambda: cache_append(c, k.double(), k.double(), t, n), lambda: cache_append(c, k[:, :1], k[:, :1], t, n),
        lambda: KVCache(c.k, c.v.view(torch.float8_e4m3fn), c.k_scale, c.v_scale), lambda: KVCache(c.k[..., :20], c.v[..., :20], c.k_scale, c.v_scale),
        lambda: KVCache(c.k, c.v, c.k_scale[..., :3], c.v_scale), lambda: KVCache(c.k, c.v, c.k_scale.float(), c.v_scale), lambda: KVCache(c.k, c.v, torch.ones((4, 2), device=DEV), c.v_scale),
        lambda: KVCache(c.k, c.v, c.k_scale.transpose(1, 2).contiguous().transpose(1, 2), c.v_scale), lambda: KVCache(c.k[:, :, ::2], c.v[:, :, ::2], c.k_scale, c.v_scale),
        lambda: KVCache.empty(4, 2, 72, device=DEV, bits=4), lambda: KVCache.empty(4, 2, 144, device=DEV, bits=4), lambda: KVCache.empty(0, 2, 64, device=DEV, bits=4),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    odd = torch.zeros(c.k_scale.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(c.k_scale.shape)
    with pytest.raises(ValueError, match="aligned"):
        KVCache(c.k, c.v, odd, c.v_scale)
    with pytest.raises(RuntimeError, match="no_grad"):
        cache_attention(q.clone().requires_grad_(), c, t, n)


def test_bad_lengths_and_pages_are_reported_and_left_out():
    """The tables and lengths of these calls are wrong on purpose; the kernels check every one of them before they form an address."""
    from kerneldev_b200 import cache_append, cache_attention, cache_evict, cache_read
    rng = np.random.default_rng(1)
    c, table = filled(rng, 2, 2, 64, [200, 100], torch.bfloat16, False)
    q = rand_kv(rng, (2, 4, 1, 64), torch.bfloat16, False).to(DEV)
    x = rand_kv(rng, (2, 2, 2, 3, 64), torch.bfloat16).to(DEV)
    w = torch.zeros((2, 2, 300), device=DEV)
    wrong = table.copy()
    wrong[0, 1] = c.k.shape[0]
    wrong[1, 0] = -1
    before = as_oracle(c)
    with pytest.raises(ValueError, match="page number"):
        cache_attention(q, c, i32(wrong), i32([200, 100]), weights=w)
    with pytest.raises(ValueError, match="page number"):
        cache_read(c, i32(wrong), i32([200, 100]), 200)
    with pytest.raises(ValueError, match="page number"):
        cache_attention(q.expand(2, 4, 1, 64).repeat(1, 10, 1, 1), c, i32(wrong), i32([200, 100]))
    with pytest.raises(ValueError, match="length"):
        cache_attention(q, c, i32(table), i32([257, -1]), weights=w)
    with pytest.raises(ValueError, match="length"):
        cache_read(c, i32(table), i32([2 ** 31 - 1, 100]), 200)
    with pytest.raises(ValueError, match="page number"):
        cache_evict(c, i32(table), i32([200, 100]), w, i32([[-5], [2 ** 31 - 1]]), 64)
    with pytest.raises(ValueError, match="page number"):
        cache_append(c, x[0], x[1], i32(wrong), i32([100, 50]))
    with pytest.raises(ValueError, match="length"):
        cache_append(c, x[0], x[1], i32(table), i32([256, 256]))
    with pytest.raises(ValueError, match="length"):
        cache_append(c, x[0], x[1], i32(table), i32([-3, 5]), i32([4, -1]))
    after = as_oracle(c)
    assert all(np.array_equal(before[n], after[n]) for n in ("k", "v", "k_scale", "v_scale"))
    got = cache_attention(q, c, i32(table), i32([200, 100]), return_lse=True)
    check_attention(c, q, table, [200, 100], [1, 1], got)


def test_empty_calls():
    from kerneldev_b200 import KVCache, cache_append, cache_attention, cache_evict, cache_read
    c = KVCache.empty(4, 2, 64, device=DEV, bits=4)
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    none = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    assert cache_attention(z(0, 4, 1, 64), c, none, i32([])).shape == (0, 4, 1, 64)
    cache_append(c, z(1, 2, 0, 64), z(1, 2, 0, 64), i32([[1]]), i32([5]))
    cache_append(c, z(0, 2, 1, 64), z(0, 2, 1, 64), none, i32([]))
    assert cache_read(c, i32([[1]]), i32([5]), 0)[0].shape == (1, 2, 0, 64)
    empty = torch.zeros((2, 0), dtype=torch.int32, device=DEV)
    o, lse = cache_attention(z(2, 4, 1, 64), c, empty, i32([0, 0]), return_lse=True)
    assert not o.any() and torch.isinf(lse).all()
    index, lens, w = cache_evict(c, empty, i32([0, 0]), torch.zeros((2, 2, 0), device=DEV), i32([[1], [2]]), 3)
    assert (index == -1).all() and not lens.any() and not w.any()


def test_offsets_beyond_32_bits():
    """A pool of more than 2**32 bytes: the last pages are reached."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    free, _ = torch.cuda.mem_get_info()
    H, D = 8, 128
    pages = (1 << 32) // (H * 64 * D // 2) + 40
    if free < 3 * pages * H * 64 * D:
        pytest.skip("needs 26 GB")
    rng = np.random.default_rng(0)
    c = KVCache.empty(pages, H, D, device=DEV, bits=4)
    table = np.array([[pages - 1, pages - 33, 5, pages - 7]])
    x = rand_kv(rng, (2, 1, H, 230, D), torch.bfloat16).to(DEV)
    cache_append(c, x[0], x[1], i32(table), i32([0]))
    used = torch.tensor(table[0], device=DEV)
    small = KVCache(*(t[used] for t in (c.k, c.v, c.k_scale, c.v_scale)))
    for T in (1, 20):
        q = rand_kv(rng, (1, 2 * H, T, D), torch.bfloat16, False).to(DEV)
        check_attention(small, q, np.array([[0, 1, 2, 3]]), [230], [T], cache_attention(q, c, i32(table), i32([230]), return_lse=True))


@pytest.mark.parametrize("drop", [5, 6, 7, 8], ids=["K", "V", "S", "PV"])
def test_wait_timeout_in_the_attention_of_many_rows(drop):
    """As for the 8-bit cache: waits that run out end the launch, the next call raises, and the device is usable and correct."""
    from kerneldev_b200.build import build
    from tests.test_gpu_timeout import CHILD_CACHE, ROOT, WAITTEST_FLAGS
    lib = build(name="waittest", extra_flags=WAITTEST_FLAGS)
    env = dict(os.environ, KD_LIB_PATH=str(lib))
    env.pop("KD_CHECK_STATUS", None)
    child = (CHILD_CACHE % {"root": ROOT, "D": 128, "drop": drop}).replace("KVCache.empty(12, 2, D, device=dev)", "KVCache.empty(12, 2, D, device=dev, metadata=True, bits=4)")
    assert "bits=4" in child
    r = subprocess.run([sys.executable, "-c", child], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "unwound and recovered" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.parametrize("B,Hkv,G,T", [(2, 2, 3, 1), (2, 1, 8, 3), (40, 8, 1, 1), (2, 2, 2, 40), (40, 4, 1, 40)])
@pytest.mark.parametrize("weigh", [False, True], ids=["plain", "weigh"])
def test_share_whose_visible_keys_are_all_nan(B, Hkv, G, T, weigh):
    """All keys of a run of pages are NaN: no row that sees them has a number, whichever CTA's share they are."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(B + T)
    lens = rng.integers(1200, 1900, B)
    c, table = filled(rng, B, Hkv, 64, lens, torch.bfloat16, False)
    q = rand_kv(rng, (B, Hkv * G, T, 64), torch.bfloat16, False).to(DEV)
    clean = cache_attention(q, c, i32(table), i32(lens), return_lse=True)
    b, blocks = B - 1, -(-int(lens[B - 1]) // 64)
    for first in (0, blocks // 2, blocks - 8):
        pages = table[b, first:first + 7]
        old = c.k_scale[pages, Hkv - 1].clone()
        c.k_scale[pages, Hkv - 1] = 0xFF
        w = torch.zeros((B, Hkv, 1900), device=DEV) if weigh else None
        o, lse = cache_attention(q, c, i32(table), i32(lens), return_lse=True, weights=w)
        c.k_scale[pages, Hkv - 1] = old
        hit = torch.zeros(lse.shape, dtype=torch.bool, device=DEV)
        hit[b, (Hkv - 1) * G:] = True
        assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(o[~hit], clean[0][~hit]) and torch.equal(lse[~hit], clean[1][~hit])
        if weigh:
            assert torch.isnan(w[b, Hkv - 1, :int(lens[b]) - T + 1]).all() and torch.isfinite(w[b, :Hkv - 1]).all() and torch.isfinite(w[:b]).all()


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("G,T", [(3, 1), (4, 3), (2, 40)])
def test_nan_of_single_groups_at_every_head_dim(D, G, T):
    """Groups of values that are NaN, in tokens that some rows see and others do not: their columns are NaN in the rows that see them, all else is as without them."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(D + T)
    B, n = 2, 900
    c, table = filled(rng, B, 1, D, [n, n], torch.bfloat16, False)
    q = rand_kv(rng, (B, G, T, D), torch.bfloat16, False).to(DEV)
    clean = cache_attention(q, c, i32(table), i32([n, n]), return_lse=True)
    nan = torch.zeros((B, T, D), dtype=torch.bool, device=DEV)
    for b in range(B):
        for g in range(b, D // 16, 2):
            at = n - 1 - int(rng.integers(T)) if g % 2 else int(rng.integers(n))
            c.v_scale[table[b, at // 64], 0, at % 64, g] = 0xFF
            nan[b, max(at - (n - T), 0):, 16 * g:16 * g + 16] = True
    o, lse = cache_attention(q, c, i32(table), i32([n, n]), return_lse=True)
    nan = nan[:, None].expand(B, G, T, D)
    assert torch.isnan(o[nan]).all() and torch.isfinite(o[~nan]).all() and torch.equal(lse, clean[1])
    assert torch.equal(o[~nan], clean[0][~nan])   # a column's NaN took the place of a number: the others are sums of the same products
