"""The 8-bit key/value cache on the GPU against its definition in 64 bits (oracle/kv_cache_oracle.py).

Tolerances, derived before the first run. Bytes, scales, descriptors and indices are equal. Attention: a probability is rounded
to a half (2**-11), the output to its type (eps / 2); scores are sums of exact products in 32 bits, off by some 2**-21 of the sum of
magnitudes (32-bit sums of up to 128 terms in an order of the hardware's), which is a relative error of the probabilities, as is 2**-21 of the
exponential; sums over n tokens in 32 bits add n * 2**-24 at most."""
import os

import numpy as np
import pytest
import torch

from oracle import kv_cache_oracle as ko

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def make_cache(pages, H, D, metadata=False, fill=0x7F):
    """A cache whose pages hold NaN bytes and odd scales before anything is appended."""
    from kerneldev_b200 import KVCache
    c = KVCache.empty(pages, H, D, device=DEV, metadata=metadata)
    c.k.view(torch.uint8).fill_(fill)
    c.v.view(torch.uint8).fill_(fill)
    c.k_scale.fill_(2.0 ** 31)
    c.v_scale.fill_(2.0 ** 31)
    return c


def as_oracle(c):
    wide = lambda t: t.float().cpu().double().numpy()  # noqa: E731
    return {"k": wide(c.k), "v": wide(c.v), "k_scale": wide(c.k_scale), "v_scale": wide(c.v_scale),
            "desc": None if c.desc is None else c.desc.cpu().numpy().astype(np.int64) & 0xFFFFFFFF}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def tables(rng, B, blocks, pages):
    return rng.permutation(pages)[:B * blocks].reshape(B, blocks)


def rand_kv(rng, shape, dtype, outliers=True):
    x = rng.standard_normal(shape) * np.exp(0.7 * rng.standard_normal(shape[:-2] + (1, shape[-1])))
    if outliers:
        x = np.where(rng.random(shape) < 0.01, x * 30, x)
    return torch.tensor(x).to(dtype)


def strided(t, layout):
    """The values of a (B, H, T, D) tensor in another memory order."""
    if layout == "bthd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":   # rows that are not 16-byte aligned
        B, H, T, D = t.shape
        wide = torch.zeros((B, H, T, D + 3), dtype=t.dtype, device=t.device)
        wide[..., 1:D + 1] = t
        return wide[..., 1:D + 1]
    if layout == "dlast":   # head dim not the fastest
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    return t.contiguous()


def metadata(rng, B, T):
    ins = rng.random((B, T)) < 0.35
    sid = np.where(ins, rng.integers(0, 4, (B, T)), 0)
    sid[rng.random((B, T)) < 0.05] = -1
    pre = rng.random((B, T)) < 0.2
    return ins, sid, pre


def same(a, b):
    return np.array_equal(np.nan_to_num(a, nan=1e300), np.nan_to_num(b, nan=1e300))


def assert_cache(c, want):
    got = as_oracle(c)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert same(got[name], want[name]), name
    if want["desc"] is not None:
        assert np.array_equal(got["desc"], want["desc"])


# ---- appending and reading ----------------------------------------------------------------------------------------

APPENDS = [
    # D, H, type, layout, lens, new tokens
    (64, 2, "bf16", "bhtd", [0, 1, 63, 64, 65, 200], [1, 1, 1, 1, 1, 1]),
    (128, 3, "f16", "bthd", [0, 5, 60, 128], [130, 64, 4, 0]),
    (16, 1, "f32", "odd", [7, 0], [3, 66]),
    (80, 2, "bf16", "dlast", [31, 64], [100, 129]),
    (112, 1, "f32", "bhtd", [0, 63], [64, 2]),
    (48, 5, "f16", "odd", [190], [1]),
]


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
        ko.append(want, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, start, count, ko.descriptors(*m))
        assert_cache(c, want)
    total = np.array(lens) + np.array(new)
    start = np.maximum(total - 70, 0)
    for out in (torch.bfloat16, torch.float32):
        k, v = cache_read(c, i32(table), i32(total), 75, start=i32(start), dtype=out)
        for b in range(B):
            for h in range(H):
                for got, name in ((k, "k"), (v, "v")):
                    x = np.zeros((75, D))
                    held = ko.values(want, table[b], int(total[b]), h, name)[start[b]:]
                    x[:len(held)] = held
                    assert np.array_equal(got[b, h].double().cpu().numpy(), x)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_one_by_one_lets_the_scale_grow(dtype):
    """Magnitudes that double from token to token: every append moves what is there to a coarser grid, down into the subnormals."""
    from kerneldev_b200 import cache_append
    rng = np.random.default_rng(3)
    c = make_cache(3, 2, 32)
    want, table = as_oracle(c), np.array([[2, 0]])
    for t in range(90):
        x = (rng.standard_normal((2, 1, 2, 1, 32)) * 2.0 ** min(t - 20 if dtype != "f16" else t / 4 - 8, 12))
        x = torch.tensor(x).to(DT[dtype]).to(DEV)
        cache_append(c, x[0], x[1], i32(table), i32([t]))
        ko.append(want, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, [t], [1])
        assert_cache(c, want)


def test_append_numbers_without_a_place():
    """Infinities, NaN, numbers beyond the largest scale, numbers below the smallest, zeros of both signs."""
    from kerneldev_b200 import cache_append
    c = make_cache(2, 1, 16)
    x = torch.zeros((1, 1, 66, 16))
    x[0, 0, 0, :5] = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0, -0.0])
    x[0, 0, 64, :4] = torch.tensor([1e30, -1e30, 1.0, 1e-45])
    y = torch.zeros((1, 1, 66, 16))
    y[0, 0, 0, :3] = torch.tensor([2.0 ** -41, 1.5 * 2.0 ** -41, 2.0 ** -44])
    y[0, 0, 64:] = float("nan")
    want, table = as_oracle(c), np.array([[0, 1]])
    cache_append(c, x.to(DEV), y.to(DEV), i32(table), i32([0]))
    ko.append(want, x.double().numpy(), y.double().numpy(), table, [0], [66])
    assert_cache(c, want)
    assert c.k_scale.tolist() == [[2.0 ** -7], [2.0 ** 31]] and c.v_scale.tolist() == [[2.0 ** -32], [2.0 ** -32]]


def test_roll_back_and_append_again():
    """A shorter length given back (drafted tokens that were refused): what lies behind it is overwritten."""
    from kerneldev_b200 import cache_append
    rng = np.random.default_rng(5)
    c = make_cache(4, 2, 64)
    want, table = as_oracle(c), np.array([[1, 3, 0]])
    for start, n, scale in ((0, 100, 1.0), (100, 7, 50.0), (101, 3, 1.0), (64, 5, 0.1), (20, 60, 0.01)):
        x = (rand_kv(rng, (2, 1, 2, n, 64), torch.float32) * scale).to(DEV)
        cache_append(c, x[0], x[1], i32(table), i32([start]))
        ko.append(want, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, [start], [n])
        assert_cache(c, want)


# ---- attention ----------------------------------------------------------------------------------------------------

def filled(rng, B, H, D, lens, dtype, meta):
    from kerneldev_b200 import cache_append
    blocks = max(-(-int(max(lens)) // 64), 1)
    pages = B * blocks + 2
    c = make_cache(pages, H, D, metadata=meta)
    table = tables(rng, B, blocks, pages)
    T = max(int(max(lens)), 1)
    x = rand_kv(rng, (2, B, H, T, D), dtype).to(DEV)
    m = metadata(rng, B, T)
    extra = dict(zip(("in_span", "span_id", "is_prefix"), (torch.tensor(t, device=DEV) for t in m))) if meta else {}
    cache_append(c, x[0], x[1], i32(table), i32(np.zeros(B)), i32(lens), **extra)
    return c, table


def check_attention(c, q, table, lens, q_lens, got, causal=True, scale=None, weights=None, before=None):
    D = q.shape[3]
    dtype = q.dtype
    o, lse = got
    scale = D ** -0.5 if scale is None else scale
    ro, rl, rw, a, mag = ko.attention(as_oracle(c), q.cpu().double().numpy(), table, lens, q_lens, scale, causal)
    n = max(int(max(lens)), 1)
    delta = 2.0 ** -21 * (mag * 1.5 + 2) + n * 2.0 ** -24
    err = np.abs(o.double().cpu().numpy() - ro)
    tol = torch.finfo(dtype).eps / 2 * (np.abs(ro) + 0.01 * a) + a * (2.0 ** -11 + 2 * delta[..., None]) + 2.0 ** -25
    assert np.isfinite(o.double().cpu().numpy()).all()
    assert (err <= tol).all(), f"O: {(err / tol).max()} of the tolerance at {np.unravel_index((err / tol).argmax(), err.shape)}"
    l = lse.double().cpu().numpy()
    assert np.array_equal(np.isinf(l), np.isinf(rl)) and (l[np.isinf(l)] < 0).all()
    fin = np.isfinite(rl)
    assert (np.abs(l[fin] - rl[fin]) <= (2 * delta)[fin] + 2.0 ** -22 * np.abs(rl[fin])).all(), "LSE"
    if weights is not None:
        w = weights.double().cpu().numpy() - (0 if before is None else before.double().cpu().numpy())
        rw = np.pad(rw, ((0, 0), (0, 0), (0, max(0, w.shape[2] - rw.shape[2]))))[..., :w.shape[2]]
        size = np.abs(rw) if before is None else np.abs(rw) + np.abs(before.double().cpu().numpy())
        G, rows = q.shape[1] // rw.shape[1], q.shape[1] // rw.shape[1] * q.shape[2]
        top = delta.reshape(rw.shape[0], rw.shape[1], G, -1).max((2, 3))[..., None]
        assert (np.abs(w - rw) <= rw * 3 * top + size * rows * 2.0 ** -24 + 1e-30).all(), "weights"


ATTENTION = [
    # B, H, Hkv, D, T, type, mask, layout, lens, q_lens
    (6, 4, 2, 64, 1, "bf16", "causal", "bthd", [1, 63, 64, 65, 200, 0], None),
    (3, 8, 1, 128, 1, "f16", "causal", "bhtd", [300, 129, 1], None),
    (2, 16, 16, 64, 1, "bf16", "hier", "bthd", [173, 64], None),
    (2, 40, 2, 128, 1, "bf16", "causal", "bhtd", [130, 700], None),
    (3, 6, 2, 80, 5, "f16", "hier", "bthd", [5, 133, 260], [5, 2, 0]),
    (2, 3, 3, 16, 3, "f16", "full", "odd", [3, 70], [3, 1]),
    (2, 4, 4, 48, 9, "bf16", "hier", "dlast", [64, 191], None),
    (1, 5, 1, 112, 2, "bf16", "causal", "bhtd", [1029], None),
    (2, 2, 1, 32, 33, "f16", "causal", "bthd", [33, 97], [33, 20]),
    (2, 12, 4, 96, 17, "bf16", "hier", "bhtd", [17, 450], [16, 17]),
    (1, 8, 2, 128, 130, "bf16", "causal", "bthd", [333], None),
    (2, 4, 2, 64, 200, "f16", "hier", "bthd", [200, 515], [131, 200]),
    (1, 4, 4, 128, 70, "f16", "full", "bhtd", [64], [64]),
    (2, 6, 2, 112, 65, "bf16", "causal", "bhtd", [3, 640], [65, 65]),   # more queries than tokens: those before the first see nothing
]


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
    if layout == "bthd" and B > 1 and T > 1:
        assert o2.stride() == q.stride()


@pytest.mark.parametrize("T,G", [(1, 4), (6, 3), (80, 2)])
def test_attention_does_not_read_what_is_masked(T, G):
    """NaN and infinities in keys and values that a query does not see, and behind the sequences, reach nothing; those that it sees do."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    rng = np.random.default_rng(8)
    B, Hkv, D, n = 2, 2, 64, 330
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
    # a value that a query does see: NaN in its column alone
    c2 = KVCache(c.k.clone(), c.v.clone(), c.k_scale, c.v_scale)   # without metadata, causal: the spans are seen
    v = c2.v.view(torch.uint8)
    c2.k.view(torch.uint8)[(c2.k.view(torch.uint8) & 0x7F) == 0x7F] = 0
    v[(v & 0x7F) == 0x7F] = 0
    v[table[0, 2], :, 9, 3] = 0xFF
    o, lse = cache_attention(q, c2, i32(table), i32(lens), return_lse=True)
    assert torch.isfinite(lse).all() and torch.isfinite(o[1]).all()
    assert torch.isnan(o[0, ..., 3]).all() and torch.isfinite(o[0, ..., :3]).all() and torch.isfinite(o[0, ..., 4:]).all()


@pytest.mark.parametrize("B,Hkv,G,T,D,meta", [(70, 2, 2, 1, 64, True), (300, 1, 8, 1, 32, False), (140, 4, 1, 3, 48, True), (300, 8, 1, 1, 16, False), (40, 8, 5, 8, 64, False),
                                              (7, 1, 12, 3, 128, True)])
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


def test_attention_scales_far_apart():
    """Blocks whose scales lie 2**40 apart, keys that make scores of hundreds, a block of zeros."""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(4)
    c = make_cache(6, 1, 32)
    table, n = np.array([[4, 1, 0, 5, 2]]), 300
    x = rand_kv(rng, (2, 1, 1, n, 32), torch.float32, False)
    x[1, :, :, :64] *= 2.0 ** 20
    x[1, :, :, 64:128] *= 2.0 ** -20
    x[1, :, :, 128:192] = 0
    x[0, :, :, 64:128] *= 100
    cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32([0]))
    q = (rand_kv(rng, (1, 3, 4, 32), torch.float32, False) * 3).to(torch.float16).to(DEV)
    check_attention(c, q, table, [n], [4], cache_attention(q, c, i32(table), i32([n]), return_lse=True, sm_scale=0.5), scale=0.5)


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


# ---- eviction -----------------------------------------------------------------------------------------------------

EVICTIONS = [
    # H, D, lens, keep, recent, first, weights
    (2, 64, [1000, 300, 128, 100, 0, 1], 128, 32, 4, "spread"),
    (1, 128, [130, 2100], 65, 0, 0, "ties"),
    (3, 16, [500], 499, 499, 0, "spread"),
    (2, 80, [5000, 64], 1, 1, 0, "spread"),
    (1, 48, [700], 64, 10, 20, "zeros"),
    (2, 96, [900, 901], 200, 0, 3, "odd"),
    (1, 32, [300], 100, 0, 0, "short"),
    (2, 16, [4096, 4097, 9000], 1000, 100, 1, "ties"),       # one CTA of 256 threads, and clusters
    (1, 16, [40000, 3], 30000, 5, 0, "spread"),              # clusters of larger CTAs
    (1, 16, [131072 + 700], 70000, 64, 64, "ties"),          # keys beyond what stays in registers
    (2, 16, [9000, 100, 5000], 5000, 3000, 2000, "spread"),  # clusters that have nothing to search for
]


@pytest.mark.parametrize("case", EVICTIONS, ids=lambda c: f"d{c[1]}-keep{c[3]}-{c[6]}")
def test_evict(case):
    from kerneldev_b200 import cache_evict, cache_read
    H, D, lens, keep, recent, first, kind = case
    rng = np.random.default_rng(keep)
    B, n = len(lens), max(lens)
    c, table = filled(rng, B, H, D, lens, torch.bfloat16, True)
    out_blocks = -(-keep // 64)
    pages = c.k.shape[0]
    from kerneldev_b200 import KVCache
    grow = lambda t, x: torch.cat([t.view(torch.uint8), torch.full((B * out_blocks + 1,) + t.shape[1:], x, dtype=torch.uint8, device=DEV)]).view(torch.float8_e4m3fn)  # noqa: E731
    more = lambda t: torch.cat([t, torch.ones((B * out_blocks + 1,) + t.shape[1:], dtype=t.dtype, device=DEV)])  # noqa: E731
    c = KVCache(grow(c.k, 0x7F), grow(c.v, 0x7F), more(c.k_scale), more(c.v_scale), more(c.desc))
    out = pages + rng.permutation(B * out_blocks + 1)[:B * out_blocks].reshape(B, out_blocks)
    w = {"spread": np.exp(2 * rng.standard_normal((B, H, n))), "ties": rng.integers(0, 3, (B, H, n)) * 0.5, "zeros": np.zeros((B, H, n)),
         "odd": np.where(rng.random((B, H, n)) < 0.1, np.nan, rng.standard_normal((B, H, n))), "short": rng.random((B, H, 200))}[kind]
    if kind == "odd":
        w[:, :, 50], w[:, :, 60], w[:, :, 70:75], w[:, :, 80] = np.inf, -np.inf, -0.0, 1e-42
    w = torch.tensor(w, dtype=torch.float32, device=DEV)
    before = as_oracle(c)
    index, new_lens, kept = cache_evict(c, i32(table), i32(lens), w, i32(out), keep, recent=recent, first=first)
    ri, rl = ko.evict(w.cpu().numpy(), lens, keep, recent, first)
    assert np.array_equal(index.cpu().numpy(), ri) and np.array_equal(new_lens.cpu().numpy(), rl)
    wide = np.pad(w.cpu().numpy(), ((0, 0), (0, 0), (0, max(0, n - w.shape[2]))))
    rw = np.where(ri >= 0, np.take_along_axis(wide, np.maximum(ri, 0), 2), 0)
    assert np.array_equal(kept.cpu().numpy(), rw, equal_nan=True)
    # as if the kept tokens had been appended to the new pages
    want = {k: v.copy() for k, v in before.items()}
    T = max(int(rl.max()), 1)
    kv, desc = np.zeros((2, B, H, T, D)), np.zeros((B, H, T), np.int64)
    for b in range(B):
        for h in range(H):
            at = ri[b, h][ri[b, h] >= 0]
            d = np.concatenate([before["desc"][p, h] for p in table[b]])
            desc[b, h, :len(at)] = d[at]
            for i, name in enumerate(("k", "v")):
                kv[i, b, h, :len(at)] = ko.values(before, table[b], int(lens[b]), h, name)[at]
    for h in range(H):
        one = {x: (want[x][:, h:h + 1] if want[x] is not None else None) for x in want}
        ko.append(one, kv[0][:, h:h + 1], kv[1][:, h:h + 1], out, np.zeros(B, int), rl, desc[:, h])
    assert_cache(c, want)
    k, v = cache_read(c, i32(out), new_lens, keep, dtype=torch.float32)
    assert np.isfinite(k.cpu().numpy()).all() and np.isfinite(v.cpu().numpy()).all()


# ---- together -----------------------------------------------------------------------------------------------------

def test_cache_attention_equals_flash_attention_over_the_same_numbers():
    """The whole sequence as queries over its cached keys and values is flash_attention of those numbers, metadata and all."""
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
    k, v = cache_read(c, i32(table), i32(lens), T)
    fo, fl = flash_attention(x[2], k, v, lens=i32(lens), return_lse=True, **m)
    # both round probabilities (to a half, to bfloat16) and outputs: 2**-11 + 2**-8 of sum p |v| and two output roundings, |v| < 4 sigma * 30
    a = flash_attention(x[2], k, v.abs(), lens=i32(lens), **m).float()
    # a half has no steps below 2**-24, and probabilities are rounded in units of at least 2**-8 of the row's largest: of a token with less than 2**-14 / 2**8
    # of it up to 2**-25 / 2**8 = 2**-33 is lost, whatever the row's output is (here 3e-10 where the one heavy token's value is 0)
    floor = 2.0 ** -33 * v.float().abs().sum(2, keepdim=True)
    assert ((o.float() - fo.float()).abs() <= a * (2.0 ** -11 + 2.0 ** -8) + (o.float().abs() + fo.float().abs()) * 2.0 ** -8 + a * 2.0 ** -8 + floor).all()
    live = torch.isfinite(fl)
    assert torch.equal(live, torch.isfinite(lse)) and ((fl - lse)[live].abs() <= 2e-3).all()


def test_generation_with_eviction():
    """Prompt, steps that weigh, an eviction, more steps: every output against 64 bits on what the cache holds."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention, cache_evict
    rng = np.random.default_rng(12)
    B, H, Hkv, D = 2, 6, 2, 64
    c = KVCache.empty(24, Hkv, D, device=DEV)
    order = rng.permutation(24)
    table, spare = order[:12].reshape(2, 6), order[12:18].reshape(2, 3)
    lens = np.zeros(B, int)
    weights = torch.zeros((B, Hkv, 400), device=DEV)
    keep = 100

    def step(n):
        nonlocal lens
        T = max(n)
        x = rand_kv(rng, (2, B, Hkv, T, D), torch.bfloat16).to(DEV)
        q = rand_kv(rng, (B, H, T, D), torch.bfloat16, False).to(DEV)
        cache_append(c, x[0], x[1], i32(table), i32(lens), i32(n))
        lens = lens + np.array(n)
        before = weights.clone()
        got = cache_attention(q, c, i32(table), i32(lens), i32(n), return_lse=True, weights=weights)
        check_attention(c, q, table, lens, n, got, weights=weights, before=before)

    step([150, 70])
    for _ in range(3):
        step([1, 1])
    index, new, w = cache_evict(c, i32(table), i32(lens), weights, i32(spare), keep, recent=16, first=4)
    ri, rl = ko.evict(weights.cpu().numpy(), lens, keep, 16, 4)
    assert np.array_equal(index.cpu().numpy(), ri) and np.array_equal(new.cpu().numpy(), rl)
    table, lens = spare, rl
    weights = torch.cat([w, torch.zeros((B, Hkv, 100), device=DEV)], 2).contiguous()
    step([3, 2])
    for _ in range(3):
        step([1, 1])


def test_captured_step_follows_lengths_and_pages_on_the_device(monkeypatch):
    """A step captured once serves every later token: lengths and the table are read at replay. Two graphs, another stream."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    monkeypatch.delenv("KD_CHECK_STATUS", raising=False)
    rng = np.random.default_rng(2)
    B, H, Hkv, D = 2, 4, 2, 128
    c = KVCache.empty(16, Hkv, D, device=DEV)
    table = tables(rng, B, 8, 16)
    t, lens = i32(table), i32([60, 3])
    start = rand_kv(rng, (2, B, Hkv, 60, D), torch.float16).to(DEV)
    cache_append(c, start[0], start[1], t, i32([0, 0]), lens)
    x = torch.zeros((2, B, Hkv, 1, D), dtype=torch.float16, device=DEV)
    q = torch.zeros((B, H, 1, D), dtype=torch.float16, device=DEV)
    w = torch.zeros((B, Hkv, 512), device=DEV)

    def step():
        cache_append(c, x[0], x[1], t, lens)
        lens.add_(1)
        return cache_attention(q, c, t, lens, return_lse=True, weights=w)

    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    n = np.array([60, 3])
    side = torch.cuda.Stream()
    for i in range(9):
        x.copy_(rand_kv(rng, (2, B, Hkv, 1, D), torch.float16))
        q.copy_(rand_kv(rng, (B, H, 1, D), torch.float16, False))
        before = w.clone()
        g, out = graphs[i % 2]
        if i % 3 == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            g.replay()
        torch.cuda.synchronize()
        n = n + 1
        assert lens.tolist() == n.tolist()
        check_attention(c, q, table, n, [1, 1], out, weights=w, before=before)


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


# ---- what is refused ----------------------------------------------------------------------------------------------

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
    with pytest.raises(ValueError, match="length"):
        cache_attention(q, c, i32(table), i32([257, -1]), weights=w)
    with pytest.raises(ValueError, match="length"):
        cache_attention(q, c, i32(table), i32([200, 100]), i32([2, 1]))
    with pytest.raises(ValueError, match="length"):
        cache_read(c, i32(table), i32([2 ** 31 - 1, 100]), 200)
    with pytest.raises(ValueError, match="page number"):
        cache_evict(c, i32(table), i32([200, 100]), w, i32([[-5], [2 ** 31 - 1]]), 64)
    with pytest.raises(ValueError, match="length"):
        cache_append(c, x[0], x[1], i32(table), i32([256, 256]))
    with pytest.raises(ValueError, match="length"):
        cache_append(c, x[0], x[1], i32(table), i32([-3, 5]), i32([4, -1]))
    assert as_oracle(c)["k"].shape == before["k"].shape
    # a later call is well
    o, lse = cache_attention(q, c, i32(table), i32([200, 100]), return_lse=True)
    check_attention(c, q, table, [200, 100], [1, 1], (o, lse))


def test_refusals():
    from kerneldev_b200 import KVCache, cache_append, cache_attention, cache_evict, cache_read
    c = KVCache.empty(4, 2, 64, device=DEV)
    q, k = torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device=DEV)
    t, n = i32([[0, 1]]), i32([5])
    w = torch.zeros((1, 2, 128), device=DEV)
    bad = [
        lambda: cache_attention(q.float(), c, t, n), lambda: cache_attention(q[0], c, t, n), lambda: cache_attention(q[:, :3], c, t, n),
        lambda: cache_attention(q[..., :48], c, t, n), lambda: cache_attention(q, c, t.long(), n), lambda: cache_attention(q, c, t, n.long()),
        lambda: cache_attention(q, c, t, i32([1, 2])), lambda: cache_attention(q, c, t[0], n), lambda: cache_attention(q, c, t.cpu(), n),
        lambda: cache_attention(q, c, t, n.cpu()), lambda: cache_attention(q, c, t, n, sm_scale=0.0), lambda: cache_attention(q, c, t, n, sm_scale=float("nan")),
        lambda: cache_attention(q, c, t, n, weights=w.half()), lambda: cache_attention(q, c, t, n, weights=w[:, :1]),
        lambda: cache_attention(q, c, t, n, weights=w[:, :, ::2]), lambda: cache_attention(q, c, t, n, weights=w[:, :1].expand(1, 2, 128)),
        lambda: cache_attention(q, c, t, n, out_layout="heads"),
        lambda: cache_append(c, k, k[:, :1], t, n), lambda: cache_append(c, k, k.half(), t, n), lambda: cache_append(c, k.double(), k.double(), t, n),
        lambda: cache_append(c, k, k, t, n, in_span=torch.zeros((1, 3), dtype=torch.bool, device=DEV)), lambda: cache_append(c, k, k, t, n, i32([1, 1])),
        lambda: cache_evict(c, t, n, w, i32([[2]]), 65), lambda: cache_evict(c, t, n, w, i32([[2]]), 0), lambda: cache_evict(c, t, n, w, i32([[2]]), 10, recent=8, first=3),
        lambda: cache_evict(c, t, n, w, i32([[2]]), 10, recent=-1), lambda: cache_evict(c, t, n, w.double(), i32([[2]]), 10),
        lambda: cache_read(c, t, n, -1), lambda: cache_read(c, t, n, 4, dtype=torch.float64), lambda: cache_read(c, t, n, 4, start=i32([1, 2])),
        lambda: KVCache(c.k.half(), c.v, c.k_scale, c.v_scale), lambda: KVCache(c.k[:, :, :32], c.v[:, :, :32], c.k_scale, c.v_scale),
        lambda: KVCache(c.k, c.v, c.k_scale[:2], c.v_scale), lambda: KVCache(c.k, c.v, c.k_scale, c.v_scale.cpu()),
        lambda: KVCache(c.k, c.v, c.k_scale, c.v_scale, torch.zeros((4, 2, 64), device=DEV)), lambda: KVCache.empty(4, 2, 40, device=DEV), lambda: KVCache.empty(0, 2, 64, device=DEV),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    m = KVCache.empty(4, 2, 64, device=DEV, metadata=True)
    with pytest.raises(ValueError, match="bool"):
        cache_append(m, k, k, t, n, in_span=torch.zeros((1, 3), dtype=torch.int32, device=DEV))
    for f in (lambda: cache_attention(q.clone().requires_grad_(), c, t, n), lambda: cache_append(c, k, k.clone().requires_grad_(), t, n)):
        with pytest.raises(RuntimeError, match="no_grad"):
            f()
    with torch.no_grad():
        assert not cache_attention(q.clone().requires_grad_(), c, t, n).requires_grad


def test_empty_calls():
    from kerneldev_b200 import KVCache, cache_append, cache_attention, cache_evict, cache_read
    c = KVCache.empty(4, 2, 64, device=DEV)
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    none = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    assert cache_attention(z(0, 4, 1, 64), c, none, i32([])).shape == (0, 4, 1, 64)
    o, lse = cache_attention(z(1, 4, 0, 64), c, i32([[1]]), i32([5]), return_lse=True)
    assert o.shape == (1, 4, 0, 64) and lse.shape == (1, 4, 0)
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
    pages = (1 << 32) // (H * 64 * D) + 40
    if free < 3 * pages * H * 64 * D:
        pytest.skip("needs 13 GB")
    rng = np.random.default_rng(0)
    c = KVCache.empty(pages, H, D, device=DEV)
    table = np.array([[pages - 1, pages - 33, 5, pages - 7]])
    x = rand_kv(rng, (2, 1, H, 230, D), torch.bfloat16).to(DEV)
    cache_append(c, x[0], x[1], i32(table), i32([0]))
    q = rand_kv(rng, (1, 2 * H, 1, D), torch.bfloat16, False).to(DEV)
    got = cache_attention(q, c, i32(table), i32([230]), return_lse=True)
    used = torch.tensor(table[0], device=DEV)
    small = KVCache(c.k.view(torch.uint8)[used].view(torch.float8_e4m3fn), c.v.view(torch.uint8)[used].view(torch.float8_e4m3fn), c.k_scale[used], c.v_scale[used])
    check_attention(small, q, np.array([[0, 1, 2, 3]]), [230], [1], got)


def test_on_another_stream_and_host_thread():
    """Two threads with a stream and a cache each."""
    import threading
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(30)
    work, errors = [], []
    for i in range(2):
        c, table = filled(rng, 2, 2, 64, [300, 129], torch.float16, i == 1)
        work.append((c, table, rand_kv(rng, (2, 6, 2, 64), torch.float16, False).to(DEV)))
    torch.cuda.synchronize()

    def go(c, table, q):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = cache_attention(q, c, i32(table), i32([300, 129]), return_lse=True)
                torch.cuda.current_stream().synchronize()
                check_attention(c, q, table, [300, 129], [2, 2], got)
        except BaseException as e:   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=go, args=w) for w in work]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


@pytest.mark.parametrize("T,G", [(1, 3), (20, 4)])
def test_sequences_that_share_pages_and_padding_that_is_nan(T, G):
    """One table for all (a batch stride of zero) whose last page comes twice, queries of one head for all heads, rows without a query full of NaN, sequences
    without any among them."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(40 + T)
    c, table = filled(rng, 1, 2, 64, [200], torch.bfloat16, False)
    B, rows = 3, np.array([table[0].tolist()[:3] + [table[0, 2]]] * 3)
    shared = i32(rows[:1]).expand(B, 4)
    q_lens = [T, 0, max(T // 2, 1)]
    lens = [256, 192, 70]
    one = rand_kv(rng, (B, 1, T, 64), torch.bfloat16, False).to(DEV)
    for b in range(B):
        one[b, :, q_lens[b]:] = float("nan")
    q = one.expand(B, 2 * G, T, 64)
    w = torch.zeros((2, B, 256), device=DEV).transpose(0, 1)
    got = cache_attention(q, c, shared, i32(lens), i32(q_lens), return_lse=True, weights=w)
    check_attention(c, q, rows, lens, q_lens, got, weights=w)


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


def test_memory_that_is_not_the_calls_own_is_refused():
    from kerneldev_b200 import KVCache, cache_append, cache_attention, cache_evict, cache_read
    c = KVCache.empty(4, 2, 64, device=DEV)
    q, k = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16, device=DEV), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16, device=DEV)
    t, n, wide = i32([[0], [1]]), i32([5, 6]), torch.zeros(1000, device=DEV)
    for strides in ((0, 64, 1), (64, 0, 1), (100, 63, 1), (64, 100, 1), (128, 127, 1), (63, 128, 1)):   # heads or sequences over one another
        with pytest.raises(ValueError, match="weights"):
            cache_attention(q, c, t, n, weights=wide.as_strided((2, 2, 64), strides))
    for strides in ((128, 64, 1), (64, 128, 1), (300, 70, 1)):
        w = wide.zero_().as_strided((2, 2, 64), strides)
        cache_attention(q, c, t, n, weights=w)
        assert torch.allclose(w.sum(2), torch.full((2, 2), 2.0, device=DEV)) and float(wide.sum()) == pytest.approx(8.0)
    w = torch.zeros((2, 2, 64), device=DEV)
    old = c.k_scale.data
    c.k_scale.data = old.clone()   # the cache would go on with the storage that this leaves
    for f in (lambda: cache_attention(q, c, t, n), lambda: cache_append(c, k, k, t, n), lambda: cache_evict(c, t, n, w, t, 2), lambda: cache_read(c, t, n, 2)):
        with pytest.raises(ValueError, match="other memory"):
            f()
    KVCache(c.k, c.v, c.k_scale, c.v_scale)
    c.k_scale.data = old
    cache_attention(q, c, t, n)


def test_status_is_checked_after_every_call():
    assert os.environ.get("KD_CHECK_STATUS") == "1"
