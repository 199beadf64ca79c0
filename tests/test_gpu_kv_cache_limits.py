"""The 8-bit cache at the limits of its numbers and of its arguments: NaN in live rows, scales and queries far apart, what invalid arguments leave alone.

The sequences are longer than 8 pages where an item's pages are to be shared by several CTAs and joined."""
import numpy as np
import pytest
import torch

from oracle import kv_cache_oracle as ko
from tests.test_gpu_kv_cache import DEV, as_oracle, assert_cache, check_attention, filled, i32, make_cache, rand_kv, tables

pytestmark = pytest.mark.gpu

# B, key heads, heads of a group, queries: few items and many items (even shares), one tile of rows and more, and the kernel for many rows
SHARED = [(2, 2, 3, 1), (2, 1, 4, 4), (2, 1, 8, 3), (40, 8, 1, 1), (2, 2, 2, 40), (40, 4, 1, 40)]


@pytest.mark.parametrize("B,Hkv,G,T", SHARED)
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


@pytest.mark.parametrize("B,Hkv,G,T", SHARED)
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
        k = c.k.view(torch.uint8)
        pages = table[b, first:first + 7]
        old = k[pages, Hkv - 1].clone()
        k[pages, Hkv - 1] = 0x7F
        w = torch.zeros((B, Hkv, 1900), device=DEV) if weigh else None
        o, lse = cache_attention(q, c, i32(table), i32(lens), return_lse=True, weights=w)
        k[pages, Hkv - 1] = old
        hit = torch.zeros(lse.shape, dtype=torch.bool, device=DEV)
        hit[b, (Hkv - 1) * G:] = True
        assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
        assert torch.equal(o[~hit], clean[0][~hit]) and torch.equal(lse[~hit], clean[1][~hit])
        if weigh:
            assert torch.isnan(w[b, Hkv - 1, :int(lens[b]) - T + 1]).all() and torch.isfinite(w[b, :Hkv - 1]).all() and torch.isfinite(w[:b]).all()


@pytest.mark.parametrize("D", [16, 48, 64, 80, 112, 128])
@pytest.mark.parametrize("G,T", [(3, 1), (2, 40)])
def test_nan_of_single_values_at_every_head_dim(D, G, T):
    """Values that are NaN in one column each, in tokens that some rows see and others do not: the column is NaN in the rows that see it, all else is as without them."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(D + T)
    B, n = 2, 900
    c, table = filled(rng, B, 1, D, [n, n], torch.bfloat16, False)
    q = rand_kv(rng, (B, G, T, D), torch.bfloat16, False).to(DEV)
    clean = cache_attention(q, c, i32(table), i32([n, n]), return_lse=True)
    v = c.v.view(torch.uint8)
    nan = torch.zeros((B, T, D), dtype=torch.bool, device=DEV)
    for b in range(B):
        for d in range(b, D, 3):
            at = n - 1 - int(rng.integers(T)) if d % 2 else int(rng.integers(n))
            v[table[b, at // 64], 0, at % 64, d] = 0x7F if d % 4 else 0xFF
            nan[b, max(at - (n - T), 0):, d] = True
    o, lse = cache_attention(q, c, i32(table), i32([n, n]), return_lse=True)
    nan = nan[:, None].expand(B, G, T, D)
    assert torch.isnan(o[nan]).all() and torch.isfinite(o[~nan]).all() and torch.equal(lse, clean[1])
    change = (o - clean[0]).float().abs()[~nan]   # a column's NaN took the place of a number: the others are sums of the same products
    assert not change.any()


def values_of(rng, B, Hkv, n, D, kind):
    """Keys and values of which a page holds numbers of 2**38 and the next one of 2**-20; the large ones are few, so that in their page all other channels become zeros."""
    x = rand_kv(rng, (2, B, Hkv, n, D), torch.float32, False)
    if kind == "alternate":   # every second page has one large number, each in another channel
        for page in range(1, n // 64, 2):
            x[1, :, :, 64 * page + int(rng.integers(64)), int(rng.integers(D))] = 2.0 ** int(rng.integers(20, 38))
        return x
    for b in range(B):
        for h in range(Hkv):
            for at in rng.integers(0, 1100, 2 if kind == "two" else 1):
                x[1, b, h, at, int(rng.integers(D))] = 2.0 ** int(rng.integers(10, 39))
                if kind == "unlikely":   # a token of 2**-40 of the others' probability and a value that makes up for it
                    x[0, b, h, at] = -80 * np.log(2.0) / D ** 0.5
    if kind == "two":
        x[1, :, :, 640:768] *= 2.0 ** -20
    return x


def check_causal(c, q, table, lens, o, lse, weights):
    """Against the definition in 64 bits, without metadata. Tolerances as derived in test_gpu_kv_cache.py, and one term more: probabilities are rounded to halves, whose steps end at
    2**-24. With M the row's largest p 2**ev (ev: the exponent of the page's V scale), P its largest p and m the largest p 2**ev of a page, the kernels bring a token's p 2**ev to a half after a
    factor of at least 2**8 / (sqrt(2) M), and of 2**8 / (sqrt(2) 2**4 P 2**ev) or 2**-4 / (sqrt(2) m) (their reference may be the whole number next to the largest, hence the root): it is off by 2**-25 / factor, which is
    sqrt(2) 2**-33 min(M, max(2**4 P 2**ev, 2**12 m)), times the stored number. A tile of many rows has two pages whose exponents are at most 4 apart: m of a page and its neighbours. Taken as 2**-32."""
    want = as_oracle(c)
    B, H, T, D = q.shape
    Hkv = want["k"].shape[1]
    G = H // Hkv
    o, lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
    qs = q.double().cpu().numpy()
    assert np.isfinite(o).all() and np.isfinite(lse).all()
    for b in range(B):
        n, pages = int(lens[b]), table[b, :-(-int(lens[b]) // 64)]
        blocks = len(pages)
        for h in range(Hkv):
            k, v = ko.values(want, table[b], n, h, "k"), ko.values(want, table[b], n, h, "v")
            scale = np.repeat(want["v_scale"][pages, h], 64)[:n]
            total = np.zeros(n)
            deltas = []
            for g in range(G):
                x = qs[b, h * G + g]
                see = np.arange(n)[None] <= (n - T + np.arange(T))[:, None]
                s = np.where(see, x @ k.T * D ** -0.5, -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - top)
                l = p.sum(1, keepdims=True)
                p /= l
                ref = p @ v
                a = p @ np.abs(v)
                mag = np.where(see, np.abs(x) @ np.abs(k).T, 0).max(1) * D ** -0.5
                delta = 2.0 ** -21 * (mag * 1.5 + 2) + n * 2.0 ** -24
                m = np.pad(p * scale, ((0, 0), (0, 64 * blocks - n))).reshape(T, blocks, 64).max(2)
                near = np.abs(np.diff(np.log2(want["v_scale"][pages, h]))) <= 4   # page and next one
                m = np.maximum(m, np.maximum(np.pad(np.where(near, m[:, :-1], 0), ((0, 0), (1, 0))), np.pad(np.where(near, m[:, 1:], 0), ((0, 0), (0, 1)))))
                step = 2.0 ** -32 * np.minimum(m.max(1, keepdims=True), np.maximum(2.0 ** 12 * np.repeat(m, 64, axis=1)[:, :n], 2.0 ** 4 * p.max(1, keepdims=True) * scale))
                floor = np.where(see, step, 0) @ np.abs(v / scale[:, None])
                got = o[b, h * G + g]
                tol = torch.finfo(q.dtype).eps / 2 * (np.abs(ref) + 0.01 * a) + a * (2.0 ** -11 + 2 * delta[:, None]) + floor + 2.0 ** -25
                err = np.abs(got - ref)
                assert (err <= tol).all(), f"O: {(err / tol).max()} of the tolerance at {b, h, g, np.unravel_index((err / tol).argmax(), err.shape)}"
                rl = (top + np.log(l))[:, 0] / np.log(2.0)
                assert (np.abs(lse[b, h * G + g] - rl) <= 2 * delta + 2.0 ** -22 * np.abs(rl)).all(), "LSE"
                total += p.sum(0)
                deltas.append(delta.max())
            w = weights[b, h].double().cpu().numpy()
            assert (np.abs(w[:n] - total) <= total * (3 * max(deltas) + G * T * 2.0 ** -24) + 1e-30).all() and not w[n:].any(), "weights"


@pytest.mark.parametrize("B,Hkv,G,T", [(1, 1, 1, 1), *SHARED])
@pytest.mark.parametrize("kind", ["one", "two", "unlikely", "alternate"])
@pytest.mark.parametrize("D", [64, 128])
def test_values_far_apart(B, Hkv, G, T, kind, D):
    """A page's large number takes nothing from the other channels, which the other pages alone have, whatever their scales. (bfloat16, whose range the outputs need.)"""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(B + T)
    n = 1300 if B > 1 else 500   # (one sequence: a short table, whose pages are not shared)
    lens = rng.integers(n - 200, n, B)
    pages = B * (-(-n // 64))
    c = make_cache(pages, Hkv, D)
    table = tables(rng, B, pages // B, pages)
    x = values_of(rng, B, Hkv, max(n, 1100), D, kind)[:, :, :, :n]
    cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32(np.zeros(B)), i32(lens))
    q = rand_kv(rng, (B, Hkv * G, T, D), torch.float32, False)
    if kind == "unlikely":
        q = 0.5 + 0.1 * q.clamp(-1, 1)   # about -40 bits with the key above
    q = q.to(torch.bfloat16).to(DEV)
    w = torch.zeros((B, Hkv, n), device=DEV)
    o, lse = cache_attention(q, c, i32(table), i32(lens), return_lse=True, weights=w)
    check_causal(c, q, table, lens, o, lse, w)


# ---- lengths and pages that do not fit ----------------------------------------------------------------------------

def appended(rng, c, T):
    x = rand_kv(rng, (2, 3, 2, T, 64), torch.bfloat16).to(DEV)
    m = rng.random((2, 3, T)) < 0.5
    return x, dict(in_span=torch.tensor(m[0], device=DEV), is_prefix=torch.tensor(m[1], device=DEV))


@pytest.mark.parametrize("lens,new", [([-1, 40, 0], None), ([-3, -2 ** 31, 2 ** 31 - 1], None), ([257, 256, 300], None), ([100, 64, 63], [-1, 5, -2 ** 31]), ([0, 0, 0], [71, 2 ** 31 - 1, 70]),
                                      ([-70, 10, 10], [70, 70, 0]), ([230, 200, 255], None)])
def test_append_of_lengths_that_cannot_be_changes_nothing(lens, new):
    """A negative length, one beyond the table, a negative number of tokens, more than there are: bytes, scales and descriptors of that sequence stay, the other ones get their tokens. What
    goes beyond the last page is cut."""
    from kerneldev_b200 import cache_append
    rng = np.random.default_rng(abs(lens[0]))
    T = 70
    c, table = filled(rng, 3, 2, 64, [256, 200, 100], torch.bfloat16, True)
    want = as_oracle(c)
    x, m = appended(rng, c, T)
    n = [T] * 3 if new is None else new
    valid = [0 <= a <= 256 and 0 <= b <= T for a, b in zip(lens, n)]
    count = [min(b, 256 - a) if ok else 0 for a, b, ok in zip(lens, n, valid)]
    with pytest.raises(ValueError, match="length"):
        cache_append(c, x[0], x[1], i32(table), i32(lens), None if new is None else i32(new), **m)
    d = ko.descriptors(m["in_span"].cpu().numpy(), np.zeros((3, T), int), m["is_prefix"].cpu().numpy())
    ko.append(want, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, [a if ok else 0 for a, ok in zip(lens, valid)], count, d)
    assert_cache(c, want)


def test_calls_with_bad_lengths_and_pages_keep_what_is_valid(monkeypatch):
    """Readers leave out what does not fit and nothing else; writers change no page but the ones that are named."""
    from kerneldev_b200 import cache_append, cache_attention, cache_evict, cache_read
    rng = np.random.default_rng(1)
    c, table = filled(rng, 2, 2, 64, [250, 100], torch.bfloat16, False)
    want = as_oracle(c)
    q = rand_kv(rng, (2, 4, 1, 64), torch.bfloat16, False).to(DEV)
    w = torch.tensor(rng.random((2, 2, 256)), dtype=torch.float32, device=DEV)
    good, lens = i32(table), i32([250, 100])
    free = [p for p in range(c.k.shape[0]) if p not in table]
    index, kept_lens, kept = cache_evict(c, good, lens, w, i32([[free[0]], [free[1]]]), 64)
    c.k.view(torch.uint8)[free] = 0x7F
    c.v.view(torch.uint8)[free] = 0x7F
    c.k_scale[free] = c.v_scale[free] = 2.0 ** 31
    assert_cache(c, want)
    k, v = cache_read(c, good, lens, 256)
    monkeypatch.delenv("KD_CHECK_STATUS")

    def reported(match):
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match=match):
            cache_read(c, good, lens, 1)
        assert_cache(c, want)

    wrong = table.copy()
    wrong[0, 1], wrong[1, 0] = c.k.shape[0], -1
    bk, bv = cache_read(c, i32(wrong), lens, 256)
    reported("page number")
    for got, full in ((bk, k), (bv, v)):
        full = full.clone()
        full[0, :, 64:128] = full[1, :, :64] = 0
        assert torch.equal(got, full)
    o, lse = cache_attention(q, c, i32(wrong), lens, return_lse=True)
    reported("page number")
    for b, pages, n in ((0, [table[0, i] for i in (0, 2, 3)], 186), (1, [table[1, 1]], 36)):   # the same tokens without the page: one query, which sees all
        po, pl = cache_attention(q[b:b + 1], c, i32([pages]), i32([n]), return_lse=True)
        assert torch.allclose(pl, lse[b:b + 1], atol=1e-5) and torch.allclose(po.float(), o[b:b + 1].float(), rtol=2.0 ** -7, atol=1e-3)
    for bad, same in (([257, -1], [256, 0]), ([2 ** 31 - 1, 100], [256, 100])):
        got = cache_attention(q, c, good, i32(bad), return_lse=True)
        reported("length")
        assert all(torch.equal(x, y) for x, y in zip(got, cache_attention(q, c, good, i32(same), return_lse=True)))
    got = cache_evict(c, good, lens, w, i32([[-5], [2 ** 31 - 1]]), 64)
    reported("page number")
    assert all(torch.equal(x, y) for x, y in zip(got, (index, kept_lens, kept)))
    x = rand_kv(rng, (2, 2, 2, 3, 64), torch.bfloat16).to(DEV)
    cache_append(c, x[0], x[1], i32([[-1] * 4, [c.k.shape[0]] * 4]), lens)
    reported("page number")
    check_attention(c, q, table, [250, 100], [1, 1], cache_attention(q, c, good, lens, return_lse=True))


@pytest.mark.parametrize("sid", [2 ** 23, -2 ** 23 - 1, 2 ** 24 + 1, -2 ** 63])
def test_span_ids_that_a_descriptor_cannot_hold_are_reported(sid):
    """Two ids that agree in their low 24 bits would see one another; the ones at the ends of the range are well, and so is a wrong one behind the new tokens."""
    from kerneldev_b200 import KVCache, cache_append
    c = KVCache.empty(3, 2, 64, device=DEV, metadata=True)
    k = torch.zeros((2, 2, 70, 64), dtype=torch.bfloat16, device=DEV)
    t, n = i32([[0, 1], [2, 2]]), i32([0, 0])
    ins = torch.ones((2, 70), dtype=torch.bool, device=DEV)
    ids = torch.full((2, 70), 2 ** 23 - 1, dtype=torch.int64, device=DEV)
    ids[0, 3] = -2 ** 23
    ids[1, 9] = sid
    cache_append(c, k, k, t, n, i32([70, 9]), in_span=ins, span_id=ids)
    with pytest.raises(ValueError, match="24 signed bits"):
        cache_append(c, k, k, t, n, i32([70, 10]), in_span=ins, span_id=ids)
    cache_append(c, k, k, t, n, i32([70, 9]), in_span=ins, span_id=ids)   # reported once


def test_a_graph_keeps_the_status_word_of_its_cache(monkeypatch):
    """A replay reports into the word that the capture has seen. The cache is gone, and as many others have come as there are words: none of them, and no plan, hears of it."""
    from kerneldev_b200 import KVCache, cache_append, cache_read
    monkeypatch.delenv("KD_CHECK_STATUS", raising=False)
    c = KVCache.empty(2, 1, 64, device=DEV)
    tensors = (c.k, c.v, c.k_scale, c.v_scale)
    x = torch.zeros((1, 1, 1, 64), dtype=torch.float16, device=DEV)
    t, lens, outs = i32([[0]]), i32([3]), []
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):   # two captures in turn, and a call outside between them
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache_append(c, x, x, t, lens)
            outs.append(cache_read(c, t, lens, 4))
        graphs.append(g)
        cache_append(c, x, x, t, lens)
    del c
    others = [KVCache(*tensors) for _ in range(2100)]
    lens.fill_(-1)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in others:
        cache_read(o, t, lens, 0)   # looks at the word and launches nothing
    del graphs, g
    torch.cuda.synchronize()
    lens.fill_(3)
    others.append(KVCache(*tensors))
    cache_append(others[-1], x, x, t, lens)
    cache_read(others[0], t, lens, 1)


@pytest.mark.parametrize("T,G,weigh", [(1, 8, False), (1, 8, True), (40, 2, False)])
def test_a_length_that_has_just_been_written(monkeypatch, T, G, weigh):
    """The join looks the lengths up while the attention before it runs, on SMs of which many had the old length in their L1 from an append."""
    from kerneldev_b200 import KVCache, cache_append, cache_attention
    rng = np.random.default_rng(9)
    c = KVCache.empty(64, 4, 64, device=DEV)
    t, lens, back = i32([list(range(64))]), i32([600]), i32([600])
    x = rand_kv(rng, (2, 1, 4, 2000, 64), torch.float16, False).to(DEV)
    cache_append(c, x[0], x[1], t, i32([0]))
    q = rand_kv(rng, (1, 4 * G, T, 64), torch.float16, False).to(DEV)
    w = torch.zeros((1, 4, 4096), device=DEV) if weigh else None
    lengths = rng.integers(600, 2000, 60)
    want = []
    for n in lengths:
        want.append(cache_attention(q, c, t, i32([n]), return_lse=True))
    torch.cuda.synchronize()
    new = [i32([n]) for n in lengths]
    got = []
    monkeypatch.delenv("KD_CHECK_STATUS", raising=False)   # without a wait after each call
    for n in new:
        cache_append(c, x[0, :, :, 600:], x[1, :, :, 600:], t, lens.copy_(back))
        lens.copy_(n)
        got.append(cache_attention(q, c, t, lens, return_lse=True, weights=w))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- scores and queries at the ends of their range ----------------------------------------------------------------

@pytest.mark.parametrize("B,Hkv,G,T", [(1, 1, 2, 1), *SHARED])
@pytest.mark.parametrize("power,kind", [(10, "bf16"), (17, "bf16"), (20, "negative"), (21, "nan"), (45, "bf16"), (80, "bf16"), (100, "negative"), (110, "nan"), (30, "f16"), (-90, "bf16"), (-120, "bf16")])
def test_scores_far_from_zero(B, Hkv, G, T, power, kind):
    """Every second head's queries are whole numbers times 2**power (or, with f16, all keys are), the others' are whole numbers. All products and sums are exact, so that scores that are
    equal are equal in any order of summation, and the others are at least 2**power log2(e) / 8 apart in powers of two: from 2**9 on a row's weight belongs to its largest scores, evenly. (Their
    error in powers of two, on which the tolerance of the other rows rests, does not matter.) nan: a value that the last query alone sees."""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(abs(power) + T)
    D, n = 64, 1300 if B > 1 else 400
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    lens = rng.integers(n - 200, n, B)
    pages = B * (-(-n // 64))
    c = make_cache(pages, Hkv, D)
    table = tables(rng, B, pages // B, pages)
    k = rng.integers(1, 4, (B, Hkv, n, D)) if kind == "negative" else rng.integers(-3, 4, (B, Hkv, n, D))
    v = rand_kv(rng, (B, Hkv, n, D), torch.float32, False).numpy()
    v[:, :, 192:256] *= 2.0 ** 20 if kind != "f16" else 2.0 ** 7
    q = rng.integers(-2, 0, (B, Hkv * G, T, D)) if kind == "negative" else rng.integers(-2, 3, (B, Hkv * G, T, D))
    k, q = k.astype(np.float64), q.astype(np.float64)
    large = (np.arange(Hkv * G) % 2 == 0) if kind != "f16" else np.ones(Hkv * G, bool)
    if kind == "f16":
        k *= 2.0 ** power
    else:
        q[:, large] *= 2.0 ** power
    if kind == "nan" and T > 1:
        for b in range(B):
            v[b, :, lens[b] - 1] = np.nan
    cache_append(c, torch.tensor(k, dtype=torch.float32, device=DEV), torch.tensor(v, device=DEV), i32(table), i32(np.zeros(B)), i32(lens))
    w = torch.zeros((B, Hkv, n), device=DEV)
    o, lse = cache_attention(torch.tensor(q).to(dtype).to(DEV), c, i32(table), i32(lens), return_lse=True, weights=w)
    o, lse, w = (t.double().cpu().numpy() for t in (o, lse, w))
    want = as_oracle(c)
    eps = torch.finfo(dtype).eps
    for b in range(B):
        for h in range(Hkv):
            keys, vals = ko.values(want, table[b], int(lens[b]), h, "k"), ko.values(want, table[b], int(lens[b]), h, "v")
            assert np.array_equal(keys, k[b, h, :lens[b]])
            total, slack = np.zeros(lens[b]), np.zeros(lens[b])
            for g in range(G):
                hq = h * G + g
                rows = T - 1 if kind == "nan" and T > 1 else T
                if rows < T:
                    assert np.isnan(o[b, hq, rows]).all()
                see = np.arange(lens[b])[None] <= (lens[b] - T + np.arange(T))[:, None]
                s = np.where(see, q[b, hq] @ keys.T / 8, -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - top)
                l = p.sum(1, keepdims=True)
                p /= l
                clean = np.nan_to_num(vals)
                ref, a = p @ clean, p @ np.abs(clean)
                mag = np.where(see, np.abs(q[b, hq]) @ np.abs(keys).T, 0).max(1) / 8
                delta = (np.full(T, 2.0 ** -20) if large[hq] and power >= 9 else 2.0 ** -21 * (mag * 1.5 + 2)) + lens[b] * 2.0 ** -24
                floor = 2.0 ** -28 * (see @ np.abs(clean)) * p.max(1, keepdims=True) * (1 - (large[hq] and power >= 9))   # see cache_attention on weights
                tol = eps / 2 * (np.abs(ref) + 0.01 * a) + a * (2.0 ** -11 + 2 * delta[:, None]) + floor + 2.0 ** -25
                err = np.abs(o[b, hq] - ref)[:rows]
                assert (err <= tol[:rows]).all(), f"O: {(err / tol[:rows]).max()} of the tolerance at {b, hq, np.unravel_index((err / tol[:rows]).argmax(), err.shape)}"
                rl = (top / np.log(2.0) + np.log2(l))[:, 0]
                assert (np.abs(lse[b, hq] - rl) <= 2 * delta + 2.0 ** -21 * np.abs(rl)).all(), "LSE"
                total += p.sum(0)
                # below 2**16 a row's sum is of exact products and the weights are of scores rounded to 2**-24 of them: their ratio is off by that times log(2), in the scores' units
                steps = np.where(np.abs(top) < 2.0 ** 16, 2.0 ** -23 * np.abs(top), 0)
                slack += (p * (3 * delta[:, None] + steps + G * T * 2.0 ** -24)).sum(0)
            assert (np.abs(w[b, h, :lens[b]] - total) <= slack + total * G * T * 2.0 ** -24 + 1e-30).all(), "weights"


def test_a_query_of_large_numbers_over_keys_of_small_ones():
    """The products are ordinary numbers, whatever their factors are: queries of 2**100 over keys of 2**-32 * 448 and less, and the other way round."""
    from kerneldev_b200 import cache_append, cache_attention
    rng = np.random.default_rng(3)
    for T in (1, 40):
        for power in (-34, 30):
            c = make_cache(20, 1, 64)
            table = tables(rng, 1, 20, 20)
            x = rand_kv(rng, (2, 1, 1, 1200, 64), torch.float32, False)
            x[0] *= 2.0 ** power
            cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32([0]))
            q = (rand_kv(rng, (1, 2, T, 64), torch.float32, False) * 2.0 ** (100 if power < 0 else -100)).to(torch.bfloat16).to(DEV)
            scale = 2.0 ** (-100 - power if power < 0 else 100 - power) / 8
            if scale >= 1e30:
                continue
            o, lse = cache_attention(q, c, i32(table), i32([1200]), return_lse=True, sm_scale=scale)
            got = cache_attention((q.float() * 2.0 ** (-100 if power < 0 else 100)).to(torch.bfloat16), c, i32(table), i32([1200]), return_lse=True, sm_scale=2.0 ** -power / 8)
            assert torch.equal(o, got[0]) and torch.equal(lse, got[1])
            check_attention(c, (q.float() * 2.0 ** (-100 if power < 0 else 100)).to(torch.bfloat16), table, [1200], [T], got, scale=2.0 ** -power / 8)


def test_weights_of_few_rows_over_page_tables_that_are_wide():
    """Tables for more tokens than there is room for scores: the weights come from K once more."""
    from kerneldev_b200 import cache_attention
    rng = np.random.default_rng(70)
    B, Hkv, G = 6, 4, 8
    lens = rng.integers(1, 700, B)
    c, table = filled(rng, B, Hkv, 64, lens, torch.bfloat16, False)
    q = rand_kv(rng, (B, Hkv * G, 1, 64), torch.bfloat16, False).to(DEV)
    for width in (1 << 14, 1 << 10):   # 768 MB of scores, 48 MB
        wide = torch.zeros((B, width), dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = i32(table)
        w = torch.zeros((B, Hkv, 700), device=DEV)
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        o, lse = cache_attention(q, c, wide, i32(lens), return_lse=True, weights=w)
        assert torch.cuda.max_memory_allocated() - held < (64 << 20)
        check_causal(c, q, table, lens, o, lse, w)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G,T", [(1, 1), (12, 1), (2, 16), (1, 40), (4, 40)])
def test_a_token_that_has_all_the_weight_gives_its_value(dtype, G, T):
    """The first query of a sequence sees its own token alone, another one a key that makes 60 bits of difference: their outputs are the cached numbers, which both types hold."""
    from kerneldev_b200 import cache_append, cache_attention, cache_read
    rng = np.random.default_rng(G + T)
    D, lens = 64, [T, 1, 1300]
    c = make_cache(70, 1, D)
    table = tables(rng, 3, 21, 70)
    x = rand_kv(rng, (2, 3, 1, 1300, D), torch.float32, False)
    x[0, 2, 0, 700] = 40.0
    cache_append(c, x[0].to(DEV), x[1].to(DEV), i32(table), i32([0, 0, 0]), i32(lens))
    q = rand_kv(rng, (3, G, T, D), torch.float32, False)
    q[2] = 1.0 + 0.1 * torch.tensor(rng.random((G, T, D)))
    o = cache_attention(q.to(dtype).to(DEV), c, i32(table), i32(lens), i32([T, 1, T]))
    v = cache_read(c, i32(table), i32(lens), 1300, dtype=dtype)[1]
    assert torch.equal(o[0, :, 0], v[0, 0, :1].expand(G, D)) and torch.equal(o[1, :, 0], v[1, 0, :1].expand(G, D))
    assert torch.equal(o[2], v[2, 0, 700].expand(G, T, D))
