"""The 8-bit cache at the limits of its numbers and of its arguments: NaN in live rows, scales and queries far apart, what invalid arguments leave alone.

The sequences are longer than 8 pages where an item's pages are to be shared by several CTAs and joined."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv_cache import DEV, filled, i32, rand_kv

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
