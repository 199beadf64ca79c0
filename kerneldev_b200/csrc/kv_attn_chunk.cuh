// Attention over the cache for many query rows of a key head (a chunk of a prompt), for both number formats (kBits): 128 rows of a CTA on tcgen05, two CTAs an SM.
//
// The products are GEMMs here, so the cache's tiles are converted once for 128 rows: to halves (exact; numbers of 4 bits with their scales) into swizzled shared memory, and both
// products run on halves with S, P and O in TMEM. Roles (256 threads, so that each has 128 registers):
//   warps 0-3  softmax, a thread to a row: masks, running maximum, P over the scores it was made from. Warp 0 issues the products: P V when all four
//              warps' P is there, directly behind it the next scores
//   warps 4-7  converters: 128 tokens (two pages) at a time from global memory through registers, one tile ahead. They decide which tiles are worked on:
//              one that no row of the CTA sees is left out (spans of a hierarchical mask, tokens behind the chunk)
// Q, one K tile and one V tile are 96 KB at head dim 128 and S and O 256 columns, so that two CTAs share an SM: the exponentials of one run under
// the products of the other. Scales, the offset of the probabilities and the slack of the maximum are as in kv_attn_rows.cuh.
//
// A tile's chain is: K converted -> S -> softmax -> P V, and the next S directly behind P V. Barriers, each used once a tile:
//   K   converters: K and the tile's record are there     S   S is complete (K is free)
//   V   converters: V is there                            P   softmax: P is there         PV  P V is complete (V, P's columns and O are free)
// Every wait is bounded. One that runs out is reported through status_mirror, and all roles end. The converter warps meet at named barriers, which have no limit, to
// exchange a tile's words: so they agree at the first of them whether all go on, and leave together.
//
// NaN: an item whose output has any is done once more with NaN values as zeros and a bit for each (token, dim) that was one; a row that sees the
// token gets NaN there. So is one that has met scores beyond KA_FAR, from rounded scores, with V's scale in the units of O.
#pragma once
#include <stddef.h>

#include <algorithm>

#include "attn_common.cuh"
#include "kv_attn.cuh"

namespace kd {

constexpr int CH_THREADS = 256, CH_TOKENS = 128, CH_RECORDS = 3;
// registers: 128 a thread at launch; the converters release what the softmax warps take
constexpr uint32_t CH_REGS_LIGHT = 96, CH_REGS_COMPUTE = 160;
static_assert(CH_REGS_LIGHT + CH_REGS_COMPUTE <= 2 * 128, "register pool");
constexpr uint32_t CH_SITE = 0x900u;   // wait sites 0x900 .. : role << 4 | barrier

// One tile of the walk, written by the converters for the others. Three slots in turn: the words of the tile ahead are written while the tile in hand is worked on, and the
// one before it may be.
struct ChunkRecord {
  int j0;                // first token
  int end;               // there is no tile: the item is done
  float ks[2];           // the pages' K scales and V exponents
  int ev[2];
  uint32_t words[3][4];  // tokens that are prefix, context, in a span (without metadata: all that exist, as context)
  uint32_t desc[CH_TOKENS];
};

// What no row of the CTA sees can be left out: what its rows see, put together.
struct ChunkRows {
  uint32_t sees, causal;   // classes
  int max_limit;
  int spans;               // some row looks for its own span
};

template <int D>
struct ChunkShared {
  static constexpr int BLOCKS = D > 64 ? 2 : 1, BLOCK = 128 * 128, TILE = BLOCKS * BLOCK;   // blocks of 64 head dims of 128 rows (16 KB: see koff_kmajor and desc_lo_mnmajor)
  uint8_t q[TILE], k[TILE], v[TILE];
  ChunkRecord record[CH_RECORDS];
  alignas(16) uint16_t nan_bits[CH_TOKENS][8];   // second pass alone: which of a token's head dims are NaN, 16 to a word; read 16 bytes at a time
  float factor[KC_ROWS];
  RowMask mask[KC_ROWS];
  ChunkRows rows;
  ItemShare item;                    // in shared memory: the roles need their registers (with 30 of them taken, the converters' loads were spilled, which waits for them)
  uint64_t bar[5];
  uint32_t tmem, redo;               // redo: a pass has met NaN (1), far rows (2: see KA_FAR)
  int tiles;                         // of the pass
  AbortFlag abort;
};
static_assert(offsetof(ChunkShared<64>, nan_bits) % 16 == 0 && offsetof(ChunkShared<128>, nan_bits) % 16 == 0, "nan_bits are read 16 bytes at a time");
enum { CB_K, CB_S, CB_V, CB_P, CB_PV };

// byte of element (row, d) in a tile: 64 head dims of a row are 128 bytes, swizzled
__device__ __forceinline__ uint32_t chunk_place(int row, int d) { return (d >> 6) * (128 * 128) + sw128_offset(row, (d & 63) >> 3) + (d & 7) * 2; }

// words of what a row sees of a tile
__device__ __forceinline__ void row_words(const RowMask& m, const ChunkRecord& r, bool metadata, int lane, uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t upto = low_bits(m.limit - r.j0 - 32 * i);
    w[i] = r.words[1][i] & (((m.sees & TD_CTX) != 0u ? 0xFFFFFFFFu : 0u) | ((m.causal & TD_CTX) != 0u ? upto : 0u));
    if (metadata) {
      if ((m.sees & TD_PRE) != 0u) w[i] |= r.words[0][i];
      if ((m.sees & TD_INS) != 0u) w[i] |= r.words[2][i];
    }
  }
  if (!metadata || (r.words[2][0] | r.words[2][1] | r.words[2][2] | r.words[2][3]) == 0u) return;
  uint32_t todo = __ballot_sync(0xffffffffu, m.span_key != 1u);   // one round for each span among the rows
  while (todo != 0u) {
    const uint32_t key = __shfl_sync(0xffffffffu, m.span_key, __ffs(todo) - 1);
    const bool mine = m.span_key == key;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t hit = __ballot_sync(0xffffffffu, span_match_key(key, r.desc[32 * i + lane]) != 0u);
      if (mine) w[i] |= hit;
    }
    todo &= ~__ballot_sync(0xffffffffu, mine);
  }
}

// 16 numbers of a token as they are stored
template <int kBits>
struct Piece16;
template <>
struct Piece16<8> {
  uint4 v;
};
template <>
struct Piece16<4> {
  uint2 v;
  uint32_t scale;   // the byte
};

// A converter thread's bytes of a tile as halves: rounds of 32 tokens and a block of 64 head dims, at fixed distances from the first one's two places.
// kWithoutNan: NaN as zeros, and a bit for each in nan_bits (of the first round's token and head dims).
template <int D, bool kWithoutNan>
__device__ __forceinline__ void store_tile(uint8_t* to, const uint32_t (&place)[2], const Piece16<8> (&reg)[4 * ChunkShared<D>::BLOCKS], uint16_t (*nan_bits)[8], int col) {
#pragma unroll
  for (int i = 0; i < 4 * ChunkShared<D>::BLOCKS; ++i) {
    uint32_t w[4] = {reg[i].v.x, reg[i].v.y, reg[i].v.z, reg[i].v.w};
    if constexpr (kWithoutNan) {
      uint32_t bits = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t n = __vcmpeq4(w[x] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
        w[x] &= ~n;
        bits |= ((n & 1u) | (n >> 7 & 2u) | (n >> 14 & 4u) | (n >> 21 & 8u)) << (4 * x);
      }
      const int d = (i >> 2) * 64 + col;
      if (d < D) nan_bits[32 * (i & 3)][d / 16] = static_cast<uint16_t>(bits);
    }
    const HalfPairs h0 = e4m3x4_to_f16x4(w[0]), h1 = e4m3x4_to_f16x4(w[1]), h2 = e4m3x4_to_f16x4(w[2]), h3 = e4m3x4_to_f16x4(w[3]);
    uint8_t* at = to + (i & 3) * 4096 + (i >> 2) * ChunkShared<D>::BLOCK;
    *reinterpret_cast<uint4*>(at + place[0]) = make_uint4(h0.lo, h0.hi, h1.lo, h1.hi);
    *reinterpret_cast<uint4*>(at + place[1]) = make_uint4(h2.lo, h2.hi, h3.lo, h3.hi);
  }
}

// ... of 4 bits: a group's numbers times its scale
template <int D, bool kWithoutNan>
__device__ __forceinline__ void store_tile(uint8_t* to, const uint32_t (&place)[2], const Piece16<4> (&reg)[4 * ChunkShared<D>::BLOCKS], uint16_t (*nan_bits)[8], int col) {
#pragma unroll
  for (int i = 0; i < 4 * ChunkShared<D>::BLOCKS; ++i) {
    uint32_t s = both_halves(reg[i].scale);
    if constexpr (kWithoutNan) {
      const uint32_t gone = nan_scales(s);
      s &= ~gone;
      const int d = (i >> 2) * 64 + col;
      if (d < D) nan_bits[32 * (i & 3)][d / 16] = static_cast<uint16_t>(gone);
    }
    uint32_t h[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) h[x] = times(e2m1x2_to_f16x2<true>(x < 4 ? reg[i].v.x : reg[i].v.y, x & 3), s);
    uint8_t* at = to + (i & 3) * 4096 + (i >> 2) * ChunkShared<D>::BLOCK;
    *reinterpret_cast<uint4*>(at + place[0]) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(at + place[1]) = make_uint4(h[4], h[5], h[6], h[7]);
  }
}

template <int kBits, int D>
__global__ void __launch_bounds__(CH_THREADS, KC_CTAS)
cache_attention_chunk_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                             const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  using Sh = ChunkShared<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Sh& sh = *reinterpret_cast<Sh*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const bool metadata = c.desc != nullptr;
  auto bar = [&](int i) { return smem_u32(&sh.bar[i]); };
  if (tid == 0) {
    sh.abort.v = 0;
    mbar_init(bar(CB_K), 4);
    mbar_init(bar(CB_S), 1);
    mbar_init(bar(CB_V), 4);
    mbar_init(bar(CB_P), 4);
    mbar_init(bar(CB_PV), 1);
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(&sh.tmem), 256);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tS = __reduce_max_sync(0xffffffffu, sh.tmem), tO = tS + CH_TOKENS;   // warp-uniform for the compiler
  touch_parameters(c, s, p, shape, ws);
  pdl_wait();
  pdl_launch_dependents();

  int n_k = 0, n_t = 0;   // uses of barrier K (one more than tiles for each pass over an item) and of the others
  auto wait = [&](int i, int use, int role) {
    return __all_sync(0xffffffffu, mbar_wait(bar(i), use & 1, &sh.abort, CH_SITE | role << 4 | i));
  };
  auto all_sync = [&]() { named_bar_sync(2, CH_THREADS); };   // (from the roles' own code)
  uint32_t done = 0;   // pages that this CTA has worked on
  // The CTA's next item, its rows in shared memory; false: it has none. All threads.
  auto open_item = [&]() -> bool {
    if (warp == 0) {
      const ItemShare n = share_of_cta(c, s, p, shape, done);
      if (lane == 0) sh.item = n;
    }
    all_sync();
    if (sh.item.here < 0) return false;
    const Item it = sh.item.it;

    // ---- Q as halves (bfloat16 times a power of two, see kv_attn_rows.cuh), masks and what the rows see together ----
    if (tid == 0) {
      sh.rows = ChunkRows{0u, 0u, 0, 0};
      sh.redo = 0u;
    }
    all_sync();
    constexpr int BATCH = 8, WARPS = CH_THREADS / 32;   // rows that a warp has on their way at once
#pragma unroll 1
    for (int r0 = warp; r0 < KC_ROWS; r0 += WARPS * BATCH) {
      const int d = 4 * lane;
      uint2 v[BATCH];
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int row = it.tile * KC_ROWS + r0 + x * WARPS;
        v[x] = make_uint2(0u, 0u);
        if (row < shape.rows && d < D) {
          const int n = row / shape.G, hq = it.h * shape.G + row - n * shape.G;
          v[x] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q.ptr) + it.b * p.q.stride_b + hq * p.q.stride_h + n * p.q.stride_t + d);
        }
      }
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int r = r0 + x * WARPS;
        int e = 0;
        if (p.dtype == KD_BF16) e = row_to_halves(v[x]);
        if (lane == 0) sh.factor[r] = row_factor(p.sm_scale, e);
        if (d < D) *reinterpret_cast<uint2*>(sh.q + chunk_place(r, d)) = v[x];
      }
    }
    if (tid < KC_ROWS) {
      const RowMask m = row_mask(c, s, p, it, it.tile * KC_ROWS + tid, shape.G, shape.rows, query_count(c, p, it.b));
      sh.mask[tid] = m;
      const uint32_t sees = __reduce_or_sync(0xffffffffu, m.sees), causal = __reduce_or_sync(0xffffffffu, m.causal);
      const int limit = __reduce_max_sync(0xffffffffu, m.limit);
      const bool spans = __any_sync(0xffffffffu, m.span_key != 1u);
      if (lane == 0) {
        atomicOr(&sh.rows.sees, sees);
        atomicOr(&sh.rows.causal, causal);
        atomicMax(&sh.rows.max_limit, limit);
        if (spans) sh.rows.spans = 1;
      }
    }
    fence_proxy_async_smem();
    all_sync();
    return true;
  };
  // After a pass over an item: whether there is to be another one. All threads.
  auto again = [&](int pass) -> bool {
    all_sync();
    const int tiles = sh.tiles;
    n_k += tiles + 1;
    n_t += tiles;
    const bool more = pass == 0 && sh.redo != 0u && sh.abort.v == 0u;   // once more, with care
    if (!more) done += max(sh.item.here, 1);
    all_sync();
    return more;
  };
  if (warp >= 4) {
    reg_dealloc<CH_REGS_LIGHT>();
    while (open_item()) {
      const Item it = sh.item.it;
      int pass = 0;
      do {
        const bool safe = pass == 1;
        const int most_apart = safe && (sh.redo & 2u) != 0u ? 0 : KA_APART;
        // ---------------------------------------- converters ----------------------------------------
        const int r = tid - 128;   // this thread's token of the tile for the descriptors
        const ChunkRows rows = sh.rows;
        // thread: 16 head dims of tokens; a quarter of a warp has two tokens' 64 head dims of a block, so that its stores take all banks
        const int col = (r & 3) * 16, row0 = r >> 2;
        constexpr int ROUNDS = 4 * Sh::BLOCKS;   // 32 tokens and one block of 64 head dims each
        struct Tile {
          int page[2], j0, ev[2];
          float ks[2];
          uint32_t desc;
        } cur;
        Piece16<kBits> reg[ROUNDS];   // K of a tile, then its V: each is asked for when the other has been stored, and awaited when its place is free
        bool ok = true;
        // Page numbers and scales of 32 blocks in the lanes of each warp, the page numbers of the 32 behind them already asked for: with a look-up for each tile, its
        // chain of loads (page, scale) stood between two tiles.
        const int32_t* table = s.table + it.b * s.table_stride;
        const int page0 = sh.item.page0, page_end = page0 + sh.item.here;
        int next = page0, batch = page0, batch_page, raw_ahead = 0, batch_ev;
        float batch_ks;
        uint32_t alone;   // bit l: the V scales of page l of the batch and the next one are too far apart for one reference of the exponents
        auto ask = [&](int from) { return from + lane < page_end ? table[from + lane] : -1; };
        auto open_batch = [&](int from, int raw) {
          batch = from;
          batch_page = from + lane < page_end ? checked_page(c, raw) : -1;
          const size_t place = block_index(c, max(batch_page, 0), it.h);
          batch_ks = kBits == 8 && batch_page >= 0 ? c.k_scale[place] : 1.f;
          batch_ev = kBits == 8 && batch_page >= 0 ? scale_exponent(c.v_scale[place]) : 0;
          raw_ahead = ask(from + 32);
          if constexpr (kBits == 4) {
            alone = 0u;
            return;
          }
          const int apart = batch_ev - __shfl_down_sync(0xffffffffu, batch_ev, 1), page_behind = __shfl_down_sync(0xffffffffu, batch_page, 1);
          alone = __ballot_sync(0xffffffffu, batch_page >= 0 && page_behind >= 0 && (apart < -most_apart || apart > most_apart));
        };
        open_batch(page0, ask(page0));
        auto is_alone = [&]() { return (alone >> (next - batch) & 1u) != 0u; };
        // The descriptor of this thread's token of the tile at `next`, asked for when the tile before it was found, and the tile's pages: two, or one that is alone.
        uint32_t ahead_desc = 0u;
        auto peek = [&]() {
          if (next - batch > 30) open_batch(next, next - batch == 32 ? raw_ahead : ask(next));
          const int p0 = __shfl_sync(0xffffffffu, batch_page, next - batch), p1 = __shfl_sync(0xffffffffu, batch_page, next - batch + 1), page = r < KC_PAGE ? p0 : p1;
          const bool alive = next < page_end && next * KC_PAGE + r < it.len && page >= 0 && (r < KC_PAGE || !is_alone());
          ahead_desc = !alive ? 0u : metadata ? c.desc[block_index(c, page, it.h) * KC_PAGE + (r & (KC_PAGE - 1))] : TD_CTX;
        };
        peek();
        // The next tile that some row sees, from `next` on. All four warps come to the same answer: the words are exchanged through the record that is to have them.
        auto find = [&](int slot) {
          ChunkRecord& rec = sh.record[slot];
          for (bool first = true; next < page_end; first = false) {
            cur.j0 = next * KC_PAGE;
            cur.desc = ahead_desc;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              cur.page[x] = __shfl_sync(0xffffffffu, batch_page, next - batch + x);
              cur.ks[x] = __shfl_sync(0xffffffffu, batch_ks, next - batch + x);
              cur.ev[x] = __shfl_sync(0xffffffffu, batch_ev, next - batch + x);
            }
            const bool single = is_alone();
            if (single) cur.page[1] = -1;
            if (cur.page[1] < 0) cur.ev[1] = cur.ev[0];   // (a page that is not there says nothing about scales)
            if (cur.page[0] < 0) cur.ev[0] = cur.ev[1];
            const uint32_t ctx = __ballot_sync(0xffffffffu, (cur.desc & TD_CTX) != 0u);
            next += single ? 1 : 2;
            if (!metadata) {
              if (cur.j0 >= rows.max_limit) return false;   // (the limits are no more than the length)
              peek();
              if (lane == 0) rec.words[1][r >> 5] = ctx;
              return true;
            }
            const uint32_t pre = __ballot_sync(0xffffffffu, (cur.desc & TD_PRE) != 0u), ins = __ballot_sync(0xffffffffu, (cur.desc & TD_INS) != 0u);
            peek();
            if (!first) named_bar_sync(1, 128);   // everyone has looked at the words of the tile before, in this slot
            if (lane == 0) {
              rec.words[0][r >> 5] = pre;
              rec.words[1][r >> 5] = ctx;
              rec.words[2][r >> 5] = ins;
            }
            named_bar_sync(1, 128);
            uint32_t any[3];
#pragma unroll
            for (int x = 0; x < 3; ++x) any[x] = rec.words[x][0] | rec.words[x][1] | rec.words[x][2] | rec.words[x][3];
            if (((rows.sees & TD_PRE) != 0u && any[0] != 0u) || ((rows.sees & TD_CTX) != 0u && any[1] != 0u) || (((rows.sees & TD_INS) != 0u || rows.spans != 0) && any[2] != 0u) ||
                ((rows.causal & TD_CTX) != 0u && any[1] != 0u && cur.j0 < rows.max_limit))
              return true;
          }
          return false;
        };
        const uint32_t place[2] = {chunk_place(row0, col), chunk_place(row0, col + 8)};   // of later rounds at fixed distances: 32 tokens 4 KB, a block 16 KB
        auto fetch = [&](const void* from, const float* scales) {
          const uint8_t *base[2], *scale[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const size_t row = block_index(c, max(cur.page[x], 0), it.h) * KC_PAGE + row0;
            base[x] = static_cast<const uint8_t*>(from) + (kBits == 8 ? row * D + col : row * (D / 2) + col / 2);
            scale[x] = kBits == 4 ? scales4(scales) + row * (D / K4_GROUP) + col / K4_GROUP : nullptr;
          }
#pragma unroll
          for (int i = 0; i < ROUNDS; ++i) {   // tokens 32 (i & 3) + row0, head dims 64 (i >> 2) + col
            const int x = (i & 3) >> 1;
            const bool there = cur.page[x] >= 0 && (i >> 2) * 64 + col < D;
            if constexpr (kBits == 8) {
              reg[i].v = make_uint4(0u, 0u, 0u, 0u);
              if (there) reg[i].v = __ldg(reinterpret_cast<const uint4*>(base[x] + (i & 1) * 32 * D + (i >> 2) * 64));
            } else {
              reg[i].v = make_uint2(0u, 0u);
              reg[i].scale = 0u;
              if (there) {
                reg[i].v = __ldg(reinterpret_cast<const uint2*>(base[x] + (i & 1) * 32 * (D / 2) + (i >> 2) * 32));
                reg[i].scale = __ldg(scale[x] + (i & 1) * 32 * (D / K4_GROUP) + (i >> 2) * 4);
              }
            }
          }
        };
        // A wait of one warp can run out while another's is met: with metadata all hear of it at a barrier that every one of them comes to, before the next words are exchanged.
        auto drop = [&](int which, int tile) {   // wait time-out test build: the first converter warp of CTA 0 takes the wait as one that has run out
#ifdef KD_TEST_DROP_LOAD
          if (shape.test_drop == which && blockIdx.x == 0 && warp == 4 && tile == 1) {
            raise_abort(&sh.abort, CH_SITE | 1 << 4 | which);
            return true;
          }
#endif
          return false;
        };
        int u = 0;   // tiles of this pass
        bool have = find(n_k % CH_RECORDS);
        if (have) fetch(c.k, c.k_scale);
        for (;; ++u) {
          // (K's place and the record's slot are free when the scores of the tile before are complete; the slot of two tiles before by then, too)
          if (u > 0) ok = ok && !drop(7, u) && wait(CB_S, n_t + u - 1, 1);
          if (metadata) ok = named_bar_all(1, 128, ok);
          if (!ok) break;
          ChunkRecord& rec = sh.record[(n_k + u) % CH_RECORDS];
          if (r == 0) {
            rec.ks[0] = cur.ks[0];
            rec.ks[1] = cur.ks[1];
            rec.ev[0] = cur.ev[0];
            rec.ev[1] = cur.ev[1];
            rec.j0 = cur.j0;
            rec.end = have ? 0 : 1;
          }
          if (have) {
            if (metadata) rec.desc[r] = cur.desc;
            store_tile<D, false>(sh.k, place, reg, nullptr, col);
          }
          fence_proxy_async_smem();
          __syncwarp();
#ifdef KD_TEST_DROP_LOAD
          if (shape.test_drop == 5 && blockIdx.x == 0 && u == 0) {
          } else
#endif
          if (lane == 0) mbar_arrive(bar(CB_K));
          if (!have) break;
          fetch(c.v, c.v_scale);
          have = find((n_k + u + 1) % CH_RECORDS);
          if (u > 0 && (drop(8, u) || !(ok = wait(CB_PV, n_t + u - 1, 1)))) {
            ok = false;
            continue;   // (to the barrier)
          }
          if (safe) store_tile<D, true>(sh.v, place, reg, sh.nan_bits + row0, col);
          else store_tile<D, false>(sh.v, place, reg, nullptr, col);
          fence_proxy_async_smem();
          __syncwarp();
#ifdef KD_TEST_DROP_LOAD
          if (shape.test_drop == 6 && blockIdx.x == 0 && u == 0) {
          } else
#endif
          if (lane == 0) mbar_arrive(bar(CB_V));
          if (have) fetch(c.k, c.k_scale);
        }
      } while (again(pass++));
      if (sh.abort.v != 0u || !shape.even) break;
    }
  } else {
    reg_alloc<CH_REGS_COMPUTE>();
    while (open_item()) {
      const Item it = sh.item.it;
      int pass = 0;
      do {
        const bool safe = pass == 1, far = safe && (sh.redo & 2u) != 0u;
        // ---------------------------------------- softmax ----------------------------------------
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, mS = tS + lanes, mO = tO + lanes;
        const RowMask mask = sh.mask[tid];
        const float factor = sh.factor[tid];
        const uint32_t idesc_s = make_idesc_f16(0, 0, 0, KC_ROWS, CH_TOKENS), idesc_o = make_idesc_f16(0, 0, 1, KC_ROWS, 64 * Sh::BLOCKS);
        const uint32_t hi = desc_hi_sw128();
        auto issue_scores = [&]() {   // of a tile whose K is there
          tc_fence_after_sync();
          const uint32_t q = desc_lo_kmajor(smem_u32(sh.q)), k = desc_lo_kmajor(smem_u32(sh.k));
#pragma unroll
          for (int i = 0; i < D / 16; ++i) mma_ss_uniform(tS, q + koff_kmajor(i), k + koff_kmajor(i), hi, idesc_s, i > 0 ? 1u : 0u);
          commit_uniform(bar(CB_S));
        };
        auto issue_values = [&](bool first) {   // with P and V there
          tc_fence_after_sync();
          const uint32_t v = desc_lo_mnmajor(smem_u32(sh.v));
#pragma unroll
          for (int i = 0; i < CH_TOKENS / 16; ++i) mma_ts_uniform(tO, tS + (i / 4) * 64 + (i & 3) * 8, v + koff_mnmajor(i), hi, idesc_o, !first || i > 0 ? 1u : 0u);
          commit_uniform(bar(CB_PV));
        };
        float ref = -INFINITY, sum = 0.f;
        Scales scales;
        int o_unit = 0;
        const float slack = far ? 0.f : KA_SLACK, offset = far ? 0.f : KA_OFFSET;   // (far: 8 - ref would round)
        uint32_t nan_cols[4] = {0u, 0u, 0u, 0u};
        bool ok = true;
        int u = 0;
        for (;; ++u) {
          if (!(ok = wait(CB_K, n_k + u, 0))) break;
          const ChunkRecord& rec = sh.record[(n_k + u) % CH_RECORDS];
          if (*const_cast<const volatile int*>(&rec.end) != 0) break;
          if (warp == 0) issue_scores();
          uint32_t w[4];
          row_words(mask, rec, metadata, lane, w);
          float kf[2] = {score_factor(kBits == 8 ? rec.ks[0] : 1.f, factor), score_factor(kBits == 8 ? rec.ks[1] : 1.f, factor)};
          // (far: both pages of a tile have one V scale, and it goes into the units of O)
          const int ev_tile = kBits == 8 ? rec.ev[0] : 0, ev[2] = {far ? 0 : ev_tile, far || kBits == 4 ? 0 : rec.ev[1]};
          if (safe) {
            if (!(ok = wait(CB_V, n_t + u, 0))) break;
            for (int j = 0; j < CH_TOKENS; ++j) {
              if ((w[j >> 5] >> (j & 31) & 1u) == 0u) continue;
              const uint4 n = *reinterpret_cast<const uint4*>(sh.nan_bits[j]);
              nan_cols[0] |= n.x;
              nan_cols[1] |= n.y;
              nan_cols[2] |= n.z;
              nan_cols[3] |= n.w;
            }
          }
          if (!(ok = wait(CB_S, n_t + u, 0))) break;
          tc_fence_after_sync();
          // Scores of 64 tokens (a page) in registers at a time: page 0's for its maximum alone, then page 1's, which stay there; after the exponentials of a half page its
          // registers take page 0's scores again.
          uint32_t x[2][32];
          if (far) {   // rounded scores in the place of the products
#pragma unroll 1
            for (int i = 0; i < CH_TOKENS; i += 16) {
              uint32_t y[16];
              tmem_ld16(mS + i, y);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__fmul_rn(__uint_as_float(y[j]), i < KC_PAGE ? kf[0] : kf[1]));
              tmem_st16(mS + i, y);
            }
            tmem_wait_st();
            kf[0] = kf[1] = 1.f;
          }
          auto masked = [&](uint32_t (&y)[32], uint32_t bits) {
            if (__all_sync(0xffffffffu, bits == 0xFFFFFFFFu)) return;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if ((bits & (1u << j)) == 0u) y[j] = 0xFF800000u;
          };
          auto highest = [&](const uint32_t (&y)[32]) {
            float m4[4] = {__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]), __uint_as_float(y[3])};
#pragma unroll
            for (int j = 4; j + 8 <= 32; j += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) m4[k] = fmax3(m4[k], __uint_as_float(y[j + k]), __uint_as_float(y[j + 4 + k]));
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], __uint_as_float(y[28 + k]));
            return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          };
          float top[2];
#pragma unroll
          for (int page = 0; page < 2; ++page) {
            tmem_ld32(mS + 64 * page, x[0]);
            tmem_ld32(mS + 64 * page + 32, x[1]);
            tmem_wait_ld();
            masked(x[0], w[2 * page]);
            masked(x[1], w[2 * page + 1]);
            top[page] = fmaxf(highest(x[0]), highest(x[1]));
          }
          const float high = fmaxf(fmaf(top[0], kf[0], static_cast<float>(ev[0])), fmaf(top[1], kf[1], static_cast<float>(ev[1])));
          if (kBits == 8) scales.see(min(ev[0], ev[1]), max(ev[0], ev[1]));
          else scales.apart = false;
          const bool up = high > ref + slack, down = scales.apart && below_reference(high, ref);
          const bool units = far && ev_tile != o_unit;   // the whole CTA
          if (__any_sync(0xffffffffu, up || down || units)) {
            float to = up ? high : ref, shrink = up ? fast_exp2(ref - to) : 1.f;
            if (kBits == 8 && scales.ever()) {
              to = up ? rintf(high) : down ? reference_below(high, ref, sum) : ref;
              shrink = rescale(ref, to);
            }
            const float shrink_o = units ? shrink * exp2i(o_unit - ev_tile) : shrink;
            scales.look(to);
            if (units) o_unit = ev_tile;
            if (u > 0 && __any_sync(0xffffffffu, units || (to != ref && ref != -INFINITY))) {   // O is complete: its last product came before these scores
#pragma unroll 1
              for (int i = 0; i < D; i += 16) {
                uint32_t y[16];
                tmem_ld16(mO + i, y);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * shrink_o);
                tmem_st16(mO + i, y);
              }
            }
            sum *= shrink;
            ref = to;
          }
          const float base = ref == -INFINITY ? 0.f : offset - ref;
#pragma unroll
          for (int half = 0; half < 4; ++half) {   // page 1's halves, then page 0's; P of a page over its first 32 columns
            const int page = half < 2 ? 1 : 0, part = half & 1;
            if (half >= 2) {
              tmem_wait_ld();   // (both halves' loads, at the first of them)
              masked(x[part], w[part]);
            }
            const float k = kf[page], add = base + static_cast<float>(ev[page]);
            const uint64_t k2 = pack_f32x2(k, k), add2 = pack_f32x2(add, add);
            uint64_t sums[2] = {0u, 0u};
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t y = fma_f32x2(pack_u32x2(x[part][2 * j], x[part][2 * j + 1]), k2, add2);
              const float a = fast_exp2(lo_f32x2(y)), b = fast_exp2(hi_f32x2(y));
              sums[j & 1] = add_f32x2(sums[j & 1], pack_f32x2(a, b));
              pk[j] = pack2<false>(a, b);
            }
            const uint64_t both = add_f32x2(sums[0], sums[1]);
            sum = fmaf(lo_f32x2(both) + hi_f32x2(both), exp2i(-ev[page]), sum);
            if (half < 2) tmem_ld32(mS + 32 * part, x[part]);
            tmem_st16(mS + 64 * page + 16 * part, pk);
          }
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(CB_P));
          if (warp == 0) {
            if (!(ok = wait(CB_V, n_t + u, 0) && wait(CB_P, n_t + u, 0))) break;
            issue_values(u == 0);
          }
        }
        if (ok && u > 0) ok = wait(CB_PV, n_t + u - 1, 0);
        tc_fence_after_sync();
        if (far) {   // as with the offset
          sum *= 256.f;
          o_unit += 8;
        }
        // ---- this row's output ----
        const int row = it.tile * KC_ROWS + tid;
        const bool live = mask.limit > 0, exists = row < shape.rows, whole = sh.item.here == sh.item.pages;
        const size_t part = sh.item.part;
        const int i = row / shape.G, hq = it.h * shape.G + row - i * shape.G;
        const float inv = (!whole ? 1.f : live && sum != 0.f ? 1.f / sum : 0.f) * exp2i(o_unit);   // (of far rows: O's units)
        bool bad = false;
        if (ok) {
          if (exists && whole) write_stats(p, ws, shape.stats, (static_cast<size_t>(it.b) * p.H + hq) * p.T + i, live, ref, sum);
          if (exists && !whole) ws.part_ml[part * KC_ROWS + tid] = make_float2(ref, sum);
          uint16_t* out = static_cast<uint16_t*>(p.o.ptr) + it.b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t;
          float* part_o = ws.part_o + (part * KC_ROWS + tid) * D;
#pragma unroll
          for (int d = 0; d < D; d += 16) {
            uint32_t x[16];
            if (u > 0) {
              tmem_ld16(mO + d, x);
              tmem_wait_ld();
            }
            float f[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              f[j] = u > 0 && inv != 0.f ? __uint_as_float(x[j]) * inv : 0.f;
              if (safe && inv != 0.f && (nan_cols[d >> 5] >> ((d & 16) + j) & 1u) != 0u) f[j] = __uint_as_float(0x7FC00000u);
              bad = bad || is_nan(f[j]);
            }
            if (exists && whole) {
              if (p.dtype == KD_BF16) store16<KD_BF16>(out + d, f);
              else store16<KD_F16>(out + d, f);
            } else if (exists) {
              store16<KD_F32>(part_o + d, f);
            }
          }
          tc_fence_before_sync();
        }
        if (bad || scales.met_far()) atomicOr(&sh.redo, (bad ? 1u : 0u) | (scales.met_far() ? 2u : 0u));
        if (tid == 0) sh.tiles = u;   // (the converters' count is the same)
        if (!ok && warp == 0) {   // what has been issued ends before TMEM is given back
          if (u > 0) drain_wait(bar(CB_PV), (n_t + u - 1) & 1);
          drain_wait(bar(CB_S), (n_t + u) & 1);
        }
      } while (again(pass++));
      if (sh.abort.v != 0u || !shape.even) break;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (tid == 0 && sh.abort.v != 0u) cache_report(c, sh.abort.v);
  if (warp == 4) tmem_dealloc(tS, 256);
}

template <int kBits, int D>
static cudaError_t launch_chunk(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  constexpr size_t kShared = sizeof(ChunkShared<D>);
  static_assert(kShared <= 113 * 1024, "two CTAs share an SM");
  static SmemOptIn opt_in;
  static SharedFirst shared_first;
  cudaError_t e = opt_in(cache_attention_chunk_kernel<kBits, D>, kShared);
  if (e == cudaSuccess) e = shared_first(cache_attention_chunk_kernel<kBits, D>);
  const int64_t items = static_cast<int64_t>(s.B) * c.H * a.tiles;
  return e != cudaSuccess ? e : launch_shares(a.ctas > 0 && a.even, cache_attention_chunk_kernel<kBits, D>, static_cast<unsigned>(a.ctas > 0 ? a.ctas : items), CH_THREADS, kShared, stream, c, s, p, a, ws);
}

}  // namespace kd
