// Attention of the newest tokens over the 8-bit cache, and the weight that each cached token receives.
//
// One key head at a time has few query rows (its group's heads times the new tokens), so what bounds these kernels is reading the cache: 2 D bytes
// a token. Every warp walks units of 32 tokens on its own, straight from memory to registers, with no shared tile and no barrier:
//   S = Q K^T   mma m16n8k16, 16 query rows; a lane's 16 bytes of a key row are the B operand of four steps (the order of the head dim
//               inside a step is free as long as Q's registers have the same)
//   P = exp2(S) stays in the registers that the second product takes it from (the accumulators of two 8-token tiles are the A operand of one step)
//   O += P V    a lane's 16 bytes of four value rows are the B operands of 16 column tiles: the columns of tile m are the
//               m-th bytes of the eight lanes' pieces, so that loads stay 16 bytes wide and no transpose is needed
// e4m3 numbers become halves by one instruction for two, exactly. Rounded are P (to a half: 2**-11, in place of the output's 2**-8 or 2**-11) and the output;
// bfloat16 queries become halves exactly, after a power of two for each row.
//
// Scales. A page's K scale multiplies its scores. Its V scale 2^ev goes into the exponent, p' = 2^(s + ev - ref), where ref is the
// running maximum of s + ev; then O = sum p' v / sum p' 2^-ev, and no product of its own is spent on it. The exponents differ by at most 63, which
// leaves p' far from the bottom of a float. p' is kept below 2^(8 + 6): the maximum is followed only in steps of 6 or more (the accumulators are rescaled then), and the offset
// of 8 keeps probabilities down to 2^-22 of the largest out of the half's subnormals: long tails keep their weight.
//
// NaN. A masked token has p' = 0, and 0 * NaN of a masked value would be NaN. A warp that ends with a NaN walks its units once more, with NaN values
// taken as zeros and, beside the product, one of indicators (row sees token, value is NaN) that puts NaN where it belongs.
#include <algorithm>

#include "attn_common.cuh"
#include "kv_cache.cuh"

namespace kd {

constexpr int KA_WARPS = 4, KA_THREADS = KA_WARPS * 32, KA_ROWS = 16, KA_UNIT = 32, KA_STAGES = 2, KA_CTAS = 3;   // CTAs of an SM
constexpr float KA_OFFSET = 8.f, KA_SLACK = 6.f, KA_LOG2E = 1.4426950408889634f;
constexpr float KA_TINY = 1e-37f;   // in place of factors that a float flushes to 0 (every score is as good as 0 then): masked scores stay -inf, and not 0 * inf

// What the mask needs of a query row. A row that does not exist, or sees nothing, has limit 0, sees 0 and a key that no descriptor matches.
struct RowMask {
  int limit;          // keys j < limit are no later than the row's own token (or all, without causality)
  uint32_t sees;      // classes seen wherever they are
  uint32_t causal;    // classes seen up to limit
  uint32_t span_key;  // see span_key_of_query
};

struct AttnShape {
  int G, rows, tiles;   // heads of a group, query rows of a key head, tiles of KA_ROWS of them
  int ctas;             // 0: a CTA for each (sequence, head, tile); else that many CTAs share all pages evenly
  bool stats;           // leave every row's maximum and sum for the weights
};
// Workspace: the rows' statistics (float2 for each, with weights), then for each CTA two parts: KA_ROWS rows of D floats, and their maxima and sums.
struct AttnWorkspace {
  float2* stats;
  float* part_o;
  float2* part_ml;
};

// ---- a unit in shared memory --------------------------------------------------------------------------------------

template <int N>
__device__ __forceinline__ void lds(uint32_t at, uint32_t* w) {
  if constexpr (N == 16) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  } else if constexpr (N == 8) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  } else if constexpr (N == 4) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
  } else {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at));
    w[0] = h;
  }
}
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// How a row of D bytes is spread over lanes. K: the four lanes t of a quad own pieces of KU bytes, 4 KU apart; V: the eight lanes g pieces of VU bytes.
template <int D>
struct Spread {
  static constexpr int KU = D % 64 == 0 ? 16 : D % 32 == 0 ? 8 : 4, K_PIECES = D / 4 / KU, K_WORDS = D / 16;
  static constexpr int VU = D == 128 ? 16 : D == 64 ? 8 : D % 32 == 0 ? 4 : 2, V_PIECES = D / 8 / VU, V_WORDS = V_PIECES * (VU > 4 ? VU / 4 : 1);
  static constexpr int TILES = D / 8;   // column tiles of O
  // the first of the head dims that lane t holds in step s of Q K^T; the step has four of them
  static __device__ __forceinline__ int k_dim(int s, int t) { return 4 * KU * (s / (KU / 4)) + KU * t + 4 * (s % (KU / 4)); }
  // the column of O that column n of tile m is
  static __device__ __forceinline__ int v_dim(int m, int n) { return 8 * VU * (m / VU) + VU * n + m % VU; }
};

// A warp's copy of a unit: K, V, descriptors, scales. Rows of 128 or 64 bytes would put all rows into the same banks: the 16-byte pieces of a
// row change places, so that the eight lanes of a part of a load (two g, four t) find theirs in eight different ones: for K by the row's lowest bit,
// for V by the two above it.
template <int D>
struct Stage {
  static constexpr int V_AT = KA_UNIT * D, DESC_AT = 2 * V_AT, SCALE_AT = DESC_AT + KA_UNIT * 4, BYTES = SCALE_AT + 128;
  static __device__ __forceinline__ uint32_t k_place(uint32_t o) { return D == 128 ? o ^ ((o >> 1) & 64u) : o; }
  static __device__ __forceinline__ uint32_t v_place(uint32_t o) { return D == 128 ? o ^ ((o >> 3) & 96u) : D == 64 ? o ^ ((o >> 2) & 96u) : o; }
};
// Where a lane finds things in its stage. The places of later steps and tokens are at fixed distances: the bits that a place depends on are the lane's own, but
// for every second step of V's copy at 128 bytes (bit 9) and V's odd tokens at 64 (bit 6).
template <int D>
struct Lane {
  uint32_t copy_k, copy_v[2], k[Spread<D>::K_PIECES], v[2];
  __device__ __forceinline__ Lane() {
    using S = Stage<D>;
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    copy_k = S::k_place(lane * 16);
    copy_v[0] = S::V_AT + S::v_place(lane * 16);
    copy_v[1] = S::V_AT + S::v_place(lane * 16 + 512);
#pragma unroll
    for (int i = 0; i < Spread<D>::K_PIECES; ++i) k[i] = S::k_place(g * D + 4 * Spread<D>::KU * i + Spread<D>::KU * t);
    v[0] = S::V_AT + S::v_place(2 * t * D + Spread<D>::VU * g);
    v[1] = S::V_AT + S::v_place((2 * t + 1) * D + Spread<D>::VU * g);
  }
  // one operand's bytes, 16 a lane and step
  template <bool kV>
  __device__ __forceinline__ void copy(uint32_t stage, const uint8_t* from) const {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) cp_async16(stage + (!kV ? copy_k + 512 * i : copy_v[i & 1] + 512 * (i & ~1)), from + (threadIdx.x & 31) * 16 + 512 * i);
  }
  // lane (g, t): its pieces of an 8-token tile of K
  __device__ __forceinline__ void load_keys(uint32_t stage, int j, uint32_t (&w)[Spread<D>::K_WORDS]) const {
    using S = Spread<D>;
#pragma unroll
    for (int i = 0; i < S::K_PIECES; ++i) lds<S::KU>(stage + k[i] + 8 * D * j, &w[i * (S::KU / 4)]);
  }
  // ... its pieces of the tokens 2t, 2t + 1, 2t + 8, 2t + 9 of 16
  __device__ __forceinline__ void load_values(uint32_t stage, int half, uint32_t (&w)[4][Spread<D>::V_WORDS]) const {
    using S = Spread<D>;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < S::V_PIECES; ++i) lds<S::VU>(stage + v[r & 1] + (16 * half + 8 * (r >> 1)) * D + 8 * S::VU * i, &w[r][i * (S::VU > 4 ? S::VU / 4 : 1)]);
  }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// S of a unit: 16 rows against 32 tokens. q: the A operands of every step, [step][lane]
template <int D>
__device__ __forceinline__ void scores(uint32_t stage, const Lane<D>& at, const uint4* q, float (&c)[4][4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int x = 0; x < 4; ++x) c[j][x] = 0.f;
  uint32_t k[4][Spread<D>::K_WORDS];
#pragma unroll
  for (int j = 0; j < 4; ++j) at.load_keys(stage, j, k[j]);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint4 a = q[s * 32 + lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const HalfPairs b = e4m3x4_to_f16x4(k[j][s]);
      mma_f16(c[j], a, b.lo, b.hi);
    }
  }
}

// bytes 0 and 1 (2 and 3) of two words in turn: for two tokens' values of two columns
__device__ __forceinline__ uint32_t interleave(uint32_t a, uint32_t b, bool high) { return __byte_perm(a, b, high ? 0x7362 : 0x5140); }
// the bytes that are NaN, as bytes of ones
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// O += P V for 16 tokens. kSafe: see the head of the file; vis: the A operand of indicators
template <int D, bool kSafe>
__device__ __forceinline__ void add_values(float (&o)[D / 8][4], const uint4& p, const uint4& vis, const uint32_t (&v)[4][Spread<D>::V_WORDS]) {
  using S = Spread<D>;
  constexpr int PER = S::VU >= 4 ? 4 : 2;   // columns of a word
#pragma unroll
  for (int w = 0; w < S::V_WORDS; ++w) {
#pragma unroll
    for (int half = 0; half < PER / 2; ++half) {
      uint32_t b0 = interleave(v[0][w], v[1][w], half != 0), b1 = interleave(v[2][w], v[3][w], half != 0);
      const int m = w * PER + 2 * half;
      if constexpr (kSafe) {
        const uint32_t n0 = nan_bytes(b0), n1 = nan_bytes(b1);
        b0 &= ~n0;
        b1 &= ~n1;
        const HalfPairs one0 = e4m3x4_to_f16x4(n0 & 0x38383838u), one1 = e4m3x4_to_f16x4(n1 & 0x38383838u);   // 0x38: 1 in e4m3
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float hit[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(hit, vis, x == 0 ? one0.lo : one0.hi, x == 0 ? one1.lo : one1.hi);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) o[m + x][i] = __uint_as_float(0x7FC00000u);
        }
      }
      const HalfPairs h0 = e4m3x4_to_f16x4(b0), h1 = e4m3x4_to_f16x4(b1);
      mma_f16(o[m], p, h0.lo, h1.lo);
      mma_f16(o[m + 1], p, h0.hi, h1.hi);
    }
  }
}

__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) > 0x7F800000u; }

// ---- query rows ---------------------------------------------------------------------------------------------------

struct Item {
  int b, h, tile, len;
};

__device__ __forceinline__ int query_count(const kd_cache& c, const kd_cache_queries& p, int b) {
  return p.q_lens != nullptr ? checked_count(c, p.q_lens[b], p.T) : p.T;
}

// one row's mask; r: row of the key head (query r / G of head r % G of the group)
__device__ __forceinline__ RowMask row_mask(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const Item& it, int r, int G, int rows, int n_queries) {
  const int i = r / G, at = it.len - n_queries + i;
  RowMask m{0, 0u, 0u, 1u};
  if (r >= rows || i >= n_queries || at < 0) return m;
  uint32_t d = pack_plain(true);
  m.limit = p.causal != 0 || c.desc != nullptr ? at + 1 : it.len;
  if (c.desc != nullptr) {
    const int page = page_of(c, s, it.b, at / KC_PAGE);
    d = page >= 0 ? c.desc[block_index(c, page, it.h) * KC_PAGE + at % KC_PAGE] : 0u;
    m.span_key = span_key_of_query(d);
  }
  m.sees = (d >> TD_SEES_SHIFT) & 7u;
  m.causal = d & TD_CTX;
  return m;
}

template <int D>
struct QueryTile {
  uint4 frag[D / 16][32];
  RowMask mask[KA_ROWS];
  float factor[KA_ROWS];   // what its products are to be multiplied with, sm_scale and log2(e) among it
  int min_limit;           // of the rows that see anything
};

// Q's tile as A operands in shared memory, all threads of the CTA; ends with a barrier. bfloat16 rows are multiplied with a power of two that brings the largest
// finite number to 2^14, so that halves hold them (what falls below a half's subnormals is 2^-38 of the largest).
template <int D>
__device__ __forceinline__ void load_queries(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const Item& it, int G, int rows, QueryTile<D>& q) {
  constexpr int PER = KA_ROWS / KA_WARPS;   // rows of a warp, four numbers of each to a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = 4 * lane;
  const bool bf16 = p.dtype == KD_BF16;
  uint2 v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = it.tile * KA_ROWS + warp * PER + i;
    v[i] = make_uint2(0u, 0u);
    if (row < rows && d < D) {
      const int n = row / G, hq = it.h * G + row - n * G;
      v[i] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q.ptr) + it.b * p.q.stride_b + hq * p.q.stride_h + n * p.q.stride_t + d);
    }
  }
  if (threadIdx.x < KA_ROWS) {
    const RowMask m = row_mask(c, s, p, it, it.tile * KA_ROWS + threadIdx.x, G, rows, query_count(c, p, it.b));
    q.mask[threadIdx.x] = m;
    const int low = __reduce_min_sync(0xFFFFu, m.limit > 0 ? m.limit : INT_MAX);
    if (threadIdx.x == 0) q.min_limit = low;
  }
  // the step and quad lane that hold dims d .. d + 3 (see Spread::k_dim)
  constexpr int KU = Spread<D>::KU;
  const int step = d / (4 * KU) * (KU / 4) + d % KU / 4, quad = d % (4 * KU) / KU;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = warp * PER + i;
    int e = 0;
    if (bf16) {
      auto size = [](uint32_t u) { return (u & 0x7FFFu) < 0x7F80u ? u & 0x7FFFu : 0u; };
      const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(size(v[i].x), size(v[i].x >> 16)), max(size(v[i].y), size(v[i].y >> 16))));
      if (top != 0u) e = max(-60, min(60, 14 - (static_cast<int>(top >> 7) - 127)));
      const float f = exp2i(e);
      const float2 a = unpack2<true>(v[i].x), b = unpack2<true>(v[i].y);
      v[i] = make_uint2(pack2<false>(a.x * f, a.y * f), pack2<false>(b.x * f, b.y * f));
    }
    if (lane == 0) q.factor[r] = p.sm_scale * KA_LOG2E * exp2i(-e);
    if (d < D) {   // registers 0 and 2 of the operand are those of rows 0 to 7, 1 and 3 of rows 8 to 15
      uint32_t* w = reinterpret_cast<uint32_t*>(&q.frag[step][(r & 7) * 4 + quad]) + (r >> 3);
      w[0] = v[i].x;
      w[2] = v[i].y;
    }
  }
  __syncthreads();
}

// masks the scores of a unit: token of c[j][x]: j0 + 8 j + 2 t + (x & 1), row of c[j][x]: lo or hi
__device__ __forceinline__ void mask_scores(float (&c)[4][4], const uint32_t* desc, int j0, int t, int end, const RowMask& lo, const RowMask& hi) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int token = j0 + 8 * j + 2 * t;
    uint2 d = make_uint2(TD_CTX, TD_CTX);
    if (desc != nullptr) d = *reinterpret_cast<const uint2*>(desc + 8 * j + 2 * t);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const RowMask& m = x < 2 ? lo : hi;
      const uint32_t kd = (x & 1) != 0 ? d.y : d.x;
      const int tok = token + (x & 1);
      const bool see = tok < end && ((kd & (tok < m.limit ? m.sees | m.causal : m.sees)) != 0u || span_match_key(m.span_key, kd) != 0u);
      if (!see) c[j][x] = -INFINITY;
    }
  }
}

// ---- the walk -----------------------------------------------------------------------------------------------------

// A warp's share of units first, first + KA_WARPS, ... below `last` of one head of a sequence, through a ring of copies of its own: while
// one unit is worked on, KA_STAGES - 1 are on their way. The accumulators' rows are lane / 4 and that plus 8.
template <int D>
struct Walker {
  float o[D / 8][4];
  float ref[2], sum[2];

  // starts the copies of a unit (nothing at or beyond `last`)
  static __device__ __forceinline__ void fetch(const kd_cache& c, const Lane<D>& place, int h, int unit, int last, int page, char* stage) {
    const int lane = threadIdx.x & 31;
    if (unit < last) {
      const uint32_t to = smem_u32(stage);
      page = checked_page(c, page);
      if (page >= 0) {
        const size_t at = block_index(c, page, h), token = at * KC_PAGE + (unit & 1) * KA_UNIT;
        place.template copy<false>(to, static_cast<const uint8_t*>(c.k) + token * D);
        place.template copy<true>(to, static_cast<const uint8_t*>(c.v) + token * D);
        if (c.desc != nullptr && lane < 8) cp_async16(to + Stage<D>::DESC_AT + lane * 16, c.desc + token + lane * 4);
        if (lane < 2) cp_async4(to + Stage<D>::SCALE_AT + lane * 4, (lane == 0 ? c.k_scale : c.v_scale) + at);
      } else if (lane < 2) {
        reinterpret_cast<float*>(stage + Stage<D>::SCALE_AT)[lane] = 1.f;   // (any bytes: all of it is masked)
      }
      if (lane == 0) *reinterpret_cast<int*>(stage + Stage<D>::SCALE_AT + 8) = page;
    }
    cp_async_commit();
  }
  // the ring's first copies, and the page of the unit behind them
  static __device__ __forceinline__ int begin(const kd_cache& c, const kd_cache_seqs& s, const Lane<D>& place, const Item& it, int first, int last, char* ring) {
    const int32_t* table = s.table + it.b * s.table_stride;
    auto page_at = [&](int i) { return first + i * KA_WARPS < last ? table[(first + i * KA_WARPS) >> 1] : -1; };
    int pages[KA_STAGES];
#pragma unroll
    for (int i = 0; i < KA_STAGES; ++i) pages[i] = page_at(i);
#pragma unroll
    for (int i = 0; i + 1 < KA_STAGES; ++i) fetch(c, place, it.h, first + i * KA_WARPS, last, pages[i], ring + i * Stage<D>::BYTES);
    return pages[KA_STAGES - 1];
  }

  // next_page: what begin returned
  template <bool kSafe>
  __device__ __forceinline__ void walk(const kd_cache& c, const kd_cache_seqs& s, const Lane<D>& place, const Item& it, const QueryTile<D>& q, int first, int last, int next_page, char* ring) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    ref[0] = ref[1] = -INFINITY;
    sum[0] = sum[1] = 0.f;
#pragma unroll
    for (int m = 0; m < D / 8; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[m][x] = 0.f;
    const int32_t* table = s.table + it.b * s.table_stride;
    const int free_end = c.desc != nullptr ? 0 : q.min_limit;   // units below it need no mask
    int slot = 0;
    for (int unit = first; unit < last; unit += KA_WARPS) {
      cp_async_wait<KA_STAGES - 2>();
      __syncwarp();   // everyone's copies of this unit are there, and everyone is done with the one before it, whose place the next one takes
      const int ahead = unit + (KA_STAGES - 1) * KA_WARPS;
      fetch(c, place, it.h, ahead, last, next_page, ring + (slot == 0 ? KA_STAGES - 1 : slot - 1) * Stage<D>::BYTES);
      if (ahead + KA_WARPS < last) next_page = table[(ahead + KA_WARPS) >> 1];
      const char* stage = ring + slot * Stage<D>::BYTES;
      const uint32_t at = smem_u32(stage);
      slot = slot + 1 == KA_STAGES ? 0 : slot + 1;
      const float* scale = reinterpret_cast<const float*>(stage + Stage<D>::SCALE_AT);
      const int page = reinterpret_cast<const int*>(scale)[2], j0 = unit * KA_UNIT;
      float sc[4][4];
      scores<D>(at, place, &q.frag[0][0], sc);
      const float k_lo = fmaxf(scale[0] * q.factor[g], KA_TINY), k_hi = fmaxf(scale[0] * q.factor[g + 8], KA_TINY);
      const int ev = scale_exponent(scale[1]);
      if (page < 0 || j0 + KA_UNIT > free_end)
        mask_scores(sc, c.desc != nullptr ? reinterpret_cast<const uint32_t*>(stage + Stage<D>::DESC_AT) : nullptr, j0, t, page < 0 ? 0 : it.len, q.mask[g], q.mask[g + 8]);
      // the rows' maxima over the quad
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top[0] = fmaxf(top[0], fmaxf(sc[j][0], sc[j][1]));
        top[1] = fmaxf(top[1], fmaxf(sc[j][2], sc[j][3]));
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        top[x] = fmaf(top[x], x == 0 ? k_lo : k_hi, static_cast<float>(ev));
      }
      if (__any_sync(0xffffffffu, top[0] > ref[0] + KA_SLACK || top[1] > ref[1] + KA_SLACK)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float to = top[x] > ref[x] + KA_SLACK ? top[x] : ref[x], shrink = to == ref[x] ? 1.f : fast_exp2(ref[x] - to);
          ref[x] = to;
          sum[x] *= shrink;
#pragma unroll
          for (int m = 0; m < D / 8; ++m) {
            o[m][2 * x] *= shrink;
            o[m][2 * x + 1] *= shrink;
          }
        }
      }
      const float a_lo = ref[0] == -INFINITY ? 0.f : static_cast<float>(ev) + KA_OFFSET - ref[0];
      const float a_hi = ref[1] == -INFINITY ? 0.f : static_cast<float>(ev) + KA_OFFSET - ref[1];
      uint4 pr[2], vis[2];
      if constexpr (kSafe) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          auto seen = [&](float a, float b) { return (a == -INFINITY ? 0u : 0x3C00u) | (b == -INFINITY ? 0u : 0x3C000000u); };
          vis[i] = make_uint4(seen(sc[2 * i][0], sc[2 * i][1]), seen(sc[2 * i][2], sc[2 * i][3]), seen(sc[2 * i + 1][0], sc[2 * i + 1][1]), seen(sc[2 * i + 1][2], sc[2 * i + 1][3]));
        }
      }
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sc[j][x] = fast_exp2(fmaf(sc[j][x], x < 2 ? k_lo : k_hi, x < 2 ? a_lo : a_hi));
          part[x >> 1] += sc[j][x];
        }
      const float unscale = exp2i(-ev);
      sum[0] = fmaf(part[0], unscale, sum[0]);
      sum[1] = fmaf(part[1], unscale, sum[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pr[i] = make_uint4(pack2<false>(sc[2 * i][0], sc[2 * i][1]), pack2<false>(sc[2 * i][2], sc[2 * i][3]), pack2<false>(sc[2 * i + 1][0], sc[2 * i + 1][1]),
                           pack2<false>(sc[2 * i + 1][2], sc[2 * i + 1][3]));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t v[4][Spread<D>::V_WORDS];
        place.load_values(at, i, v);
        add_values<D, kSafe>(o, pr[i], kSafe ? vis[i] : pr[i], v);
      }
    }
    cp_async_wait<0>();
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
      sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
    }
  }

  __device__ __forceinline__ bool any_nan() const {
    bool bad = false;
#pragma unroll
    for (int m = 0; m < D / 8; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) bad = bad || is_nan(o[m][x]);
    return __any_sync(0xffffffffu, bad);
  }
};

// A row's output from its sum and accumulated values (scaled by 1 / sum): 16 bits, and its log-sum-exp and statistics.
__device__ __forceinline__ void write_stats(const kd_cache_queries& p, const AttnWorkspace& ws, bool stats, size_t row, bool live, float ref, float sum) {
  if (p.lse != nullptr) p.lse[row] = live && sum != 0.f ? ref - KA_OFFSET + log2f(sum) : -INFINITY;
  if (stats) ws.stats[row] = live && sum != 0.f ? make_float2(ref, __frcp_rn(sum)) : make_float2(0.f, 0.f);
}

// The flat order of all pages: sequences in turn, each once for every head and tile. A warp holds the page counts of the first 128 sequences, in its lanes.
struct FlatPlace {
  int b, ht, page, pages;   // page: index within the item
};
struct FlatOrder {
  static constexpr int HELD = 4;
  int held[HELD];
  int64_t total;   // pages

  static __device__ __forceinline__ int pages_of(const kd_cache& c, const kd_cache_seqs& s, int b) { return b < s.B ? (sequence_length(c, s, b) + KC_PAGE - 1) / KC_PAGE : 0; }
  __device__ __forceinline__ int pages(const kd_cache& c, const kd_cache_seqs& s, int i) const {   // of sequence 32 i + lane
    if (i < HELD) return i == 0 ? held[0] : i == 1 ? held[1] : i == 2 ? held[2] : held[3];
    return pages_of(c, s, 32 * i + (threadIdx.x & 31));
  }
  __device__ __forceinline__ FlatOrder(const kd_cache& c, const kd_cache_seqs& s, int HT) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = pages_of(c, s, 32 * i + lane);
    int64_t n = held[0] + held[1] + held[2] + held[3];
    for (int b = 32 * HELD + lane; b < s.B; b += 32) n += pages_of(c, s, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total = n * HT;
  }
  __device__ __forceinline__ FlatPlace find(const kd_cache& c, const kd_cache_seqs& s, int HT, int64_t at) const {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int i = 0; 32 * i < s.B; ++i) {
      const int mine = pages(c, s, i);
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * HT > at);
      if (past != 0u) {
        const int l = __ffs(past) - 1, n = __shfl_sync(0xffffffffu, mine, l);
        const uint64_t rest = static_cast<uint64_t>(at - (before + __shfl_sync(0xffffffffu, upto, l) - n) * HT);   // less than n * HT
        const uint64_t ht = rest <= UINT32_MAX ? static_cast<uint32_t>(rest) / static_cast<uint32_t>(n) : rest / static_cast<uint32_t>(n);
        return FlatPlace{32 * i + l, static_cast<int>(ht), static_cast<int>(rest - ht * n), n};
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return FlatPlace{-1, 0, 0, 0};
  }
  // pages of the sequences before b
  __device__ __forceinline__ int64_t before(const kd_cache& c, const kd_cache_seqs& s, int b) const {
    const int lane = threadIdx.x & 31;
    int64_t n = 0;
    for (int i = 0; 32 * i < b; ++i)
      if (32 * i + lane < b) n += pages(c, s, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  }
};

// Shared memory of the kernel. A warp's rows of O take the place of its ring when it is through.
template <int D>
struct AttnShared {
  union {
    char ring[KA_STAGES * Stage<D>::BYTES];
    float o[KA_ROWS][D + 4];
  } warp[KA_WARPS];
  QueryTile<D> q;
  float2 ml[KA_WARPS][KA_ROWS];
};

// CTAs that share the pages: two pages, a unit for each warp, are the least that one takes. (None takes no page: the join reads a part of every CTA of an item.)
__device__ __forceinline__ int64_t sharing_ctas(const AttnShape& shape, int64_t total) { return min(static_cast<int64_t>(shape.ctas), (total + 1) / 2); }

template <int D>
__global__ void __launch_bounds__(KA_THREADS, KA_CTAS)
cache_attention_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                       const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(1024) char smem[];
  AttnShared<D>& sh = *reinterpret_cast<AttnShared<D>*>(smem);
  QueryTile<D>& q = sh.q;
  const Lane<D> place;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, HT = c.H * shape.tiles;
  int64_t at = 0, end = 1;
  const FlatOrder order(c, s, HT);
  if (shape.ctas > 0) {
    const int64_t total = order.total;
    const int64_t ctas = sharing_ctas(shape, total);
    if (blockIdx.x >= ctas) return;
    at = total * blockIdx.x / ctas;
    end = total * (blockIdx.x + 1) / ctas;
  }
  const int64_t begin = at;
  while (at < end) {
    Item it;
    int page0, pages, here;
    if (shape.ctas > 0) {
      const FlatPlace f = order.find(c, s, HT, at);
      it.b = f.b;
      it.h = f.ht / shape.tiles;
      it.tile = f.ht - it.h * shape.tiles;
      it.len = sequence_length(c, s, it.b);
      page0 = f.page;
      pages = f.pages;
      here = static_cast<int>(min(end - at, static_cast<int64_t>(pages - page0)));
    } else {
      const int item = blockIdx.x;
      it.b = item / HT;
      it.h = (item - it.b * HT) / shape.tiles;
      it.tile = item - it.b * HT - it.h * shape.tiles;
      it.len = sequence_length(c, s, it.b);
      page0 = 0;
      pages = here = (it.len + KC_PAGE - 1) / KC_PAGE;
    }
    const int first = 2 * page0 + warp, last = min(2 * (page0 + here), (it.len + KA_UNIT - 1) / KA_UNIT);
    char* ring = sh.warp[warp].ring;
    int next = Walker<D>::begin(c, s, place, it, first, last, ring);
    load_queries<D>(c, s, p, it, shape.G, shape.rows, q);
    Walker<D> w;
    w.template walk<false>(c, s, place, it, q, first, last, next, ring);
    if (w.any_nan()) {
      next = Walker<D>::begin(c, s, place, it, first, last, ring);
      w.template walk<true>(c, s, place, it, q, first, last, next, ring);
    }
    // the warps' parts: maxima and sums first, then everyone's rows on one scale
    if (t == 0) {
      sh.ml[warp][g] = make_float2(w.ref[0], w.sum[0]);
      sh.ml[warp][g + 8] = make_float2(w.ref[1], w.sum[1]);
    }
#pragma unroll
    for (int m = 0; m < D / 8; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) sh.warp[warp].o[g + 8 * (x >> 1)][Spread<D>::v_dim(m, 2 * t + (x & 1))] = w.o[m][x];
    __syncthreads();
    const int r = tid / 8, row_of_head = it.tile * KA_ROWS + r;
    if (row_of_head < shape.rows) {
      float ref = -INFINITY, sum = 0.f, scale[KA_WARPS];
#pragma unroll
      for (int i = 0; i < KA_WARPS; ++i) ref = fmaxf(ref, sh.ml[i][r].x);
#pragma unroll
      for (int i = 0; i < KA_WARPS; ++i) {
        scale[i] = sh.ml[i][r].x == -INFINITY ? 0.f : fast_exp2(sh.ml[i][r].x - ref);
        sum = fmaf(sh.ml[i][r].y, scale[i], sum);
      }
      const int i = row_of_head / shape.G, hq = it.h * shape.G + row_of_head - i * shape.G;
      const bool whole = here == pages, live = q.mask[r].limit > 0;
      const float inv = whole ? (live && sum != 0.f ? 1.f / sum : 0.f) : 1.f;
      const size_t part = 2 * static_cast<size_t>(blockIdx.x) + (at > begin ? 1 : 0);
      uint16_t* out = static_cast<uint16_t*>(p.o.ptr) + it.b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t;
      float* part_o = ws.part_o + (part * KA_ROWS + r) * D;
      for (int d = (tid & 7) * 2; d < D; d += 16) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int k = 0; k < KA_WARPS; ++k) {
          x = fmaf(sh.warp[k].o[r][d], scale[k], x);
          y = fmaf(sh.warp[k].o[r][d + 1], scale[k], y);
        }
        if (whole) {
          if (inv == 0.f) x = y = 0.f;
          *reinterpret_cast<uint32_t*>(out + d) = p.dtype == KD_BF16 ? pack2<true>(x * inv, y * inv) : pack2<false>(x * inv, y * inv);
        } else {
          *reinterpret_cast<float2*>(part_o + d) = make_float2(x, y);
        }
      }
      if ((tid & 7) == 0) {
        if (whole) write_stats(p, ws, shape.stats, (static_cast<size_t>(it.b) * p.H + hq) * p.T + i, live, ref, sum);
        else ws.part_ml[part * KA_ROWS + r] = make_float2(ref, sum);
      }
    }
    __syncthreads();   // shared memory is free for the next item
    at += shape.ctas > 0 ? here : 1;
  }
}

// One query row whose pages several CTAs shared: their parts on one scale. Four groups of 32 threads take parts in turn.
__global__ void __launch_bounds__(128)
cache_join_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                  const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ float s_o[4][128], s_sum[4];
  const int tid = threadIdx.x, lane = tid & 31, grp = tid >> 5, HT = c.H * shape.tiles;
  const int row_of_head = blockIdx.x % shape.rows, bh = blockIdx.x / shape.rows, b = bh / c.H, h = bh - b * c.H;
  const int tile = row_of_head / KA_ROWS, r = row_of_head - tile * KA_ROWS;
  const FlatOrder order(c, s, HT);
  const int64_t total = order.total, ctas = sharing_ctas(shape, total);
  const int len = sequence_length(c, s, b), pages = (len + KC_PAGE - 1) / KC_PAGE;
  const int64_t first = order.before(c, s, b) * HT + static_cast<int64_t>(h * shape.tiles + tile) * pages;   // the item's first page in the flat order
  int c0 = 0, c1 = -1;
  if (pages > 0) {
    c0 = static_cast<int>(((first + 1) * ctas - 1) / total);
    c1 = static_cast<int>(((first + pages) * ctas - 1) / total);
    if (c0 == c1) return;   // the one CTA has written the row
  }
  auto part_of = [&](int k) { return (2 * static_cast<size_t>(k) + (total * k / ctas >= first ? 0 : 1)) * KA_ROWS + r; };
  float ref = -INFINITY;
  for (int k = c0 + lane; k <= c1; k += 32) ref = fmaxf(ref, ws.part_ml[part_of(k)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  const int d = lane * 4;
#pragma unroll 4
  for (int k = c0 + grp; k <= c1; k += 4) {
    const size_t part = part_of(k);
    const float2 ml = ws.part_ml[part];
    if (ml.x == -INFINITY) continue;
    const float scale = fast_exp2(ml.x - ref);
    sum = fmaf(ml.y, scale, sum);
    if (d < c.D) {
      const float4 v = *reinterpret_cast<const float4*>(ws.part_o + part * c.D + d);
      acc[0] = fmaf(v.x, scale, acc[0]);
      acc[1] = fmaf(v.y, scale, acc[1]);
      acc[2] = fmaf(v.z, scale, acc[2]);
      acc[3] = fmaf(v.w, scale, acc[3]);
    }
  }
  if (d < c.D)
#pragma unroll
    for (int x = 0; x < 4; ++x) s_o[grp][d + x] = acc[x];
  if (lane == 0) s_sum[grp] = sum;
  __syncthreads();
  const int i = row_of_head / shape.G, hq = h * shape.G + row_of_head - i * shape.G, n = query_count(c, p, b);
  const bool live = i < n && len - n + i >= 0;
  sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  const float inv = live && sum != 0.f ? 1.f / sum : 0.f;
  if (tid < c.D) {
    const float x = inv == 0.f ? 0.f : (s_o[0][tid] + s_o[1][tid] + s_o[2][tid] + s_o[3][tid]) * inv;
    uint16_t* out = static_cast<uint16_t*>(p.o.ptr) + b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t;
    out[tid] = static_cast<uint16_t>(p.dtype == KD_BF16 ? pack2<true>(x, 0.f) : pack2<false>(x, 0.f));
  }
  if (tid == 0) write_stats(p, ws, shape.stats, (static_cast<size_t>(b) * p.H + hq) * p.T + i, live, ref, sum);
}

// weights[j] += sum over the query rows of the head of softmax_j, from the rows' maxima and sums. A warp has a unit of tokens for all
// rows, so that nothing is added twice and the order is fixed; a CTA KW_PAGES pages of one head.
constexpr int KW_PAGES = 4, KW_UNITS = 2 * KW_PAGES;
template <int D>
__global__ void __launch_bounds__(KA_THREADS)
cache_weights_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                     const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int MINE = KW_UNITS / KA_WARPS;
  extern __shared__ __align__(1024) char smem[];
  char* stages = smem + (threadIdx.x >> 5) * MINE * Stage<D>::BYTES;
  QueryTile<D>& q = *reinterpret_cast<QueryTile<D>*>(smem + KW_UNITS * Stage<D>::BYTES);
  __shared__ float2 s_stat[KA_ROWS];
  const Lane<D> place;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, groups = (s.blocks + KW_PAGES - 1) / KW_PAGES;
  uint32_t item = blockIdx.x;
  const int first = static_cast<int>(item % static_cast<uint32_t>(groups)) * KW_UNITS + warp;
  item /= static_cast<uint32_t>(groups);
  Item it;
  it.h = static_cast<int>(item % static_cast<uint32_t>(c.H));
  it.b = static_cast<int>(item / static_cast<uint32_t>(c.H));
  it.len = sequence_length(c, s, it.b);
  if ((first - warp) * KA_UNIT >= it.len) return;
  int page[MINE];
  float ks[MINE], sums[MINE][8];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int unit = first + i * KA_WARPS;
    page[i] = unit * KA_UNIT < it.len ? page_of(c, s, it.b, unit >> 1) : -1;
    ks[i] = 1.f;
    if (page[i] >= 0) {
      const size_t at = block_index(c, page[i], it.h), token = at * KC_PAGE + (unit & 1) * KA_UNIT;
      const uint32_t to = smem_u32(stages + i * Stage<D>::BYTES);
      place.template copy<false>(to, static_cast<const uint8_t*>(c.k) + token * D);
      if (c.desc != nullptr && lane < 8) cp_async16(to + Stage<D>::DESC_AT + lane * 16, c.desc + token + lane * 4);
      ks[i] = c.k_scale[at];
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) sums[i][x] = 0.f;
  }
  cp_async_commit();
  for (it.tile = 0; it.tile < shape.tiles; ++it.tile) {
    load_queries<D>(c, s, p, it, shape.G, shape.rows, q);
    if (tid < KA_ROWS) {
      const int r = it.tile * KA_ROWS + tid, i = r / shape.G;
      s_stat[tid] = r < shape.rows ? ws.stats[(static_cast<size_t>(it.b) * p.H + it.h * shape.G + r - i * shape.G) * p.T + i] : make_float2(0.f, 0.f);
    }
    cp_async_wait<0>();
    __syncthreads();
    const float2 st[2] = {s_stat[g], s_stat[g + 8]};
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (page[i] < 0) continue;
      const char* stage = stages + i * Stage<D>::BYTES;
      const int j0 = (first + i * KA_WARPS) * KA_UNIT;
      float sc[4][4];
      scores<D>(smem_u32(stage), place, &q.frag[0][0], sc);
      if (c.desc != nullptr || j0 + KA_UNIT > q.min_limit)
        mask_scores(sc, c.desc != nullptr ? reinterpret_cast<const uint32_t*>(stage + Stage<D>::DESC_AT) : nullptr, j0, t, it.len, q.mask[g], q.mask[g + 8]);
      const float f[2] = {fmaxf(q.factor[g] * ks[i], KA_TINY), fmaxf(q.factor[g + 8] * ks[i], KA_TINY)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float pr = fast_exp2(fmaf(sc[j][x], f[x >> 1], KA_OFFSET - st[x >> 1].x)) * st[x >> 1].y;
          if (st[x >> 1].y != 0.f && sc[j][x] != -INFINITY) sums[i][2 * j + (x & 1)] += pr;   // rows that exist, tokens that they see
        }
    }
    __syncthreads();   // the tile in shared memory is free
  }
#pragma unroll
  for (int i = 0; i < MINE; ++i)
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      sums[i][x] += __shfl_xor_sync(0xffffffffu, sums[i][x], 4);
      sums[i][x] += __shfl_xor_sync(0xffffffffu, sums[i][x], 8);
      sums[i][x] += __shfl_xor_sync(0xffffffffu, sums[i][x], 16);
      const int j = (first + i * KA_WARPS) * KA_UNIT + 8 * (x >> 1) + 2 * t + (x & 1);
      if (g == 0 && page[i] >= 0 && j < it.len && j < p.w_len) p.weights[it.b * p.w_stride_b + it.h * p.w_stride_h + j] += sums[i][x];
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------

static AttnShape shape_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p) {
  AttnShape a;
  a.G = p.H / c.H;
  a.rows = a.G * p.T;
  a.tiles = (a.rows + KA_ROWS - 1) / KA_ROWS;
  a.stats = p.weights != nullptr;
  const int64_t items = static_cast<int64_t>(s.B) * c.H * a.tiles;
  // Up to eight pages a head, or with many heads for each SM, a CTA takes whole heads and nothing is joined.
  a.ctas = s.blocks <= 8 || items > 148 * 16 ? 0 : 148 * KA_CTAS;
  return a;
}

static size_t workspace_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, char* base, AttnWorkspace* ws) {
  size_t n = 0;
  auto take = [&](size_t bytes) {
    char* at = base + n;
    n += (bytes + 255) & ~size_t(255);
    return at;
  };
  ws->stats = reinterpret_cast<float2*>(take(a.stats ? static_cast<size_t>(s.B) * p.H * p.T * sizeof(float2) : 0));
  ws->part_o = reinterpret_cast<float*>(take(size_t(2) * a.ctas * KA_ROWS * c.D * sizeof(float)));
  ws->part_ml = reinterpret_cast<float2*>(take(size_t(2) * a.ctas * KA_ROWS * sizeof(float2)));
  return n;
}

size_t cache_attention_workspace(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p) {
  AttnWorkspace ws;
  return workspace_of(c, s, p, shape_of(c, s, p), nullptr, &ws);
}

template <int D>
static int launch_for(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  const int64_t heads = static_cast<int64_t>(s.B) * c.H, items = heads * a.tiles, rows = heads * a.rows, groups = heads * ((s.blocks + KW_PAGES - 1) / KW_PAGES);
  if (items > INT32_MAX || rows > INT32_MAX || (a.stats && groups > INT32_MAX)) return set_error(KD_ERR_LIMIT, "%d sequences of %d blocks are too many for one call", s.B, s.blocks);
  constexpr size_t kShared = sizeof(AttnShared<D>), kWeights = KW_UNITS * Stage<D>::BYTES + sizeof(QueryTile<D>);
  static SmemOptIn opt_in, opt_in_weights;
  cudaError_t e = opt_in(cache_attention_kernel<D>, kShared);
  if (e == cudaSuccess) e = launch(cache_attention_kernel<D>, static_cast<unsigned>(a.ctas > 0 ? a.ctas : items), KA_THREADS, kShared, stream, c, s, p, a, ws);
  if (e == cudaSuccess && a.ctas > 0) e = launch(cache_join_kernel, static_cast<unsigned>(rows), 128, 0, stream, c, s, p, a, ws);
  if (e == cudaSuccess && a.stats && groups > 0) {
    e = opt_in_weights(cache_weights_kernel<D>, kWeights);
    if (e == cudaSuccess) e = launch(cache_weights_kernel<D>, static_cast<unsigned>(groups), KA_THREADS, kWeights, stream, c, s, p, a, ws);
  }
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_attention launch: %s", cudaGetErrorString(e));
  return 0;
}

int launch_cache_attention(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, cudaStream_t stream) {
  const AttnShape a = shape_of(c, s, p);
  AttnWorkspace ws;
  workspace_of(c, s, p, a, static_cast<char*>(p.workspace), &ws);
  switch (c.D) {
    case 16: return launch_for<16>(c, s, p, a, ws, stream);
    case 32: return launch_for<32>(c, s, p, a, ws, stream);
    case 48: return launch_for<48>(c, s, p, a, ws, stream);
    case 64: return launch_for<64>(c, s, p, a, ws, stream);
    case 80: return launch_for<80>(c, s, p, a, ws, stream);
    case 96: return launch_for<96>(c, s, p, a, ws, stream);
    case 112: return launch_for<112>(c, s, p, a, ws, stream);
    default: return launch_for<128>(c, s, p, a, ws, stream);
  }
}

}  // namespace kd
