// What the two kernels of the cache's attention share (kv_attn.cu: few query rows, kv_attn_chunk.cu: many): rows and their masks, how the pages
// are shared out, the parts that a join puts together.
#pragma once
#include "kv_cache.cuh"

namespace kd {

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
  int G, rows, tiles;   // heads of a group, query rows of a key head, items that they are cut into
  int ctas;             // 0: a CTA for each (sequence, head, tile); else at most that many CTAs share all pages evenly
  int item_rows;        // query rows of an item
  int least;            // pages that such a CTA has at least
  bool stats;           // leave every row's maximum and sum for the weights
};
// Workspace: the rows' statistics (float2 for each, with weights), then for each CTA two parts: an item's rows of D floats, and their maxima and sums.
struct AttnWorkspace {
  float2* stats;
  float* part_o;
  float2* part_ml;
};

__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) > 0x7F800000u; }

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

// A row's output from its sum and accumulated values (scaled by 1 / sum): 16 bits, and its log-sum-exp and statistics.
__device__ __forceinline__ void write_stats(const kd_cache_queries& p, const AttnWorkspace& ws, bool stats, size_t row, bool live, float ref, float sum) {
  if (p.lse != nullptr) p.lse[row] = live && sum != 0.f ? ref - KA_OFFSET + log2f(sum) : -INFINITY;
  if (stats) ws.stats[row] = live && sum != 0.f ? make_float2(ref, __frcp_rn(sum)) : make_float2(0.f, 0.f);
}

// The flat order of all pages: sequences in turn, each once for every head and tile of rows that has a query, cut into even ranges for the CTAs. 32 bits are
// enough: the host sees to it that there are fewer than 2^30 pages. A warp holds the counts of the first 128 sequences, in its lanes.
struct FlatPlace {
  int b, ht, page, len, tiles;   // ht: head * tiles + tile; len and tiles: of the sequence; page: index within the item
};
__device__ __forceinline__ int pages_of_length(int len) { return (len + KC_PAGE - 1) / KC_PAGE; }
struct FlatOrder {
  static constexpr int HELD = 4;
  int held[HELD], held_tiles[HELD];   // lengths, tiles
  uint32_t total;             // pages
  uint32_t ctas, each, more;  // that share them: `each` pages, and one more for the first `more` CTAs

  static __device__ __forceinline__ int length_of(const kd_cache& c, const kd_cache_seqs& s, int b) { return b < s.B ? sequence_length(c, s, b) : 0; }
  static __device__ __forceinline__ int tiles_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int b) {
    return b < s.B ? (query_count(c, p, b) * shape.G + shape.item_rows - 1) / shape.item_rows : 0;
  }
  // of sequence 32 i + lane
  __device__ __forceinline__ int length(const kd_cache& c, const kd_cache_seqs& s, int i) const {
    if (i < HELD) return i == 0 ? held[0] : i == 1 ? held[1] : i == 2 ? held[2] : held[3];
    return length_of(c, s, 32 * i + (threadIdx.x & 31));
  }
  __device__ __forceinline__ int tiles(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int i) const {
    if (i < HELD) return i == 0 ? held_tiles[0] : i == 1 ? held_tiles[1] : i == 2 ? held_tiles[2] : held_tiles[3];
    return tiles_of(c, s, p, shape, 32 * i + (threadIdx.x & 31));
  }
  __device__ __forceinline__ void look_up(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape) {
    const int lane = threadIdx.x & 31;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      held[i] = length_of(c, s, 32 * i + lane);
      held_tiles[i] = tiles_of(c, s, p, shape, 32 * i + lane);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) n += pages_of_length(held[i]) * held_tiles[i];
    for (int b = 32 * HELD + lane; b < s.B; b += 32) n += pages_of_length(length_of(c, s, b)) * tiles_of(c, s, p, shape, b);
    total = __reduce_add_sync(0xffffffffu, n) * c.H;
    // (None of them has no page: the join reads a part of every CTA of an item.)
    ctas = max(min(static_cast<uint32_t>(shape.ctas), (total + shape.least - 1) / shape.least), 1u);
    each = total / ctas;
    more = total - each * ctas;
  }
  __device__ __forceinline__ uint32_t start(uint32_t cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ uint32_t cta_of(uint32_t page) const {
    const uint32_t longer = more * (each + 1);
    return page < longer ? page / (each + 1) : more + (page - longer) / each;
  }
  __device__ __forceinline__ FlatPlace find(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, uint32_t at) const {
    const int lane = threadIdx.x & 31;
    uint32_t before = 0;
    for (int i = 0; 32 * i < s.B; ++i) {
      const int my_len = length(c, s, i), my_tiles = tiles(c, s, p, shape, i);
      uint32_t upto = pages_of_length(my_len) * my_tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * c.H > at);
      if (past != 0u) {
        const int l = __ffs(past) - 1, len = __shfl_sync(0xffffffffu, my_len, l), n = pages_of_length(len), tiles_b = __shfl_sync(0xffffffffu, my_tiles, l);
        const uint32_t rest = at - (before + __shfl_sync(0xffffffffu, upto, l) - n * tiles_b) * c.H, ht = rest / static_cast<uint32_t>(n);
        return FlatPlace{32 * i + l, static_cast<int>(ht), static_cast<int>(rest - ht * n), len, tiles_b};
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return FlatPlace{-1, 0, 0, 0, 0};
  }
  // pages of the sequences before b
  __device__ __forceinline__ uint32_t before(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int b) const {
    const int lane = threadIdx.x & 31;
    uint32_t n = 0;
    for (int i = 0; 32 * i < b; ++i)
      if (32 * i + lane < b) n += pages_of_length(length(c, s, i)) * tiles(c, s, p, shape, i);
    return __reduce_add_sync(0xffffffffu, n) * c.H;
  }
};

// Reads a line of the kernel's parameters here and now. A first read takes as long as one of global memory, and longer once the loads of all CTAs are on
// their way: ahead of the wait for the kernel before, it costs nothing.
__device__ __forceinline__ void touch(uint32_t x) { asm volatile("" ::"r"(x)); }
__device__ __forceinline__ void touch_parameters(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, const AttnWorkspace& ws) {
  touch(c.pages);
  touch(s.blocks);
  touch(p.H);
  touch(static_cast<uint32_t>(p.q.stride_t));
  touch(static_cast<uint32_t>(p.o.stride_t));
  touch(p.causal);
  touch(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p.lse)));
  touch(static_cast<uint32_t>(p.w_len));
  touch(shape.G);
  touch(shape.least);
  touch(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ws.part_ml)));
}

// kv_attn_chunk.cu
constexpr int KC_ROWS = 128, KC_CTAS = 2;   // query rows of an item, CTAs of an SM
int launch_attention_chunk(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream);

}  // namespace kd
