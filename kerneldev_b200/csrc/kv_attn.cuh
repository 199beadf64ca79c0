// What the two kernels of the cache's attention share (kv_attn.cu: few query rows, kv_attn_chunk.cu: many): rows and their masks, how the pages
// are shared out, the parts that a join puts together.
#pragma once
#include <atomic>
#include <utility>

#include "kv_cache.cuh"

namespace kd {

constexpr float KA_OFFSET = 8.f, KA_SLACK = 6.f, KA_DEPTH = 12.f, KA_LOG2E = 1.4426950408889634f;
constexpr int KA_APART = 4;   // exponents of V scales that share a reference
// What products of halves are multiplied with to be scores: the K scale, up to 2^31, and the query row's factor. Not infinite, so that zeros stay 0 (a row's factor ends at 2^96: with
// sm_scale 1 that of numbers of 2^110), and not 0, so that masked scores stay -inf (where a float flushes it, every score is as good as 0).
__device__ __forceinline__ float row_factor(float sm_scale, int e) { return fminf(sm_scale * KA_LOG2E * exp2i(-e), 7.9e28f); }
__device__ __forceinline__ float score_factor(float k_scale, float row) { return fmaxf(k_scale * row, 1e-37f); }
// s - ref comes from one fused product, with the steps of the exact product, where a rounded score has steps of 2^-24 of its size: from 2^24 on (in powers of two) the largest
// probability could be any power of two, and the weights, which are from rounded scores, leave those of the statistics before. Rows that come across scores
// from here on are done once more from rounded scores (the second passes).
constexpr float KA_FAR = 65536.f;
__device__ __forceinline__ bool is_far(float ref) { return fabsf(ref) >= KA_FAR && fabsf(ref) != INFINITY; }

// What the mask needs of a query row. A row that does not exist, or sees nothing, has limit 0, sees 0 and a key that no descriptor matches.
struct RowMask {
  int limit;          // keys j < limit are no later than the row's own token (or all, without causality)
  uint32_t sees;      // classes seen wherever they are
  uint32_t causal;    // classes seen up to limit
  uint32_t span_key;  // see span_key_of_query
};

struct AttnShape {
  int G, rows, tiles;   // heads of a group, query rows of a key head, items that they are cut into
  int ctas;             // 0: a CTA for each (sequence, head, tile); else that many share the pages (FlatOrder)
  int spread;           // ... those beyond one for each item
  bool even;            // see FlatOrder
  int item_rows;        // query rows of an item
  int least;            // pages that such a CTA has at least
  bool stats;           // leave every row's maximum and sum for the weights
#ifdef KD_TEST_DROP_LOAD
  int test_drop;        // wait time-out test build: the converters of CTA 0 do not announce the first K (5) or V (6) tile, or one of their warps takes its second wait for S (7) or PV (8) as run out
#endif
  int score_rows;       // 0, or the rows of a key head rounded up to 2, 4 or 8: leave the scores too
};
// Workspace: the rows' statistics (float2 for each, with weights), then the parts (see FlatOrder): an item's rows of D floats, and their maxima and sums. With weights and
// few rows, every score (times log2(e)) as well: for each token of each key head of the table, score_rows of them.
struct AttnWorkspace {
  float* scores;
  float2* stats;
  float* part_o;
  float2* part_ml;
};

__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) > 0x7F800000u; }

// The reference of a row's exponents (see the head of kv_attn.cu). high: the largest s + ev of the tokens in hand, -inf where the row sees none, NaN where it has no number: neither moves it. Up it
// goes to the largest number itself, whose probability is then rounded without an error: the weight of one token is often most of a row's. Down only where the scale of the tokens
// in hand is the cause (apart). (With the limit for all tokens, 2 x 512 queries at 8192 took 200 us in place of 190: most rows of a hierarchical mask have tiles of which they see
// a few unlikely tokens.) From the first such tokens on it stays whole, so that it may move with every page and what has been added up is not rounded.
struct Scales {
  uint32_t seen = 64 + KC_EXP_MIN;   // the largest exponent so far + 64 (8 bits); 256: some were far below it; 512: a row was far (see KA_FAR). One register
  bool apart;                        // the ones in hand are far below it
  __device__ __forceinline__ void see(int low, int high) {
    const int top = max(static_cast<int>(seen & 255u), high + 64);
    apart = top - (low + 64) > KA_APART;
    seen = (seen & ~255u) | static_cast<uint32_t>(top) | (apart ? 256u : 0u);
  }
  __device__ __forceinline__ bool ever() const { return (seen & 256u) != 0u; }
  __device__ __forceinline__ void look(float ref) { seen |= is_far(ref) ? 512u : 0u; }
  __device__ __forceinline__ bool met_far() const { return (seen & 512u) != 0u; }
};
__device__ __forceinline__ bool below_reference(float high, float ref) { return high < ref - KA_DEPTH && high != -INFINITY; }
// Downwards no further than lets the row's sum reach 2^64: O is below 2^40 times that.
__device__ __forceinline__ float reference_below(float high, float ref, float sum) {
  const int room = max(64 - (static_cast<int>(__float_as_uint(sum) >> 23) - 127), 0);
  return fmaxf(rintf(high), ref - static_cast<float>(room));
}
// what was added up with reference `from` is worth with `to`: 2^(from - to), of whole numbers exactly, and 1 where nothing moves (-inf, too)
__device__ __forceinline__ float rescale(float from, float to) {
  const float x = from - to, y = fast_exp2(x), whole = __uint_as_float(static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x))) + 127) << 23);
  return from == to ? 1.f : x == rintf(x) ? whole : y;
}

// four numbers of a bfloat16 row, a lane each, to halves: times the power of two that brings the row's largest finite magnitude to 2^14; returns its exponent
__device__ __forceinline__ int row_to_halves(uint2& v) {
  auto size = [](uint32_t u) { return (u & 0x7FFFu) < 0x7F80u ? u & 0x7FFFu : 0u; };
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(size(v.x), size(v.x >> 16)), max(size(v.y), size(v.y >> 16))));
  const int e = top != 0u ? min(112, 14 - (static_cast<int>(top >> 7) - 127)) : 0;   // -113 .. 112: a float, as its inverse
  const float f = exp2i(e);
  const float2 a = unpack2<true>(v.x), b = unpack2<true>(v.y);
  v = make_uint2(pack2<false>(a.x * f, a.y * f), pack2<false>(b.x * f, b.y * f));
  return e;
}

struct Item {
  int b, h, tile, len;
};

template <bool kAhead = false>
__device__ __forceinline__ int query_count(const kd_cache& c, const kd_cache_queries& p, int b) {
  return p.q_lens != nullptr ? checked_count(c, length_word<kAhead>(p.q_lens + b), p.T) : p.T;
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

// How the pages are shared out. An item is a sequence, a head and a tile of rows that has a query. A flat order counts the units of all items: sequences in turn, each once for
// every head and tile. Two ways:
//   shares  an item of n pages goes to ceil(n / most) CTAs, evenly, and `most` is such that there are CTAs enough for all. A CTA has one item's pages alone.
//           The way of few items in one wave of CTAs: their time is mostly latency, and a CTA with two items has it twice (16 x 1357 tokens of 4 heads, 5 queries: 15 us, 20 with even pages).
//   even    every CTA of one wave has the same number of pages, wherever that begins and ends. The way of many items: 32 x 4096 tokens of 8 heads 42 us, 46 to 49 with
//           one to three waves of shares.
// The units of the flat order are CTAs or pages. 32 bits are enough: the host sees to it that there are fewer than 2^30 pages. A warp holds what it needs of the first 32
// sequences in its lanes; a loop over the ones behind reads them again, from L1: the code is what a CTA that starts waits for.
struct FlatPlace {
  int b, ht, at, units, len, tiles;   // ht: head * tiles + tile; unit `at` of `units` of the item; len and tiles: of the sequence
};
__device__ __forceinline__ int pages_of_length(int len) { return (len + KC_PAGE - 1) / KC_PAGE; }
template <bool kAhead = false>   // see length_word
struct FlatOrder {
  int held, held_tiles;       // length and tiles of sequence `lane`
  uint32_t most;              // pages of a unit
  uint32_t total;             // even: pages ...
  uint32_t ctas, each, more;  // ... and the CTAs that have them: `each`, and one more for the first `more`

  static __device__ __forceinline__ int length_of(const kd_cache& c, const kd_cache_seqs& s, int b) { return b < s.B ? sequence_length<kAhead>(c, s, b) : 0; }
  static __device__ __forceinline__ int tiles_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int b) {
    if (p.q_lens == nullptr) return shape.tiles;
    return b < s.B ? (query_count<kAhead>(c, p, b) * shape.G + shape.item_rows - 1) / shape.item_rows : 0;
  }
  __device__ __forceinline__ uint32_t units_of(int len) const { return (pages_of_length(len) + most - 1) / most; }
  __device__ __forceinline__ void look_up(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape) {
    const int lane = threadIdx.x & 31;
    held = length_of(c, s, lane);
    held_tiles = tiles_of(c, s, p, shape, lane);
    uint32_t n = pages_of_length(held) * held_tiles;
#pragma unroll 1
    for (int b = 32 + lane; b < s.B; b += 32) n += pages_of_length(length_of(c, s, b)) * tiles_of(c, s, p, shape, b);
    total = __reduce_add_sync(0xffffffffu, n) * c.H;
    if (shape.even) {
      most = 1;
      // (None of them has no page: the join reads a part of every CTA of an item.)
      ctas = max(min(static_cast<uint32_t>(shape.ctas), (total + shape.least - 1) / shape.least), 1u);
      each = total / ctas;
      more = total - each * ctas;
    } else {
      // sum of ceil(n / most) <= total / most + items <= CTAs
      most = max((total + shape.spread - 1) / shape.spread, static_cast<uint32_t>(shape.least));
    }
  }
  // even: a CTA's first page, and a page's CTA
  __device__ __forceinline__ uint32_t start(uint32_t cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ uint32_t cta_of(uint32_t page) const {
    const uint32_t longer = more * (each + 1);
    return page < longer ? page / (each + 1) : more + (page - longer) / each;
  }
  // whose a unit is; b < 0: nobody's
  __device__ __forceinline__ FlatPlace find(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, uint32_t unit) const {
    const int lane = threadIdx.x & 31;
    uint32_t before = 0;
#pragma unroll 1
    for (int base = 0; base < s.B; base += 32) {
      const int my_len = base == 0 ? held : length_of(c, s, base + lane), my_tiles = base == 0 ? held_tiles : tiles_of(c, s, p, shape, base + lane);
      const uint32_t mine = units_of(my_len);
      uint32_t upto = mine * my_tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, (before + upto) * c.H > unit);
      if (past != 0u) {
        const int l = __ffs(past) - 1, len = __shfl_sync(0xffffffffu, my_len, l), tiles_b = __shfl_sync(0xffffffffu, my_tiles, l);
        const uint32_t units = __shfl_sync(0xffffffffu, mine, l), rest = unit - (before + __shfl_sync(0xffffffffu, upto, l) - units * tiles_b) * c.H, ht = rest / units;
        return FlatPlace{base + l, static_cast<int>(ht), static_cast<int>(rest - ht * units), static_cast<int>(units), len, tiles_b};
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return FlatPlace{-1, 0, 0, 0, 0, 0};
  }
  // units of the sequences before b
  __device__ __forceinline__ uint32_t before(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int b) const {
    const int lane = threadIdx.x & 31;
    uint32_t n = lane < b ? units_of(held) * held_tiles : 0u;
#pragma unroll 1
    for (int i = 32 + lane; i < b; i += 32) n += units_of(length_of(c, s, i)) * tiles_of(c, s, p, shape, i);
    return __reduce_add_sync(0xffffffffu, n) * c.H;
  }
};

// What a CTA works on next: pages page0 .. page0 + here - 1 of the `pages` of an item. here < 0: nothing.
struct ItemShare {
  Item it;
  int page0, here, pages;
  uint32_t part;   // where its rows go if that is not all of the item
};
// done: pages that the CTA has worked on
__device__ __forceinline__ ItemShare share_of_cta(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, uint32_t done) {
  ItemShare r;
  r.here = -1;
  if (shape.ctas == 0) {
    if (done > 0) return r;
    const int HT = c.H * shape.tiles, b = blockIdx.x / HT, ht = blockIdx.x - b * HT, h = ht / shape.tiles;
    r.it = Item{b, h, ht - h * shape.tiles, sequence_length(c, s, b)};
    r.page0 = 0;
    r.pages = r.here = p.q_lens != nullptr && r.it.tile * shape.item_rows >= query_count(c, p, b) * shape.G ? 0 : pages_of_length(r.it.len);   // (rows without a query: zeros)
    return r;
  }
  FlatOrder<> order;
  order.look_up(c, s, p, shape);
  uint32_t unit = blockIdx.x, left = 0;
  if (shape.even) {
    if (blockIdx.x >= order.ctas) return r;
    unit = order.start(blockIdx.x) + done;
    left = order.start(blockIdx.x + 1) - unit;
    if (left == 0) return r;
  } else if (done > 0) {
    return r;
  }
  const FlatPlace f = order.find(c, s, p, shape, unit);
  if (f.b < 0) return r;
  const int h = f.ht / f.tiles;
  r.it = Item{f.b, h, f.ht - h * f.tiles, f.len};
  r.pages = pages_of_length(f.len);
  if (shape.even) {
    r.page0 = f.at;
    r.here = min(static_cast<int>(left), r.pages - f.at);
    r.part = 2 * blockIdx.x + (done > 0 ? 1 : 0);   // (what lies between its first and its last item is whole)
  } else {
    const int each = r.pages / f.units, more = r.pages - each * f.units;   // the first `more` shares have one page more
    r.page0 = f.at * each + min(f.at, more);
    r.here = each + (f.at < more ? 1 : 0);
    r.part = blockIdx.x;
  }
  return r;
}

// The parts of an item, for the kernels that join them, ahead of their wait for the kernel that makes them. `count` of them: `first`, then one every `step` from `next` on. One part alone is no part: its CTA has written the rows.
struct ItemParts {
  uint32_t first, next, step;
  int count;
  __device__ __forceinline__ uint32_t at(int k) const { return k == 0 ? first : next + (k - 1) * step; }
};
__device__ __forceinline__ ItemParts parts_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& shape, int b, int h, int tile, int len, int n_queries) {
  FlatOrder<true> order;
  order.look_up(c, s, p, shape);
  const int tiles = (n_queries * shape.G + shape.item_rows - 1) / shape.item_rows;
  const uint32_t units = tile < tiles ? order.units_of(len) : 0, first = order.before(c, s, p, shape, b) + (h * tiles + tile) * units;
  if (units == 0) return ItemParts{0, 0, 0, 0};
  if (!shape.even) return ItemParts{first, first + 1, 1, static_cast<int>(units)};
  const uint32_t c0 = order.cta_of(first), c1 = order.cta_of(first + units - 1);
  return ItemParts{2 * c0 + (order.start(c0) >= first ? 0 : 1), 2 * c0 + 2, 2, static_cast<int>(c1 - c0 + 1)};
}

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

// An SM divides its memory between L1 and shared memory anew only while it is idle, and beside the kernels before and behind it never is. So all kernels of a call
// ask for the division that the large ones need, and one that counts on a place for every CTA (even pages) starts when the kernel before has left: on an SM that
// never gets idle one CTA of 444 found no room until others ended, again and again, and 32 x 4096 tokens took 48 us in place of 42.
struct SharedFirst {
  std::atomic<uint64_t> done{0};   // bit d: asked on device d
  template <typename Kernel>
  cudaError_t operator()(Kernel kernel) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

// launch, without the early start where pages are shared evenly
template <typename... P, typename... A>
inline cudaError_t launch_shares(bool even, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
  if (!even) return launch(kernel, grid, block, smem, stream, std::forward<A>(args)...);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// kv_attn_chunk.cu
constexpr int KC_ROWS = 128, KC_CTAS = 2;   // query rows of an item, CTAs of an SM
int launch_attention_chunk(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream);

}  // namespace kd
