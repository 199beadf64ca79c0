// The cache's attention as a call: how its work is cut, the kernels that join what several CTAs have shared, and the launches. The kernels that read the cache are in
// kv_attn_rows.cuh (few query rows) and kv_attn_chunk.cuh (many), compiled for each number format.
#include <stdlib.h>

#include <algorithm>

#include "attn_common.cuh"
#include "kv_attn.cuh"

namespace kd {

// One query row whose pages several CTAs shared: their parts on one scale, and its output. kGroups warps take the parts in turn (grp: this warp's number; with more than
// one they are the whole CTA, and meet at barriers).
constexpr int KJ_WARPS = 8;
// A part whose row has seen nothing. NaN scores leave the maximum at -inf as well (no comparison with them holds), but make the sum NaN: such a part makes the row NaN.
__device__ __forceinline__ bool empty_part(const float2& ml) { return ml.x == -INFINITY && ml.y == 0.f; }
struct JoinShared {
  float4 o[KJ_WARPS][32];
  float2 ml[KJ_WARPS];
};
template <int kGroups>
__device__ __forceinline__ void join_row(const kd_cache& c, const kd_cache_queries& p, const AttnShape& shape, const AttnWorkspace& ws, const ItemParts& parts, int b, int h,
                                         int row_of_head, int len, int n, int grp, JoinShared* sh) {
  const int lane = threadIdx.x & 31, d = lane * 4, r = row_of_head % shape.item_rows;
  float ref = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = grp; k < parts.count; k += kGroups) {
    const size_t part = static_cast<size_t>(parts.at(k)) * shape.item_rows + r;
    const float2 ml = ws.part_ml[part];
    const float4 v = d < c.D ? *reinterpret_cast<const float4*>(ws.part_o + part * c.D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (empty_part(ml)) continue;
    const float to = fmaxf(ref, ml.x), keep = ref == to ? 1.f : fast_exp2(ref - to), scale = ml.x == to ? 1.f : fast_exp2(ml.x - to);
    ref = to;
    sum = fmaf(ml.y, scale, sum * keep);
    acc = make_float4(fmaf(v.x, scale, acc.x * keep), fmaf(v.y, scale, acc.y * keep), fmaf(v.z, scale, acc.z * keep), fmaf(v.w, scale, acc.w * keep));
  }
  if constexpr (kGroups > 1) {
    sh->o[grp][lane] = acc;
    if (lane == 0) sh->ml[grp] = make_float2(ref, sum);
    __syncthreads();
    if (grp == 0) {
      ref = -INFINITY;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) ref = fmaxf(ref, sh->ml[k].x);
      sum = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        if (empty_part(sh->ml[k])) continue;
        const float scale = fast_exp2(sh->ml[k].x - ref);   // (all maxima -inf: NaN, as the sums are then)
        const float4 v = sh->o[k][lane];
        sum = fmaf(sh->ml[k].y, scale, sum);
        acc = make_float4(fmaf(v.x, scale, acc.x), fmaf(v.y, scale, acc.y), fmaf(v.z, scale, acc.z), fmaf(v.w, scale, acc.w));
      }
    }
    __syncthreads();   // (for the next row)
    if (grp > 0) return;
  }
  const int i = row_of_head / shape.G, hq = h * shape.G + row_of_head - i * shape.G;
  const bool live = i < n && len - n + i >= 0;
  const float inv = 1.f / sum;
  if (!live || sum == 0.f) acc = make_float4(0.f, 0.f, 0.f, 0.f);
  else acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  if (d < c.D) {
    uint16_t* out = static_cast<uint16_t*>(p.o.ptr) + b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t + d;
    *reinterpret_cast<uint2*>(out) = p.dtype == KD_BF16 ? make_uint2(pack2<true>(acc.x, acc.y), pack2<true>(acc.z, acc.w)) : make_uint2(pack2<false>(acc.x, acc.y), pack2<false>(acc.z, acc.w));
  }
  if (lane == 0) write_stats(p, ws, shape.stats, (static_cast<size_t>(b) * p.H + hq) * p.T + i, live, ref, sum);
}

// The rows of all items: eight warps for a row where there are few rows (a long context has dozens of parts), one where there are many. Rows without a query, and those of
// sequences without a token, get their zeros here. What it needs to know of the lengths was there before the kernel ahead of it, so it is looked up while that one runs.
// kRows: rows of a warp, of one item: what it has to know of the lengths is then looked up once for all of them (512 queries each of 2 x 8192 tokens of 8 heads, 4 rows a query: 30,000 warps went through
// all lengths and divisions for a row each, and the join took 35 us, so 27).
template <int kGroups, int kRows>
__global__ void __launch_bounds__(KJ_WARPS * 32)
cache_join_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                  const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  constexpr int ROWS = KJ_WARPS / kGroups * kRows;
  static_assert(kGroups == 1 || ROWS == 1, "join_row's barriers are the whole CTA's");
  __shared__ JoinShared sh;
  const int warp = threadIdx.x >> 5, per_head = (shape.rows + ROWS - 1) / ROWS;
  const int bh = blockIdx.x / per_head, b = bh / c.H, h = bh - b * c.H, first_row = (blockIdx.x - bh * per_head) * ROWS;
  const int len = sequence_length<true>(c, s, b), n = query_count<true>(c, p, b);
  const ItemParts parts = parts_of(c, s, p, shape, b, h, first_row / shape.item_rows, len, n);
  pdl_wait();
  pdl_launch_dependents();
  if (parts.count == 1) return;   // the one CTA has written the rows
#pragma unroll 1
  for (int row = first_row + warp / kGroups; row < min(first_row + ROWS, shape.rows); row += KJ_WARPS / kGroups)
    join_row<kGroups>(c, p, shape, ws, parts, b, h, row, len, n, warp % kGroups, &sh);
}

// The weights of few rows, from the scores that the kernel ahead has left, and the join: a CTA has KS_TOKENS tokens of a head, the first ones of a head its rows too. (One launch
// less, and K is not read again: with cache_weights_kernel behind cache_join_kernel 8 x 4096 tokens of 8 heads of 128 took 31 us, so 24.)
constexpr int KS_TOKENS = 1024;
__global__ void __launch_bounds__(KJ_WARPS * 32)
cache_join_weights_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                          const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  __shared__ JoinShared sh;
  __shared__ float2 s_stat[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = (s.blocks * KC_PAGE + KS_TOKENS - 1) / KS_TOKENS;
  const int bh = blockIdx.x / groups, group = blockIdx.x - bh * groups, b = bh / c.H, h = bh - b * c.H;
  const int len = sequence_length<true>(c, s, b), n = query_count<true>(c, p, b);
  if (group * KS_TOKENS >= len && group > 0) return;
  ItemParts parts{0, 0, 0, 1};
  if (shape.ctas > 0) parts = parts_of(c, s, p, shape, b, h, 0, len, n);
  pdl_wait();
  pdl_launch_dependents();
  if (parts.count != 1)
    for (int r = group; r < shape.rows; r += max((len + KS_TOKENS - 1) / KS_TOKENS, 1)) join_row<KJ_WARPS>(c, p, shape, ws, parts, b, h, r, len, n, warp, &sh);
  // the rows' maxima and sums, a warp for each (what join_row leaves in the workspace may be another CTA's work)
  if (warp < shape.rows) {
    const int i = warp / shape.G, hq = h * shape.G + warp - i * shape.G;
    float2 st;
    if (parts.count == 1) {
      st = ws.stats[(static_cast<size_t>(b) * p.H + hq) * p.T + i];
    } else {
      float ref = -INFINITY, sum = 0.f;
      for (int k = lane; k < parts.count; k += 32) {
        const float2 ml = ws.part_ml[static_cast<size_t>(parts.at(k)) * shape.item_rows + warp];
        if (empty_part(ml)) continue;
        const float to = fmaxf(ref, ml.x);
        sum = sum * fast_exp2(ref - to) + ml.y * fast_exp2(ml.x - to);   // (both maxima -inf: NaN, as the part's sum is then)
        ref = to;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, ref, o), other_sum = __shfl_xor_sync(0xffffffffu, sum, o), to = fmaxf(ref, other);
        sum = to != -INFINITY ? sum * fast_exp2(ref - to) + other_sum * fast_exp2(other - to) : sum + other_sum;
        ref = to;
      }
      const bool live = i < n && len - n + i >= 0;
      st = live && sum != 0.f ? make_float2(ref, __frcp_rn(sum)) : make_float2(0.f, 0.f);
    }
    if (lane == 0) s_stat[warp] = st;
  }
  __syncthreads();
  const float* scores = ws.scores + static_cast<size_t>(bh) * s.blocks * KC_PAGE * shape.score_rows;
  float* weights = p.weights + b * p.w_stride_b + h * p.w_stride_h;
#pragma unroll
  for (int x = 0; x < KS_TOKENS; x += KJ_WARPS * 32) {
    const int j = group * KS_TOKENS + x + tid;
    if (j >= len || j >= p.w_len) continue;
    float add = 0.f;
    for (int r = 0; r < shape.score_rows; r += 2) {
      const float2 v = *reinterpret_cast<const float2*>(scores + static_cast<size_t>(j) * shape.score_rows + r);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float score = y == 0 ? v.x : v.y;
        const float2 st = r + y < shape.rows ? s_stat[r + y] : make_float2(0.f, 0.f);
        if (st.y != 0.f && score != -INFINITY) add += fast_exp2((score - st.x) + KA_OFFSET) * st.y;   // rows that exist, tokens that they see
      }
    }
    weights[j] += add;
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------

// Rows of an item: as many tiles of eight as the rows fill, up to four; beyond CHUNK_FROM rows the items are those of the kernel for many rows, which fills its 128 rows up, but would be two or
// more items here, that read the cache as often. us here and there: 8 x 4096 tokens of 8 heads of 128, 20 rows 33 and 42, 32 rows 34 and 40, 36 rows 52 and 41, 64 rows 53 and 42; 32 x 4096, 32 rows
// 98 and 143, 36 rows 168 and 145. (2 x 1300 tokens of 4 heads of 64 would be faster here further on: 36 rows 14 and 21, 64 rows 17 and 22.)
constexpr int CHUNK_FROM = 32;
static int rows_of_item(int rows) { return rows > CHUNK_FROM ? KC_ROWS : rows <= KA_TILE ? KA_TILE : rows <= 2 * KA_TILE ? 2 * KA_TILE : 4 * KA_TILE; }

// The scores that few rows leave for the weights: 4 bytes for each row and token of the page table (by its width, for the lengths are on the device), 4.3 GB for 128 sequences of 8 heads, 8 rows and
// tables for 131,072 tokens. Beyond 256 MB, and an eighth of what the cache itself takes, K is read and multiplied again instead (cache_weights_kernel): 32 sequences of 8192 tokens, 8 heads of 128, 8 rows
// 137 us with the scores and 179 without; 64 sequences 276 and 350; 1 of 131,072 70 and 99; 8 of 4096, 4 rows, 21 and 34.
constexpr size_t KA_SCORES_LIMIT = size_t(256) << 20;
static size_t scores_bytes(const kd_cache& c, const kd_cache_seqs& s, const AttnShape& a) { return static_cast<size_t>(s.B) * c.H * s.blocks * KC_PAGE * a.score_rows * sizeof(float); }
static size_t cache_bytes(const kd_cache& c, int bits) { return static_cast<size_t>(c.pages) * c.H * KC_PAGE * 2 * (bits == 8 ? c.D : c.D / 2 + c.D / K4_GROUP); }
static size_t scores_limit(const kd_cache& c, int bits) { return std::max(KA_SCORES_LIMIT, cache_bytes(c, bits) / 8); }

static AttnShape shape_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, int bits) {
  AttnShape a;
  a.G = p.H / c.H;
  a.rows = a.G * p.T;
#ifdef KD_TEST_DROP_LOAD
  const char* drop = getenv("KD_TEST_DROP_LOAD");
  a.test_drop = drop != nullptr ? atoi(drop) : 0;
#endif
  const int rows = a.item_rows = rows_of_item(a.rows);
  a.tiles = (a.rows + rows - 1) / rows;
  a.stats = p.weights != nullptr;
  a.score_rows = !a.stats || a.rows > KA_TILE ? 0 : a.rows <= 2 ? 2 : a.rows <= 4 ? 4 : 8;
  if (scores_bytes(c, s, a) > scores_limit(c, bits)) a.score_rows = 0;
  const int64_t items = static_cast<int64_t>(s.B) * c.H * a.tiles, pages = items * s.blocks;
  // Up to eight pages a head, or with many heads for each SM, a CTA takes whole heads and nothing is joined; so it is where the flat order would need more than 32 bits. us with whole heads and with
  // pages shared, from 16 heads for each SM on: 300 x 2000 tokens of 8 heads of 128, 4 rows, 190 and 230; 128 x 4096 of 32 heads, a row each, 600 and 650; 1000 x 700 of 4 heads of 64 87 and 316; 5000 x 600 of one
  // head 95 and 1600 (every CTA goes through all lengths). Where one sequence is far longer than all others its heads are what a call waits for: 300 x 500 tokens of 8 heads with one of 10,000 122 and 127, with one of
  // 100,000 690 and 176. The lengths are on the device, and the table's width alone does not tell such a batch from one whose tables have room to grow.
  const int slots = 148 * (rows == KC_ROWS ? KC_CTAS : ctas_of(rows / KA_TILE));
  a.ctas = s.blocks <= 8 || items > 148 * 16 || pages >= (1 << 30) ? 0 : slots;
  a.even = a.ctas > 0 && items > slots / 2;   // see FlatOrder
  a.spread = a.even ? 1 : slots - static_cast<int>(items);
  a.least = rows == KC_ROWS ? 8 : 2;   // four tiles of 128 tokens; a unit for each warp
  return a;
}

static size_t workspace_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, char* base, AttnWorkspace* ws) {
  size_t n = 0;
  auto take = [&](size_t bytes) {
    char* at = base + n;
    n += (bytes + 255) & ~size_t(255);
    return at;
  };
  const size_t part_rows = (a.even ? size_t(2) : size_t(1)) * a.ctas * rows_of_item(a.rows);
  ws->scores = reinterpret_cast<float*>(take(scores_bytes(c, s, a)));
  ws->stats = reinterpret_cast<float2*>(take(a.stats ? static_cast<size_t>(s.B) * p.H * p.T * sizeof(float2) : 0));
  ws->part_o = reinterpret_cast<float*>(take(part_rows * c.D * sizeof(float)));
  ws->part_ml = reinterpret_cast<float2*>(take(part_rows * sizeof(float2)));
  return n;
}

size_t cache_attention_workspace(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, int bits) {
  AttnWorkspace ws;
  return workspace_of(c, s, p, shape_of(c, s, p, bits), nullptr, &ws);
}

int launch_cache_attention(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, int bits, cudaStream_t stream) {
  const AttnShape a = shape_of(c, s, p, bits);
  const int64_t heads = static_cast<int64_t>(s.B) * c.H;
  if (heads * a.rows > INT32_MAX || (a.stats && heads * s.blocks > INT32_MAX)) return set_error(KD_ERR_LIMIT, "%d sequences of %d blocks are too many for one call", s.B, s.blocks);
  AttnWorkspace ws;
  workspace_of(c, s, p, a, static_cast<char*>(p.workspace), &ws);
  cudaError_t e = cudaSuccess;
  if (a.item_rows == KC_ROWS) e = bits == 8 ? launch_attention_chunk8(c, s, p, a, ws, stream) : launch_attention_chunk4(c, s, p, a, ws, stream);
  else e = bits == 8 ? launch_attention_rows8(c, s, p, a, ws, stream) : launch_attention_rows4(c, s, p, a, ws, stream);
  if (a.score_rows > 0 && s.blocks > 0) {
    const int64_t groups = heads * ((static_cast<int64_t>(s.blocks) * KC_PAGE + KS_TOKENS - 1) / KS_TOKENS);
    static SharedFirst shared_first;
    if (e == cudaSuccess) e = shared_first(cache_join_weights_kernel);
    if (e == cudaSuccess) e = launch(cache_join_weights_kernel, static_cast<unsigned>(groups), KJ_WARPS * 32, 0, stream, c, s, p, a, ws);
    if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_attention launch: %s", cudaGetErrorString(e));
    return 0;
  }
  if (e == cudaSuccess && a.ctas > 0) {
    // (1024 CTAs for as many rows of two or three parts were two waves)
    const bool few = heads * a.rows <= 148 * 2, many = a.item_rows >= 4 * KJ_WARPS && heads * a.rows >= 148 * 2 * 4 * KJ_WARPS;
    static SharedFirst first_few, first_some, first_many;
    e = few ? first_few(cache_join_kernel<KJ_WARPS, 1>) : many ? first_many(cache_join_kernel<1, 4>) : first_some(cache_join_kernel<1, 1>);
    if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_join_kernel attribute: %s", cudaGetErrorString(e));
    auto ctas = [&](int rows) { return static_cast<unsigned>(heads * ((a.rows + rows - 1) / rows)); };
    e = few    ? launch(cache_join_kernel<KJ_WARPS, 1>, ctas(1), KJ_WARPS * 32, 0, stream, c, s, p, a, ws)
        : many ? launch(cache_join_kernel<1, 4>, ctas(4 * KJ_WARPS), KJ_WARPS * 32, 0, stream, c, s, p, a, ws)
               : launch(cache_join_kernel<1, 1>, ctas(KJ_WARPS), KJ_WARPS * 32, 0, stream, c, s, p, a, ws);
  }
  if (e == cudaSuccess) e = bits == 8 ? launch_attention_weights8(c, s, p, a, ws, stream) : launch_attention_weights4(c, s, p, a, ws, stream);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_attention launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace kd
