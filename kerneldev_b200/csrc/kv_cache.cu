// The 8-bit key/value cache without its attention: appending, reading, eviction. See kd_attention.h for the format.
// All are bound by memory traffic, for a handful of tokens by launches.
#include <algorithm>

#include "kv_cache.cuh"

namespace kd {

constexpr int KC_THREADS = 256, KC_CHUNKS = KC_PAGE * 128 / 16 / KC_THREADS;   // 16-byte chunks of a block that a thread holds, at most

// max over the block's threads; scratch: a word for each warp
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* scratch) {
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = m;
  __syncthreads();
  m = scratch[threadIdx.x & (KC_THREADS / 32 - 1)];
  return __reduce_max_sync(0xffffffffu, m);
}

// One block of one head of a sequence, K or V: reads the tokens that are new in it once, keeps them in registers while the CTA
// agrees on the scale, and writes them as bytes.
template <int kType>
__global__ void __launch_bounds__(KC_THREADS)
cache_append_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_tokens t, int W) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t scratch[KC_THREADS / 32];
  const bool is_v = (blockIdx.x & 1u) != 0u;
  uint32_t item = blockIdx.x >> 1;
  const int h = static_cast<int>(item % static_cast<uint32_t>(c.H));
  item /= static_cast<uint32_t>(c.H);
  const int w = static_cast<int>(item % static_cast<uint32_t>(W)), b = static_cast<int>(item / static_cast<uint32_t>(W));
  const int len = sequence_length(c, s, b);
  int n = t.n_new != nullptr ? checked_count(c, t.n_new[b], t.T) : t.T;
  if (n > s.blocks * KC_PAGE - len) {
    if (threadIdx.x == 0) cache_report(c, KC_BAD_LENGTH);
    n = s.blocks * KC_PAGE - len;
  }
  const int block = len / KC_PAGE + w, base = block * KC_PAGE;
  if (base >= len + n || n == 0) return;
  const int page = page_of(c, s, b, block);
  if (page < 0) return;
  const int lo = max(len - base, 0), hi = min(len + n - base, KC_PAGE);   // slots lo .. hi - 1 are new
  const size_t at = block_index(c, page, h);
  const int per_row = c.D / 16, chunks = KC_PAGE * per_row;
  uint8_t* bytes = static_cast<uint8_t*>(is_v ? c.v : c.k) + at * KC_PAGE * c.D;
  float* scale = (is_v ? c.v_scale : c.k_scale) + at;
  const kd_tensor& x = is_v ? t.v : t.k;
  constexpr int kSize = kType == KD_F32 ? 4 : 2;
  const char* rows = static_cast<const char*>(x.ptr) + (b * x.stride_b + h * x.stride_h) * kSize;

  float f[KC_CHUNKS][16];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row, col = chunk - slot * per_row;
    if (slot >= lo && slot < hi) {
      load16<kType>(rows + (static_cast<int64_t>(base + slot - len) * x.stride_t + col * 16) * kSize, f[i]);
      amax = max(amax, amax16(f[i]));
    }
  }
  int e = exponent_for(block_max(amax, scratch));
  const int old = lo > 0 ? scale_exponent(*scale) : KC_EXP_MIN;
  e = max(e, old);
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row;
    if (chunk >= chunks) break;
    uint4* to = reinterpret_cast<uint4*>(bytes) + chunk;
    if (slot >= lo && slot < hi) {
      *to = quantise16(f[i], e);
    } else if (slot < lo) {
      if (e != old) {   // what is there already, on the coarser grid
        float g[16];
        dequantise16(*to, old - e, g);
        *to = quantise16(g, 0);
      }
    } else if (lo == 0) {
      *to = make_uint4(0u, 0u, 0u, 0u);   // a page that is opened holds nothing of its earlier use
    }
  }
  __syncthreads();   // everyone has read the old scale
  if (threadIdx.x == 0) *scale = exp2i(e);
  if (!is_v && c.desc != nullptr && threadIdx.x < KC_PAGE && static_cast<int>(threadIdx.x) >= lo && static_cast<int>(threadIdx.x) < hi) {
    const int64_t i = base + static_cast<int>(threadIdx.x) - len;
    const bool ins = t.in_span != nullptr && t.in_span[b * t.in_span_stride_b + i] != 0;
    const bool pre = t.is_prefix != nullptr && t.is_prefix[b * t.is_prefix_stride_b + i] != 0;
    const int64_t sid = t.span_id != nullptr ? t.span_id[b * t.span_id_stride_b + i] : 0;
    c.desc[at * KC_PAGE + threadIdx.x] = pack_token(ins, pre, sid, true);
  }
}

int launch_cache_append(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_tokens& t, cudaStream_t stream) {
  const int W = (t.T + KC_PAGE - 2) / KC_PAGE + 1;   // blocks that T tokens can touch
  const int64_t grid = static_cast<int64_t>(s.B) * W * c.H * 2;
  if (grid > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences of %d new tokens and %d heads are too many for one call", s.B, t.T, c.H);
  auto* kernel = t.dtype == KD_F16 ? cache_append_kernel<KD_F16> : t.dtype == KD_BF16 ? cache_append_kernel<KD_BF16> : cache_append_kernel<KD_F32>;
  const cudaError_t e = launch(kernel, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, t, W);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_append_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

// ---- reading ------------------------------------------------------------------------------------------------------

// 16 numbers a thread; blockIdx.y: K or V
template <int kType>
__global__ void __launch_bounds__(KC_THREADS)
cache_read_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const int32_t* __restrict__ start, int count,
                  const __grid_constant__ kd_tensor k, const __grid_constant__ kd_tensor v) {
  pdl_wait();
  pdl_launch_dependents();
  const kd_tensor& out = blockIdx.y == 0 ? k : v;
  const uint8_t* bytes = static_cast<const uint8_t*>(blockIdx.y == 0 ? c.k : c.v);
  const float* scale = blockIdx.y == 0 ? c.k_scale : c.v_scale;
  const int per_row = c.D / 16;
  const int64_t total = static_cast<int64_t>(s.B) * c.H * count * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * KC_THREADS + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * KC_THREADS) {
    const int64_t row = i / per_row, bh = row / count;
    const int col = static_cast<int>(i - row * per_row), r = static_cast<int>(row - bh * count);
    const int b = static_cast<int>(bh / c.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * c.H);
    const int len = sequence_length(c, s, b);
    const int64_t j = static_cast<int64_t>(start != nullptr ? start[b] : 0) + r;
    float f[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) f[x] = 0.f;
    if (j >= 0 && j < len) {
      const int page = page_of(c, s, b, static_cast<int>(j / KC_PAGE));
      if (page >= 0) {
        const size_t at = block_index(c, page, h);
        dequantise16(*reinterpret_cast<const uint4*>(bytes + (at * KC_PAGE + j % KC_PAGE) * c.D + col * 16), scale_exponent(scale[at]), f);
      }
    }
    constexpr int kSize = kType == KD_F32 ? 4 : 2;
    store16<kType>(static_cast<char*>(out.ptr) + (b * out.stride_b + h * out.stride_h + r * out.stride_t + col * 16) * kSize, f);
  }
}

int launch_cache_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k,
                      const kd_tensor& v, cudaStream_t stream) {
  const int64_t total = static_cast<int64_t>(s.B) * c.H * count * (c.D / 16);
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((total + KC_THREADS - 1) / KC_THREADS, 148 * 64));
  auto* kernel = dtype == KD_F16 ? cache_read_kernel<KD_F16> : dtype == KD_BF16 ? cache_read_kernel<KD_BF16> : cache_read_kernel<KD_F32>;
  const cudaError_t e = launch(kernel, dim3(blocks, 2), KC_THREADS, 0, stream, c, s, start, count, k, v);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_read_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

// ---- eviction -----------------------------------------------------------------------------------------------------

// Weights in an order of unsigned numbers: NaN above everything, both zeros equal.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  if ((u << 1) == 0u) return 0x80000000u;
  return (u >> 31) != 0u ? ~u : u | 0x80000000u;
}

constexpr int KE_THREADS = 1024, KE_WARPS = KE_THREADS / 32;

// Which tokens one head of one sequence keeps. The smallest key that is kept comes from a radix search, 8 bits at a time from the top:
// a histogram of the candidates' next digit, and the digit in which the count from above passes what is wanted.
// Then one walk in order hands out the places.
__global__ void __launch_bounds__(KE_THREADS)
cache_select_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_eviction e) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t hist[256], s_digit, s_above, warp_keep[KE_WARPS], warp_tie[KE_WARPS];
  const int b = blockIdx.x / c.H, h = blockIdx.x - b * c.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = sequence_length(c, s, b), m = min(n, e.keep);
  const float* w = e.weights + b * e.w_stride_b + h * e.w_stride_h;
  int32_t* index = e.index + static_cast<size_t>(blockIdx.x) * e.keep;
  float* kept_w = e.out_weights + static_cast<size_t>(blockIdx.x) * e.keep;
  if (h == 0 && tid == 0) e.out_lens[b] = m;
  const bool all = n <= e.keep;
  const int lo = e.first, hi = n - e.recent;   // free to go: lo .. hi - 1
  auto weight = [&](int j) { return j < e.w_len ? w[j] : 0.f; };
  uint32_t wanted = all ? 0u : static_cast<uint32_t>(e.keep - e.first - e.recent), prefix = 0, known = 0;   // of the free ones
  if (wanted > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += KE_THREADS) {
        const uint32_t key = weight_key(weight(j));
        if ((key & known) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {   // lane l: digits 255 - 8 l .. 248 - 8 l
        uint32_t sum = 0;
        for (int i = 0; i < 8; ++i) sum += hist[255 - 8 * lane - i];
        uint32_t above = sum;
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, above, o);
          if (lane >= o) above += up;
        }
        above -= sum;
        if (above < wanted && above + sum >= wanted) {
          for (int i = 0; i < 8; ++i) {
            const uint32_t count = hist[255 - 8 * lane - i];
            if (above + count >= wanted) {
              s_digit = 255 - 8 * lane - i;
              s_above = above;
              break;
            }
            above += count;
          }
        }
      }
      __syncthreads();
      prefix |= s_digit << shift;
      known |= 255u << shift;
      wanted -= s_above;   // of those that share the digits so far
      __syncthreads();
    }
  }
  // prefix is the smallest key that is kept, `wanted` how many of those equal to it
  const bool none = !all && e.keep == e.first + e.recent;
  uint32_t placed = 0, ties = 0;
  for (int base = 0; base < n; base += KE_THREADS) {
    const int j = base + tid;
    const bool is_free = !all && j >= lo && j < hi;
    const float x = j < n ? weight(j) : 0.f;
    const uint32_t key = weight_key(x);
    const bool tie = is_free && !none && key == prefix;
    const uint32_t tie_bits = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) warp_tie[warp] = __popc(tie_bits);
    __syncthreads();
    const uint32_t other_ties = warp_tie[lane];
    const uint32_t tie_rank = ties + __reduce_add_sync(0xffffffffu, lane < warp ? other_ties : 0u) + __popc(tie_bits & ((1u << lane) - 1u));
    ties += __reduce_add_sync(0xffffffffu, other_ties);
    const bool keep = j < n && (!is_free || (!none && (key > prefix || (tie && tie_rank < wanted))));
    const uint32_t keep_bits = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_keep[warp] = __popc(keep_bits);
    __syncthreads();
    const uint32_t others = warp_keep[lane];
    const uint32_t rank = placed + __reduce_add_sync(0xffffffffu, lane < warp ? others : 0u) + __popc(keep_bits & ((1u << lane) - 1u));
    placed += __reduce_add_sync(0xffffffffu, others);
    if (keep && rank < static_cast<uint32_t>(e.keep)) {
      index[rank] = j;
      kept_w[rank] = x;
    }
    __syncthreads();
  }
  for (int r = m + tid; r < e.keep; r += KE_THREADS) {
    index[r] = -1;
    kept_w[r] = 0.f;
  }
}

// One block of what a head keeps, K or V: the bytes of its tokens from wherever they are, and a scale of its own.
__global__ void __launch_bounds__(KC_THREADS)
cache_gather_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_eviction e, int W) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t scratch[KC_THREADS / 32];
  const bool is_v = (blockIdx.x & 1u) != 0u;
  uint32_t item = blockIdx.x >> 1;
  const int w = static_cast<int>(item % static_cast<uint32_t>(W));
  item /= static_cast<uint32_t>(W);
  const int h = static_cast<int>(item % static_cast<uint32_t>(c.H)), b = static_cast<int>(item / static_cast<uint32_t>(c.H));
  const int n = sequence_length(c, s, b), m = min(n, e.keep), base = w * KC_PAGE;
  if (base >= m) return;
  const int page = checked_page(c, e.out_table[b * e.out_table_stride + w]);
  if (page < 0) return;
  const int32_t* index = e.index + static_cast<size_t>(item) * e.keep + base;
  const uint8_t* from = static_cast<const uint8_t*>(is_v ? c.v : c.k);
  const float* scale = is_v ? c.v_scale : c.k_scale;
  const int per_row = c.D / 16, chunks = KC_PAGE * per_row;
  float f[KC_CHUNKS][16];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row, col = chunk - slot * per_row;
#pragma unroll
    for (int x = 0; x < 16; ++x) f[i][x] = 0.f;
    if (chunk >= chunks || base + slot >= m) continue;
    const int j = index[slot], source = page_of(c, s, b, j / KC_PAGE);
    const size_t at = block_index(c, max(source, 0), h);
    if (source >= 0) dequantise16(*reinterpret_cast<const uint4*>(from + (at * KC_PAGE + j % KC_PAGE) * c.D + col * 16), scale_exponent(scale[at]), f[i]);
    amax = max(amax, amax16(f[i]));
    if (!is_v && col == 0 && c.desc != nullptr)
      c.desc[block_index(c, page, h) * KC_PAGE + slot] = source >= 0 ? c.desc[at * KC_PAGE + j % KC_PAGE] : 0u;
  }
  const int ex = exponent_for(block_max(amax, scratch));
  const size_t to = block_index(c, page, h);
  uint4* bytes = reinterpret_cast<uint4*>(static_cast<uint8_t*>(is_v ? c.v : c.k) + to * KC_PAGE * c.D);
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x;
    if (chunk < chunks) bytes[chunk] = quantise16(f[i], ex);
  }
  if (threadIdx.x == 0) (is_v ? c.v_scale : c.k_scale)[to] = exp2i(ex);
}

int launch_cache_evict(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, cudaStream_t stream) {
  const int W = (e.keep + KC_PAGE - 1) / KC_PAGE;
  const int64_t grid = static_cast<int64_t>(s.B) * c.H * W * 2;
  if (grid > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences that keep %d tokens of %d heads are too many for one call", s.B, e.keep, c.H);
  cudaError_t r = launch(cache_select_kernel, static_cast<unsigned>(s.B * c.H), KE_THREADS, 0, stream, c, s, e);
  if (r == cudaSuccess) r = launch(cache_gather_kernel, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, e, W);
  if (r != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_evict launch: %s", cudaGetErrorString(r));
  return 0;
}

}  // namespace kd
