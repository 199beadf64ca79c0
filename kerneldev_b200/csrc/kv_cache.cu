// The 8-bit key/value cache without its attention: appending, reading, eviction (whose search serves the 4-bit cache as well). See kd_attention.h for the format.
// All are bound by memory traffic, for a handful of tokens by launches.
#include <algorithm>

#include "kv_cache.cuh"

namespace kd {

// max over the block's threads; scratch: a word for each warp
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* scratch) {
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = m;
  __syncthreads();
  m = scratch[threadIdx.x & (KC_THREADS / 32 - 1)];
  return __reduce_max_sync(0xffffffffu, m);
}

// One block of one head of a sequence, K or V: reads the tokens that are new in it once, keeps them in registers as they came while the CTA
// agrees on the scale, and writes them as bytes. (Kept as floats they took twice the registers, and half as many CTAs had loads on their way.)
template <int kType>
__global__ void __launch_bounds__(KC_THREADS, kType == KD_F32 ? 4 : 6)
cache_append_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_tokens t, int W) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t scratch[KC_THREADS / 32];
  const bool is_v = (blockIdx.x & 1u) != 0u;
  uint32_t item = blockIdx.x >> 1;
  const int h = static_cast<int>(item % static_cast<uint32_t>(c.H));
  item /= static_cast<uint32_t>(c.H);
  const int w = static_cast<int>(item % static_cast<uint32_t>(W)), b = static_cast<int>(item / static_cast<uint32_t>(W));
  // A length or a number of tokens that cannot be says nothing of where to write: nothing is. (Clamped, as for reading, a negative length would open the first page anew.) What the
  // table has no more pages for is left out.
  const int len = s.lens[b], room = s.blocks * KC_PAGE;
  int n = t.n_new != nullptr ? t.n_new[b] : t.T;
  const bool valid = len >= 0 && len <= room && n >= 0 && n <= t.T;
  if (!valid || n > room - len) {
    if (threadIdx.x == 0) cache_report(c, KC_BAD_LENGTH);
    if (!valid) return;
    n = room - len;
  }
  const int block = len / KC_PAGE + w, base = block * KC_PAGE;
  if (base >= len + n || n == 0) return;
  const int raw_page = s.table[b * s.table_stride + block];
  const int lo = max(len - base, 0), hi = min(len + n - base, KC_PAGE);   // slots lo .. hi - 1 are new
  const int per_row = c.D / 16, chunks = KC_PAGE * per_row;
  const kd_tensor& x = is_v ? t.v : t.k;
  constexpr int kSize = kType == KD_F32 ? 4 : 2;
  const char* rows = static_cast<const char*>(x.ptr) + (b * x.stride_b + h * x.stride_h) * kSize;

  Raw16<kType> raw[KC_CHUNKS];
  uint32_t amax = 0;
  bool special = false;
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row, col = chunk - slot * per_row;
    if (slot >= lo && slot < hi) raw[i].load(rows + (static_cast<int64_t>(base + slot - len) * x.stride_t + col * 16) * kSize);
  }
  const int page = checked_page(c, raw_page);
  if (page < 0) return;
  const size_t at = block_index(c, page, h);
  uint8_t* bytes = static_cast<uint8_t*>(is_v ? c.v : c.k) + at * KC_PAGE * c.D;
  float* scale = (is_v ? c.v_scale : c.k_scale) + at;
  const int old = lo > 0 ? scale_exponent(*scale) : KC_EXP_MIN;
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int slot = (i * KC_THREADS + threadIdx.x) / per_row;
    if (slot >= lo && slot < hi) amax = max(amax, raw[i].amax(special));
  }
  const int e = max(exponent_for(block_max(amax, scratch)), old);
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row;
    if (chunk >= chunks) break;
    uint4* to = reinterpret_cast<uint4*>(bytes) + chunk;
    if (slot >= lo && slot < hi) {
      float f[16];
      raw[i].floats(f);
      *to = special ? quantise16<true>(f, e) : quantise16<false>(f, e);
    } else if (slot < lo) {
      if (e != old) {   // what is there already, on the coarser grid
        float g[16];
        dequantise16(*to, old - e, g);
        *to = quantise16<true>(g, 0);
      }
    } else if (lo == 0) {
      *to = make_uint4(0u, 0u, 0u, 0u);   // a page that is opened holds nothing of its earlier use
    }
  }
  // (everyone has read the old scale: block_max ends behind a barrier)
  if (threadIdx.x == 0) *scale = exp2i(e);
  if (!is_v && c.desc != nullptr && threadIdx.x < KC_PAGE && static_cast<int>(threadIdx.x) >= lo && static_cast<int>(threadIdx.x) < hi) {
    const int64_t i = base + static_cast<int>(threadIdx.x) - len;
    const bool ins = t.in_span != nullptr && t.in_span[b * t.in_span_stride_b + i] != 0;
    const bool pre = t.is_prefix != nullptr && t.is_prefix[b * t.is_prefix_stride_b + i] != 0;
    const int64_t sid = t.span_id != nullptr ? t.span_id[b * t.span_id_stride_b + i] : 0;
    if (span_id_out_of_range(sid)) cache_report(c, KD_STATUS_SPAN_RANGE);
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

// KR_TOKENS tokens of one head, K and V: the loads of both are on their way together
constexpr int KR_TOKENS = 64;
template <int kType>
__global__ void __launch_bounds__(KC_THREADS)
cache_read_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const int32_t* __restrict__ start, int count, int groups,
                  const __grid_constant__ kd_tensor k, const __grid_constant__ kd_tensor v) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t item = blockIdx.x / static_cast<uint32_t>(groups);
  const int r0 = static_cast<int>(blockIdx.x - item * groups) * KR_TOKENS;
  const int b = static_cast<int>(item / static_cast<uint32_t>(c.H)), h = static_cast<int>(item - static_cast<uint32_t>(b) * c.H);
  const int len = sequence_length(c, s, b), per_row = c.D / 16;
  const int64_t from = start != nullptr ? start[b] : 0;
  uint4 x[2][KC_CHUNKS];
  float scale[2][KC_CHUNKS];
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row, col = chunk - slot * per_row;
    const int64_t j = from + r0 + slot;
    x[0][i] = x[1][i] = make_uint4(0u, 0u, 0u, 0u);
    scale[0][i] = scale[1][i] = 1.f;
    if (slot < KR_TOKENS && r0 + slot < count && j >= 0 && j < len) {
      const int page = page_of(c, s, b, static_cast<int>(j / KC_PAGE));
      if (page >= 0) {
        const size_t at = block_index(c, page, h), byte = (at * KC_PAGE + j % KC_PAGE) * c.D + col * 16;
        x[0][i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(c.k) + byte);
        x[1][i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(c.v) + byte);
        scale[0][i] = c.k_scale[at];
        scale[1][i] = c.v_scale[at];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / per_row, col = chunk - slot * per_row;
    if (slot >= KR_TOKENS || r0 + slot >= count) break;
    constexpr int kSize = kType == KD_F32 ? 4 : 2;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const kd_tensor& out = y == 0 ? k : v;
      float f[16];
      dequantise16(x[y][i], scale_exponent(scale[y][i]), f);
      store16<kType>(static_cast<char*>(out.ptr) + (b * out.stride_b + h * out.stride_h + static_cast<int64_t>(r0 + slot) * out.stride_t + col * 16) * kSize, f);
    }
  }
}

int launch_cache_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k,
                      const kd_tensor& v, cudaStream_t stream) {
  const int groups = (count + KR_TOKENS - 1) / KR_TOKENS;
  const int64_t grid = static_cast<int64_t>(s.B) * c.H * groups;
  if (grid > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences of %d tokens and %d heads are too many for one call", s.B, count, c.H);
  auto* kernel = dtype == KD_F16 ? cache_read_kernel<KD_F16> : dtype == KD_BF16 ? cache_read_kernel<KD_BF16> : cache_read_kernel<KD_F32>;
  const cudaError_t e = launch(kernel, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, start, count, groups, k, v);
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

// Which tokens one head of one sequence keeps: a cluster of CTAs, each with a run of the tokens, each thread with a run of its CTA's. The first
// KE_KEYS keys of a thread stay in registers, further ones (beyond what a cluster of eight holds, 131,072 tokens) are read again.
// The smallest key that is kept comes from a radix search, 8 bits at a time from the top: a histogram of the candidates' next digit, and the digit in which
// the count from above passes what is wanted. Weights of one magnitude share their first digit, and a warp's additions to one bin queue up: equal digits of a
// warp are counted first and added once. Counts do not depend on any order. Then two sums over the threads before hand out the places.
constexpr int KE_KEYS = 16, KE_MAX_THREADS = 1024, KE_MAX_CLUSTER = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
// the address of a word of shared memory in another CTA of the cluster, and a load from there
__device__ __forceinline__ uint32_t cluster_address(uint32_t smem, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t cluster_load(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

__global__ void __launch_bounds__(KE_MAX_THREADS)
cache_select_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_eviction e, int cluster) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t hist[2][256], merged[256], s_digit, s_above, totals[2][KE_MAX_CLUSTER], warp_sum[2][KE_MAX_THREADS / 32];
  const int item = blockIdx.x / cluster, b = item / c.H, h = item - b * c.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const uint32_t rank = cluster > 1 ? cluster_rank() : 0u;
  auto sync = [&]() {
    if (cluster > 1) cluster_sync();
    else __syncthreads();
  };
  const int n = sequence_length(c, s, b), m = min(n, e.keep);
  const float* w = e.weights + b * e.w_stride_b + h * e.w_stride_h;
  int32_t* index = e.index + static_cast<size_t>(item) * e.keep;
  float* kept_w = e.out_weights + static_cast<size_t>(item) * e.keep;
  if (h == 0 && rank == 0 && tid == 0) e.out_lens[b] = m;
  const bool all = n <= e.keep;
  const int lo = e.first, hi = n - e.recent;   // free to go: lo .. hi - 1
  const int threads = cluster * blockDim.x, per = max((n + threads - 1) / threads, 1), begin = static_cast<int>(rank * blockDim.x + tid) * per;
  auto weight = [&](int j) { return j < e.w_len ? w[j] : 0.f; };
  auto is_free = [&](int j) { return j >= lo && j < hi; };
  const uint32_t wanted = all ? 0u : static_cast<uint32_t>(e.keep - e.first - e.recent);   // of the free ones

  uint32_t key[KE_KEYS];   // 0: not a free token (no free one has that: it would be a NaN with a sign, and those count as largest)
#pragma unroll
  for (int i = 0; i < KE_KEYS; ++i) {
    const int j = begin + i;
    key[i] = i < per && is_free(j) ? weight_key(weight(j)) : 0u;
  }
  uint32_t least = 0, rest = wanted;   // rest: how many of those that share the digits found so far
  if (wanted > 0) {
    if (tid < 256) hist[0][tid] = 0u;
    __syncthreads();
    uint32_t known = 0;
#pragma unroll 1
    for (int step = 0; step < 4; ++step) {
      const int shift = 24 - 8 * step;
      uint32_t* mine = hist[step & 1];
      auto count = [&](uint32_t k) {   // whole warps
        const bool in = k != 0u && (k & known) == least;
        if (!__any_sync(0xffffffffu, in)) return;
        const uint32_t digit = in ? (k >> shift) & 255u : 256u, same = __match_any_sync(0xffffffffu, digit);
        if (in && lane == __ffs(same) - 1) atomicAdd(&mine[digit], __popc(same));
      };
#pragma unroll
      for (int i = 0; i < KE_KEYS; ++i) count(key[i]);
      for (int i = KE_KEYS; i < per; ++i) {
        const int j = begin + i;
        count(is_free(j) ? weight_key(weight(j)) : 0u);
      }
      sync();
      if (tid < 256) {
        uint32_t n_all = mine[tid];
        for (int r = 0; r < cluster; ++r)
          if (static_cast<uint32_t>(r) != rank) n_all += cluster_load(cluster_address(smem_u32(&mine[tid]), r));
        merged[tid] = n_all;
        hist[(step + 1) & 1][tid] = 0u;   // the others have read it before this step's barrier
      }
      __syncthreads();
      if (warp == 0) {   // lane l: digits 255 - 8 l .. 248 - 8 l
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += merged[255 - 8 * lane - i];
        uint32_t above = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, above, o);
          if (lane >= o) above += up;
        }
        above -= sum;
        if (above < rest && above + sum >= rest) {
          for (int i = 0; i < 8; ++i) {
            const uint32_t n_here = merged[255 - 8 * lane - i];
            if (above + n_here >= rest) {
              s_digit = 255 - 8 * lane - i;
              s_above = above;
              break;
            }
            above += n_here;
          }
        }
      }
      __syncthreads();
      least |= s_digit << shift;
      known |= 255u << shift;
      rest -= s_above;
    }
  }
  // `least` is the smallest key that is kept; of those equal to it the first ones, so many that there are `wanted` in all
  auto kind_of = [&](int j, uint32_t k) -> int {   // 0: goes, 1: stays, 2: equal to the least
    if (all || !is_free(j)) return 1;
    return wanted == 0u ? 0 : k > least ? 1 : k == least ? 2 : 0;
  };
  auto kind_again = [&](int j) -> int { return j < n ? kind_of(j, weight_key(weight(j))) : 0; };   // of the tokens that are not held
  uint32_t stays = 0, ties = 0;
  uint32_t kinds = 0u;   // two bits for each held token
#pragma unroll
  for (int i = 0; i < KE_KEYS; ++i) {
    const int k = i < per && begin + i < n ? kind_of(begin + i, key[i]) : 0;
    kinds |= static_cast<uint32_t>(k) << (2 * i);
    stays += k == 1 ? 1u : 0u;
    ties += k == 2 ? 1u : 0u;
  }
  for (int i = KE_KEYS; i < per; ++i) {
    const int k = kind_again(begin + i);
    stays += k == 1 ? 1u : 0u;
    ties += k == 2 ? 1u : 0u;
  }
  // sums over the threads before this one, in this CTA and the ones before
  uint32_t before[2] = {stays, ties};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t mine = before[x];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, before[x], o);
      if (lane >= o) before[x] += up;
    }
    if (lane == 31) warp_sum[x][warp] = before[x];
    before[x] -= mine;
  }
  __syncthreads();
  uint32_t total[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t v = lane < warps ? warp_sum[x][lane] : 0u;
    total[x] = __reduce_add_sync(0xffffffffu, v);
    before[x] += __reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
  }
  uint32_t all_stay = total[0];
  if (cluster > 1) {
    if (wanted == 0u) cluster_sync();   // all have begun (the search has had its barriers)
    if (tid < cluster)
#pragma unroll
      for (int x = 0; x < 2; ++x) {   // into every CTA's table
        const uint32_t at = cluster_address(smem_u32(&totals[x][rank]), tid);
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(total[x]) : "memory");
      }
    cluster_sync();
    all_stay = 0;
    for (uint32_t r = 0; r < static_cast<uint32_t>(cluster); ++r) {
      all_stay += totals[0][r];
      if (r < rank) {
        before[0] += totals[0][r];
        before[1] += totals[1][r];
      }
    }
  }
  const uint32_t take = static_cast<uint32_t>(m) - min(all_stay, static_cast<uint32_t>(m));   // ties that stay
  // a token's place: those that stay before it and the ties among them
  uint32_t place = before[0] + min(before[1], take), tie = before[1];
  auto put = [&](int k, int j) {
    if (k == 0) return;
    if (k == 2 && tie++ >= take) return;
    if (place < static_cast<uint32_t>(e.keep)) {
      index[place] = j;
      kept_w[place] = weight(j);
    }
    ++place;
  };
#pragma unroll
  for (int i = 0; i < KE_KEYS; ++i) put((kinds >> (2 * i)) & 3u, begin + i);
  for (int i = KE_KEYS; i < per; ++i) put(kind_again(begin + i), begin + i);
  for (int r = m + static_cast<int>(rank * blockDim.x) + tid; r < e.keep; r += threads) {
    index[r] = -1;
    kept_w[r] = 0.f;
  }
}

// One block of what a head keeps, K and V: where its tokens are and their scales first, then their bytes, and a scale of the block's own. A token whose scale the new one
// equals keeps its bytes.
__global__ void __launch_bounds__(KC_THREADS)
cache_gather_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_eviction e, int W) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t scratch[2][KC_THREADS / 32];
  __shared__ size_t s_row[KC_PAGE];
  __shared__ int s_exp[2][KC_PAGE];
  const uint32_t item = blockIdx.x / static_cast<uint32_t>(W);
  const int w = static_cast<int>(blockIdx.x - item * W), b = static_cast<int>(item / static_cast<uint32_t>(c.H)), h = static_cast<int>(item - static_cast<uint32_t>(b) * c.H);
  const int n = sequence_length(c, s, b), m = min(n, e.keep), base = w * KC_PAGE;
  if (base >= m) return;
  const int page = checked_page(c, e.out_table[b * e.out_table_stride + w]);
  if (page < 0) return;
  const size_t to = block_index(c, page, h);
  if (threadIdx.x < KC_PAGE) {
    const int slot = threadIdx.x;
    size_t row = SIZE_MAX;   // there is no such token
    int ek = 0, ev = 0;
    if (base + slot < m) {
      const int j = e.index[static_cast<size_t>(item) * e.keep + base + slot], source = page_of(c, s, b, j / KC_PAGE);
      if (source >= 0) {
        const size_t at = block_index(c, source, h);
        row = at * KC_PAGE + j % KC_PAGE;
        ek = scale_exponent(c.k_scale[at]);
        ev = scale_exponent(c.v_scale[at]);
      }
      if (c.desc != nullptr) c.desc[to * KC_PAGE + slot] = source >= 0 ? c.desc[row] : 0u;
    }
    s_row[slot] = row;
    s_exp[0][slot] = ek;
    s_exp[1][slot] = ev;
  }
  __syncthreads();
  const int per_row = c.D / 16, chunks = KC_PAGE * per_row;
  uint4 x[2][KC_CHUNKS];
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x, slot = min(chunk / per_row, KC_PAGE - 1), col = chunk % per_row;
    const size_t row = chunk < chunks ? s_row[slot] : SIZE_MAX;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      x[y][i] = make_uint4(0u, 0u, 0u, 0u);
      if (row != SIZE_MAX) x[y][i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(y == 0 ? c.k : c.v) + row * c.D + col * 16);
    }
  }
  uint32_t amax[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int slot = min((i * KC_THREADS + static_cast<int>(threadIdx.x)) / per_row, KC_PAGE - 1);
#pragma unroll
    for (int y = 0; y < 2; ++y) {   // magnitudes are ordered as their bytes are; 0x7F is NaN
      uint32_t top = 0;
      const uint32_t words[4] = {x[y][i].x, x[y][i].y, x[y][i].z, x[y][i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = words[j] & 0x7F7F7F7Fu;
        top = __vmaxu4(top, u & ~__vcmpeq4(u, 0x7F7F7F7Fu));
      }
      top = __vmaxu4(top, top >> 16);
      top = max(top & 0xFFu, (top >> 8) & 0xFFu);
      float f[4];
      e4m3x4_to_f32x4(top, f);
      amax[y] = max(amax[y], __float_as_uint(f[0] * exp2i(s_exp[y][slot])));
    }
  }
  int ex[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, amax[y]);
    if ((threadIdx.x & 31) == 0) scratch[y][threadIdx.x >> 5] = top;
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 2; ++y) ex[y] = exponent_for(__reduce_max_sync(0xffffffffu, scratch[y][threadIdx.x & (KC_THREADS / 32 - 1)]));
#pragma unroll
  for (int i = 0; i < KC_CHUNKS; ++i) {
    const int chunk = i * KC_THREADS + threadIdx.x;
    if (chunk >= chunks) break;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int shift = s_exp[y][chunk / per_row] - ex[y];
      uint4 out = x[y][i];
      if (shift != 0) {
        float f[16];
        dequantise16(x[y][i], shift, f);
        out = quantise16<true>(f, 0);
      }
      reinterpret_cast<uint4*>(static_cast<uint8_t*>(y == 0 ? c.k : c.v) + to * KC_PAGE * c.D)[chunk] = out;
    }
  }
  if (threadIdx.x < 2) (threadIdx.x == 0 ? c.k_scale : c.v_scale)[to] = exp2i(ex[threadIdx.x]);
}

// A kernel launched with clusters of CTAs beside the stream's other kernels (see launch).
template <typename... P, typename... A>
static cudaError_t launch_cluster(void (*kernel)(P...), unsigned cluster, dim3 grid, dim3 block, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

int launch_cache_evict(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, int bits, cudaStream_t stream) {
  const int W = (e.keep + KC_PAGE - 1) / KC_PAGE;
  const int64_t items = static_cast<int64_t>(s.B) * c.H, grid = items * W;
  // As many CTAs, and threads of them, as hold the longest sequence's keys in registers: 256 threads for up to 4096 tokens, whose barriers are
  // the cheapest, then up to eight such CTAs, then larger ones.
  const int64_t tokens = static_cast<int64_t>(s.blocks) * KC_PAGE;
  int threads = 256, cluster = 1;
  while (cluster < KE_MAX_CLUSTER && static_cast<int64_t>(threads) * cluster * KE_KEYS < tokens) cluster *= 2;
  while (threads < KE_MAX_THREADS && static_cast<int64_t>(threads) * cluster * KE_KEYS < tokens) threads *= 2;
  if (grid > INT32_MAX || items * cluster > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences that keep %d tokens of %d heads are too many for one call", s.B, e.keep, c.H);
  cudaError_t r = launch_cluster(cache_select_kernel, cluster, static_cast<unsigned>(items * cluster), threads, stream, c, s, e, cluster);
  if (r == cudaSuccess)
    r = bits == 8 ? launch(cache_gather_kernel, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, e, W) : launch_cache4_gather(c, s, e, static_cast<unsigned>(grid), W, stream);
  if (r != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_evict launch: %s", cudaGetErrorString(r));
  return 0;
}

}  // namespace kd
