// The 4-bit key/value cache without its attention: appending, reading, and moving what eviction keeps. See kd_attention.h for the format.
// For a handful of tokens bound by launches, else by memory and instructions: appending 8 x 4093 tokens of 8 heads of 128 (bf16) takes 28 us with 74 % of the issue slots busy (floor 20; 42 with
// divisions, emulated packed maxima and 64-bit places for each group), reading them back 30 (floor 25). A group of 16 numbers has a scale of its own, so a thread has a group, nothing is agreed on among
// threads, and what a page holds already is never touched.
#include <type_traits>

#include "kv_cache.cuh"

namespace kd {

constexpr int C4_CHUNKS = 2 * KC_CHUNKS;   // groups of K and V that a thread holds, at most

struct Group4 {
  uint2 v;
  uint32_t scale;
};
__device__ __forceinline__ float inverse_of(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The largest magnitude of 16 numbers as the bits of a float, which are those of an infinity or NaN where one of the numbers is.
template <int kType>
__device__ __forceinline__ uint32_t group_max(const Raw16<kType>& raw) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < Raw16<kType>::WORDS; ++i) {
    const uint32_t w[4] = {raw.v[i].x, raw.v[i].y, raw.v[i].z, raw.v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kType == KD_F32) top = max(top, w[j] & 0x7FFFFFFFu);
      else if constexpr (kType == KD_BF16) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w[j] & 0x7FFF7FFFu));
      else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(w[j] & 0x7FFF7FFFu));
    }
  }
  if constexpr (kType == KD_F32) return top;
  const float2 two = unpack2<kType == KD_BF16>(top);
  return max(__float_as_uint(two.x), __float_as_uint(two.y)) & 0x7FFFFFFFu;
}
// A group as it is stored. The scale is the nearest to a sixth of the largest magnitude, and the numbers the nearest to what they are in its units; ties go to even.
// Floats are divided; a quotient is never rounded onto the middle of two steps: a float next to a middle times 6 or times a scale of 4 bits is 2^-24 of it away, and a quotient's rounding moves it
// less. 16-bit numbers are multiplied with a rounded inverse, and the product brought to a coarser grid (2^-16 of itself; 2^-13 by the fused sum with 1536, of which one step is that much), which puts it on a middle
// exactly where the quotient is: numbers of 11 bits have no other quotient that near to one (tests/test_kv_cache4_rounding.py goes through all of them). That takes a third of the instructions of divisions.
template <int kType>
__device__ __forceinline__ Group4 quantise_group(const Raw16<kType>& raw) {
  const uint32_t top_bits = group_max(raw);
  if (top_bits >= 0x7F800000u) return Group4{make_uint2(0u, 0u), K4_NAN};
  const float top = __uint_as_float(top_bits);
  uint32_t u;
  if constexpr (kType == KD_F32) u = __float_as_uint(__fdiv_rn(top, 6.f));
  else u = (__float_as_uint(top * (1.f / 6.f)) + 0x40u) & ~0x7Fu;
  const float sixth = __uint_as_float(u);
  const uint32_t byte = sixth < 0x1p-14f ? static_cast<uint32_t>(__float2int_rn(sixth * 0x1p17f)) : min(K4_TOP, ((u + 0x7FFFFu + (u >> 20 & 1u)) >> 20) - 896u);
  const float scale = unpack2<false>(byte << 7).x, inverse = byte != 0u ? inverse_of(scale) : 0.f;
  float f[16];
  raw.floats(f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if constexpr (kType == KD_F32) f[i] = byte != 0u ? __fdiv_rn(f[i], scale) : 0.f;
    else f[i] = __fsub_rn(__fmaf_rn(f[i], inverse, 1536.f), 1536.f);
  }
  return Group4{make_uint2(f32x8_to_e2m1x8(f), f32x8_to_e2m1x8(f + 8)), byte};
}

// One block of one head of a sequence, K and V.
template <int kType, int D>
__global__ void __launch_bounds__(KC_THREADS)
cache4_append_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_tokens t, int W) {
  pdl_wait();
  pdl_launch_dependents();
  uint32_t item = blockIdx.x;
  const int h = static_cast<int>(item % static_cast<uint32_t>(c.H));
  item /= static_cast<uint32_t>(c.H);
  const int w = static_cast<int>(item % static_cast<uint32_t>(W)), b = static_cast<int>(item / static_cast<uint32_t>(W));
  // (as for the 8-bit cache: a length or a number of tokens that cannot be says nothing of where to write, and what the table has no more pages for is left out)
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
  constexpr int GROUPS = D / K4_GROUP, CHUNKS = KC_PAGE * GROUPS, EACH = (CHUNKS + KC_THREADS - 1) / KC_THREADS, kSize = kType == KD_F32 ? 4 : 2;
  Raw16<kType> raw[2][EACH];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const kd_tensor& x = y == 0 ? t.k : t.v;
    const char* rows = static_cast<const char*>(x.ptr) + (b * x.stride_b + h * x.stride_h + (base - len) * x.stride_t) * kSize;   // of the block's first slot
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / GROUPS, col = chunk % GROUPS;
      if (slot >= lo && slot < hi) raw[y][i].load(rows + (slot * x.stride_t + col * K4_GROUP) * kSize);
    }
  }
  const int page = checked_page(c, raw_page);
  if (page < 0) return;
  const size_t at = block_index(c, page, h);
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int chunk = i * KC_THREADS + threadIdx.x, slot = chunk / GROUPS;
      if (slot >= KC_PAGE || slot < lo || (slot >= hi && lo > 0)) continue;
      Group4 g{make_uint2(0u, 0u), 0u};   // a page that is opened holds nothing of its earlier use
      if (slot < hi) g = quantise_group(raw[y][i]);
      const size_t place = at * CHUNKS + chunk;
      reinterpret_cast<uint2*>(y == 0 ? c.k : c.v)[place] = g.v;
      reinterpret_cast<uint8_t*>(y == 0 ? c.k_scale : c.v_scale)[place] = static_cast<uint8_t>(g.scale);
    }
  if (c.desc != nullptr && static_cast<int>(threadIdx.x) >= lo && static_cast<int>(threadIdx.x) < hi) {
    const int64_t i = base + static_cast<int>(threadIdx.x) - len;
    const bool ins = t.in_span != nullptr && t.in_span[b * t.in_span_stride_b + i] != 0;
    const bool pre = t.is_prefix != nullptr && t.is_prefix[b * t.is_prefix_stride_b + i] != 0;
    const int64_t sid = t.span_id != nullptr ? t.span_id[b * t.span_id_stride_b + i] : 0;
    if (span_id_out_of_range(sid)) cache_report(c, KD_STATUS_SPAN_RANGE);
    c.desc[at * KC_PAGE + threadIdx.x] = pack_token(ins, pre, sid, true);
  }
}

// call: a generic lambda that takes the type and the head dim as types
template <typename F>
static cudaError_t by_type_and_dim(int dtype, int D, F call) {
  auto dims = [&](auto type) {
    switch (D) {
      case 16: return call(type, std::integral_constant<int, 16>{});
      case 32: return call(type, std::integral_constant<int, 32>{});
      case 48: return call(type, std::integral_constant<int, 48>{});
      case 64: return call(type, std::integral_constant<int, 64>{});
      case 80: return call(type, std::integral_constant<int, 80>{});
      case 96: return call(type, std::integral_constant<int, 96>{});
      case 112: return call(type, std::integral_constant<int, 112>{});
      default: return call(type, std::integral_constant<int, 128>{});
    }
  };
  return dtype == KD_F16 ? dims(std::integral_constant<int, KD_F16>{}) : dtype == KD_BF16 ? dims(std::integral_constant<int, KD_BF16>{}) : dims(std::integral_constant<int, KD_F32>{});
}

int launch_cache4_append(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_tokens& t, cudaStream_t stream) {
  const int W = (t.T + KC_PAGE - 2) / KC_PAGE + 1;   // blocks that T tokens can touch
  const int64_t grid = static_cast<int64_t>(s.B) * W * c.H;
  if (grid > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences of %d new tokens and %d heads are too many for one call", s.B, t.T, c.H);
  const cudaError_t e = by_type_and_dim(t.dtype, c.D, [&](auto type, auto dim) {
    return launch(cache4_append_kernel<decltype(type)::value, decltype(dim)::value>, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, t, W);
  });
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache4_append_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

// ---- reading ------------------------------------------------------------------------------------------------------

// 64 tokens of one head, K and V, which lie in two pages at most: the loads of all are on their way together. A thread makes 16 bytes at a time, so that stores take whole sectors.
template <int kType, int D>
__global__ void __launch_bounds__(KC_THREADS)
cache4_read_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const int32_t* __restrict__ start, int count, int groups,
                   const __grid_constant__ kd_tensor k, const __grid_constant__ kd_tensor v) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kSize = kType == KD_F32 ? 4 : 2, N = 16 / kSize, ROW = D / N, SLOTS = KC_THREADS / ROW, EACH = (KC_PAGE + SLOTS - 1) / SLOTS;   // N numbers of a thread, SLOTS tokens at a time
  const uint32_t item = blockIdx.x / static_cast<uint32_t>(groups);
  const int r0 = static_cast<int>(blockIdx.x - item * groups) * KC_PAGE;
  const int b = static_cast<int>(item / static_cast<uint32_t>(c.H)), h = static_cast<int>(item - static_cast<uint32_t>(b) * c.H);
  const int len = sequence_length(c, s, b), first = threadIdx.x / ROW, d = threadIdx.x % ROW * N, here = min(KC_PAGE, count - r0);
  if (first >= SLOTS) return;
  const int64_t from = (start != nullptr ? start[b] : 0) + static_cast<int64_t>(r0);
  const int64_t block = from >= 0 ? from / KC_PAGE : -((KC_PAGE - 1 - from) / KC_PAGE);   // of the first token
  const int in = static_cast<int>(from - block * KC_PAGE);                                // its place there
  // tokens live .. end - 1 exist
  const int live = static_cast<int>(max(int64_t(0), min(int64_t(KC_PAGE), -from))), end = static_cast<int>(max(int64_t(0), min(int64_t(here), len - from)));
  int64_t rows[2];   // of token 0, if it were in this page; negative: there is none
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int page = live < end && block + x >= 0 && (block + x) * KC_PAGE < len && (x == 0 || in > 0) ? page_of(c, s, b, static_cast<int>(block + x)) : -1;
    rows[x] = page >= 0 ? static_cast<int64_t>(block_index(c, page, h)) * KC_PAGE + in - x * KC_PAGE : INT64_MIN / 2;
  }
  uint32_t codes[2][EACH], scale[2][EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int slot = first + i * SLOTS;
    const int64_t row = rows[in + slot >= KC_PAGE ? 1 : 0] + slot;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      codes[y][i] = scale[y][i] = 0u;
      if (slot < live || slot >= end || row < 0) continue;
      const uint8_t* at = static_cast<const uint8_t*>(y == 0 ? c.k : c.v) + (row * (D / 2) + d / 2);
      codes[y][i] = N == 8 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
      scale[y][i] = scales4(y == 0 ? c.k_scale : c.v_scale)[row * (D / K4_GROUP) + d / K4_GROUP];
    }
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const kd_tensor& out = y == 0 ? k : v;
    char* to = static_cast<char*>(out.ptr) + (b * out.stride_b + h * out.stride_h + static_cast<int64_t>(r0 + first) * out.stride_t + d) * kSize;
    const int64_t step = SLOTS * out.stride_t * kSize;
#pragma unroll
    for (int i = 0; i < EACH; ++i, to += step) {
      if (first + i * SLOTS >= here) continue;
      const uint32_t s2 = both_halves(scale[y][i]);
      uint32_t w[4];
      if constexpr (N == 4) {
        const HalfPairs four = e2m1x4_to_f16x4<false>(codes[y][i], 0, s2);
        const float2 lo = unpack2<false>(four.lo), hi = unpack2<false>(four.hi);
        w[0] = __float_as_uint(lo.x);
        w[1] = __float_as_uint(lo.y);
        w[2] = __float_as_uint(hi.x);
        w[3] = __float_as_uint(hi.y);
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          w[m] = times(e2m1x2_to_f16x2<true>(codes[y][i], m), s2);
          if (kType == KD_BF16) {
            const float2 two = unpack2<false>(w[m]);
            w[m] = pack2<true>(two.x, two.y);
          }
        }
      }
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

int launch_cache4_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k, const kd_tensor& v, cudaStream_t stream) {
  const int groups = (count + KC_PAGE - 1) / KC_PAGE;
  const int64_t grid = static_cast<int64_t>(s.B) * c.H * groups;
  if (grid > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d sequences of %d tokens and %d heads are too many for one call", s.B, count, c.H);
  const cudaError_t e = by_type_and_dim(dtype, c.D, [&](auto type, auto dim) {
    return launch(cache4_read_kernel<decltype(type)::value, decltype(dim)::value>, static_cast<unsigned>(grid), KC_THREADS, 0, stream, c, s, start, count, groups, k, v);
  });
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache4_read_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

// ---- eviction -----------------------------------------------------------------------------------------------------

// One block of what a head keeps, K and V: the tokens' bytes as they are (see cache_select_kernel for which).
__global__ void __launch_bounds__(KC_THREADS)
cache4_gather_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_eviction e, int W) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ size_t s_row[KC_PAGE];
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
    if (base + slot < m) {
      const int j = e.index[static_cast<size_t>(item) * e.keep + base + slot], source = page_of(c, s, b, j / KC_PAGE);
      if (source >= 0) row = block_index(c, source, h) * KC_PAGE + j % KC_PAGE;
      if (c.desc != nullptr) c.desc[to * KC_PAGE + slot] = source >= 0 ? c.desc[row] : 0u;
    }
    s_row[slot] = row;
  }
  __syncthreads();
  const int per_row = c.D / K4_GROUP, chunks = KC_PAGE * per_row;
  Group4 g[C4_CHUNKS];
#pragma unroll
  for (int i = 0; i < C4_CHUNKS; ++i) {
    const int both = i * KC_THREADS + threadIdx.x, chunk = both >= chunks ? both - chunks : both, slot = chunk / per_row;
    g[i] = Group4{make_uint2(0u, 0u), 0u};
    const size_t row = both < 2 * chunks ? s_row[slot] : SIZE_MAX;
    if (row != SIZE_MAX) {
      const size_t place = row * per_row + (chunk - slot * per_row);
      g[i].v = reinterpret_cast<const uint2*>(both >= chunks ? c.v : c.k)[place];
      g[i].scale = scales4(both >= chunks ? c.v_scale : c.k_scale)[place];
    }
  }
#pragma unroll
  for (int i = 0; i < C4_CHUNKS; ++i) {
    const int both = i * KC_THREADS + threadIdx.x, chunk = both >= chunks ? both - chunks : both;
    if (both >= 2 * chunks) break;
    const size_t place = to * chunks + chunk;
    reinterpret_cast<uint2*>(both >= chunks ? c.v : c.k)[place] = g[i].v;
    reinterpret_cast<uint8_t*>(both >= chunks ? c.v_scale : c.k_scale)[place] = static_cast<uint8_t>(g[i].scale);
  }
}

cudaError_t launch_cache4_gather(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, unsigned grid, int W, cudaStream_t stream) {
  return launch(cache4_gather_kernel, grid, KC_THREADS, 0, stream, c, s, e, W);
}

}  // namespace kd
