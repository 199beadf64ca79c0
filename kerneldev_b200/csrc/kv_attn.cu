// Attention of the newest tokens over the 8-bit cache, and the weight that each cached token receives.
#include <algorithm>

#include "kv_cache.cuh"

namespace kd {

constexpr int KA_THREADS = 128;   // tokens of a step, one to a thread

// Places of a query row: its token's index, whether it exists, its descriptor.
struct QueryRow {
  int at;
  bool live;
  uint32_t desc;
};
__device__ __forceinline__ QueryRow query_row(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, int b, int h, int i, int len) {
  const int n = p.q_lens != nullptr ? checked_count(c, p.q_lens[b], p.T) : p.T;
  QueryRow r;
  r.at = len - n + i;
  r.live = i < n && r.at >= 0;
  r.desc = pack_plain(p.causal != 0);
  if (r.live && c.desc != nullptr) {
    const int page = page_of(c, s, b, r.at / KC_PAGE);
    r.desc = page >= 0 ? c.desc[block_index(c, page, h) * KC_PAGE + r.at % KC_PAGE] : 0u;
  }
  return r;
}

// the dot product of a cached key with a row of floats in shared memory
__device__ __forceinline__ float key_dot(const uint8_t* key, const float* q, int D) {
  float dot = 0.f;
  for (int d = 0; d < D; d += 16) {
    float f[16];
    dequantise16(*reinterpret_cast<const uint4*>(key + d), 0, f);
#pragma unroll
    for (int x = 0; x < 16; ++x) dot = fmaf(f[x], q[d + x], dot);
  }
  return dot;
}

// One query row: a thread's token gives a score, then a thread's column takes the values of all of them; running maximum and sum.
template <bool kBf16>
__global__ void __launch_bounds__(KA_THREADS)
cache_attention_rows_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ float sq[128], sp[KA_THREADS], sred[KA_THREADS / 32];
  __shared__ const uint8_t* sv[KA_THREADS];
  const int row = blockIdx.x, i = row % p.T, hq = row / p.T % p.H, b = row / p.T / p.H, h = hq / (p.H / c.H), tid = threadIdx.x;
  const int len = sequence_length(c, s, b);
  const QueryRow r = query_row(c, s, p, b, h, i, len);
  const uint16_t* q = static_cast<const uint16_t*>(p.q.ptr) + b * p.q.stride_b + hq * p.q.stride_h + i * p.q.stride_t;
  if (tid < c.D) {
    const uint32_t u = q[tid];
    sq[tid] = unpack2<kBf16>(u).x * (p.sm_scale * 1.4426950408889634f);
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int base = 0; r.live && base < len; base += KA_THREADS) {
    const int j = base + tid;
    float x = -INFINITY;
    const uint8_t* v = nullptr;
    float vs = 0.f;
    if (j < len) {
      const int page = page_of(c, s, b, j / KC_PAGE);
      if (page >= 0) {
        const size_t at = block_index(c, page, h);
        const uint32_t kd = c.desc != nullptr ? c.desc[at * KC_PAGE + j % KC_PAGE] : pack_plain(p.causal != 0);
        if (rule_allowed(r.desc, r.at, kd, j)) {
          const size_t byte = (at * KC_PAGE + j % KC_PAGE) * c.D;
          x = key_dot(static_cast<const uint8_t*>(c.k) + byte, sq, c.D) * c.k_scale[at];
          v = static_cast<const uint8_t*>(c.v) + byte;
          vs = c.v_scale[at];
        }
      }
    }
    float top = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) sred[tid >> 5] = top;
    __syncthreads();
    const float m2 = fmaxf(fmaxf(m, fmaxf(sred[0], sred[1])), fmaxf(sred[2], sred[3])), ref = m2 == -INFINITY ? 0.f : m2;
    const float pr = fast_exp2(x - ref), shrink = fast_exp2(m - ref);
    m = m2;
    sp[tid] = pr * vs;
    sv[tid] = v;
    float sum = pr;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if ((tid & 31) == 0) sred[tid >> 5] = sum;
    __syncthreads();
    l = l * shrink + (sred[0] + sred[1] + sred[2] + sred[3]);
    acc *= shrink;
    if (tid < c.D)
      for (int t = 0; t < KA_THREADS; ++t)
        if (sv[t] != nullptr) {
          const uint32_t byte = sv[t][tid];
          acc = fmaf(sp[t], unpack2<false>(e4m3x2_to_f16x2(byte)).x, acc);
        }
    __syncthreads();
  }
  if (tid < c.D) {
    uint16_t* o = static_cast<uint16_t*>(p.o.ptr) + b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t;
    o[tid] = static_cast<uint16_t>(pack2<kBf16>(l != 0.f ? acc / l : 0.f, 0.f));
  }
  if (tid == 0 && p.lse != nullptr) p.lse[row] = l != 0.f ? m + log2f(l) : -INFINITY;
}

// weights[j] += sum over the query rows of the head of softmax_j, from the rows' log-sum-exp; one thread to a token, so that nothing is added twice
// and the order is fixed
template <bool kBf16>
__global__ void __launch_bounds__(KC_PAGE)
cache_weights_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ float sq[128];
  const int block = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, G = p.H / c.H;
  const int len = sequence_length(c, s, b), j = block * KC_PAGE + tid;
  if (block * KC_PAGE >= len) return;
  const int page = page_of(c, s, b, block);
  if (page < 0) return;
  const size_t at = block_index(c, page, h);
  const uint8_t* key = static_cast<const uint8_t*>(c.k) + (at * KC_PAGE + tid) * c.D;
  const uint32_t kd = c.desc != nullptr ? c.desc[at * KC_PAGE + tid] : pack_plain(p.causal != 0);
  float sum = 0.f;
  for (int i = 0; i < p.T; ++i) {
    const QueryRow r = query_row(c, s, p, b, h, i, len);
    if (!r.live) continue;
    for (int g = 0; g < G; ++g) {
      const int hq = h * G + g;
      __syncthreads();
      const uint16_t* q = static_cast<const uint16_t*>(p.q.ptr) + b * p.q.stride_b + hq * p.q.stride_h + i * p.q.stride_t;
      for (int d = tid; d < c.D; d += KC_PAGE) {
        const uint32_t u = q[d];
        sq[d] = unpack2<kBf16>(u).x * (p.sm_scale * 1.4426950408889634f);
      }
      __syncthreads();
      const float lse = p.lse[(static_cast<size_t>(b) * p.H + hq) * p.T + i];
      if (j < len && rule_allowed(r.desc, r.at, kd, j)) sum += fast_exp2(key_dot(key, sq, c.D) * c.k_scale[at] - lse);
    }
  }
  if (j < len && j < p.w_len) p.weights[b * p.w_stride_b + h * p.w_stride_h + j] += sum;
}

size_t cache_attention_workspace(const kd_cache&, const kd_cache_seqs&, const kd_cache_queries&) { return 0; }

int launch_cache_attention(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, cudaStream_t stream) {
  const bool bf16 = p.dtype == KD_BF16;
  cudaError_t e = launch(bf16 ? cache_attention_rows_kernel<true> : cache_attention_rows_kernel<false>, static_cast<unsigned>(s.B * p.H * p.T), KA_THREADS, 0, stream, c, s, p);
  if (e == cudaSuccess && p.weights != nullptr && s.blocks > 0)
    e = launch(bf16 ? cache_weights_kernel<true> : cache_weights_kernel<false>, dim3(s.blocks, c.H, s.B), KC_PAGE, 0, stream, c, s, p);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "cache_attention launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace kd
