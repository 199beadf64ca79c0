// What the kernels of the 8-bit key/value cache share: addresses of pages, conversions between e4m3 and wider types, scales.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "mask_rule.cuh"
#include "sm100_prims.cuh"

namespace kd {

constexpr int KC_PAGE = KD_CACHE_PAGE;
constexpr int KC_EXP_MIN = -32, KC_EXP_MAX = 31;
constexpr uint32_t KC_BAD_LENGTH = KD_STATUS_CACHE_RANGE | 1u, KC_BAD_PAGE = KD_STATUS_CACHE_RANGE | 2u;

// (no part of the callers' code: they have it at every look-up)
static __device__ __noinline__ void cache_report_to(uint32_t* mirror, uint32_t code) {
  if (mirror != nullptr) {
    *const_cast<volatile uint32_t*>(mirror) = code;
    __threadfence_system();
  }
}
__device__ __forceinline__ void cache_report(const kd_cache& c, uint32_t code) { cache_report_to(c.status_mirror, code); }

// a count from device memory, clamped to 0 .. most
__device__ __forceinline__ int checked_count(const kd_cache& c, int n, int most) {
  if (n >= 0 && n <= most) return n;
  cache_report(c, KC_BAD_LENGTH);
  return n < 0 ? 0 : most;
}
// kAhead: ahead of the wait for the kernel before (see pdl_wait), past L1: the line may be there from before the length was written
template <bool kAhead = false>
__device__ __forceinline__ int length_word(const int32_t* p) { return kAhead ? __ldcg(p) : *p; }
template <bool kAhead = false>
__device__ __forceinline__ int sequence_length(const kd_cache& c, const kd_cache_seqs& s, int b) {
  return checked_count(c, length_word<kAhead>(s.lens + b), s.blocks * KC_PAGE);
}
// the page of a sequence's block, -1 where the table names none that exists
__device__ __forceinline__ int checked_page(const kd_cache& c, int page) {
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(c.pages)) return page;
  cache_report(c, KC_BAD_PAGE);
  return -1;
}
__device__ __forceinline__ int page_of(const kd_cache& c, const kd_cache_seqs& s, int b, int block) {
  return checked_page(c, s.table[b * s.table_stride + block]);
}
// index of (page, head) in the scales; times KC_PAGE * D the first byte of its block
__device__ __forceinline__ size_t block_index(const kd_cache& c, int page, int h) { return static_cast<size_t>(page) * c.H + h; }

// ---- numbers ----------------------------------------------------------------------------------------------------

// the exponent of a scale (a power of two)
__device__ __forceinline__ int scale_exponent(float s) { return static_cast<int>((__float_as_uint(s) >> 23) & 255u) - 127; }
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// The smallest e with amax <= 448 * 2^e, clamped; amax as the bits of a float that is finite and not negative.
// With amax = 1.f * 2^x: 448 = 1.75 * 2^8, so e = x - 8, or one more where 1.f is above 1.75.
__device__ __forceinline__ int exponent_for(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return amax == 0u ? KC_EXP_MIN : max(KC_EXP_MIN, min(KC_EXP_MAX, e));
}

// Four e4m3 numbers (low byte first) as halves, which hold every e4m3 number exactly: the low two and the high two. (The unpacking is
// left to the conversion, which can take either half of a register.)
struct HalfPairs {
  uint32_t lo, hi;
};
__device__ __forceinline__ HalfPairs e4m3x4_to_f16x4(uint32_t four) {
  HalfPairs r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(r.lo), "=r"(r.hi) : "r"(four));
  return r;
}
// two floats to e4m3, nearest even; beyond 448 saturates, NaN stays NaN. lo in the low byte
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  uint32_t r;
  asm("{\n.reg .b16 d;\ncvt.rn.satfinite.e4m3x2.f32 d, %2, %1;\ncvt.u32.u16 %0, d;\n}\n" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(const float* f) { return f32x2_to_e4m3x2(f[0], f[1]) | (f32x2_to_e4m3x2(f[2], f[3]) << 16); }
__device__ __forceinline__ void e4m3x4_to_f32x4(uint32_t w, float* f) {
  const HalfPairs h = e4m3x4_to_f16x4(w);
  const float2 a = unpack2<false>(h.lo), b = unpack2<false>(h.hi);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}

// 16 numbers of a row, 32 bytes of a 16-bit type, 64 of float
template <int kType>
__device__ __forceinline__ void store16(void* p, const float (&f)[16]) {
  if constexpr (kType == KD_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4 v;
      v.x = pack2<kType == KD_BF16>(f[8 * i], f[8 * i + 1]);
      v.y = pack2<kType == KD_BF16>(f[8 * i + 2], f[8 * i + 3]);
      v.z = pack2<kType == KD_BF16>(f[8 * i + 4], f[8 * i + 5]);
      v.w = pack2<kType == KD_BF16>(f[8 * i + 6], f[8 * i + 7]);
      reinterpret_cast<uint4*>(p)[i] = v;
    }
  }
}
// 16 bytes of e4m3 to floats, times 2^e
__device__ __forceinline__ void dequantise16(const uint4& v, int e, float (&f)[16]) {
  const float s = exp2i(e);
  e4m3x4_to_f32x4(v.x, f);
  e4m3x4_to_f32x4(v.y, f + 4);
  e4m3x4_to_f32x4(v.z, f + 8);
  e4m3x4_to_f32x4(v.w, f + 12);
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] *= s;
}
// floats to e4m3 in units of 2^e: one rounding, since the division by a power of two is exact (what it flushes is far below the smallest e4m3
// number). kSpecial: there may be an infinity, which becomes NaN, what e4m3 has in its place.
template <bool kSpecial>
__device__ __forceinline__ uint4 quantise16(const float (&f)[16], int e) {
  const float s = exp2i(-e);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = kSpecial && (__float_as_uint(f[i]) & 0x7F800000u) == 0x7F800000u ? __uint_as_float(0x7FC00000u) : f[i] * s;
  return make_uint4(f32x4_to_e4m3x4(x), f32x4_to_e4m3x4(x + 4), f32x4_to_e4m3x4(x + 8), f32x4_to_e4m3x4(x + 12));
}
int launch_cache_append(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_tokens& t, cudaStream_t stream);
int launch_cache_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k,
                      const kd_tensor& v, cudaStream_t stream);
int launch_cache_evict(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, cudaStream_t stream);
size_t cache_attention_workspace(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& q);
int launch_cache_attention(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& q, cudaStream_t stream);

}  // namespace kd
