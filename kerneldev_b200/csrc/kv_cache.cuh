// What the kernels of the key/value caches in 8 and 4 bits share: addresses of pages, conversions between e4m3 and wider types, scales.
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

// ---- numbers of 4 bits: e2m1, with a scale for each 16 of a row ---------------------------------------------------
// A scale is bits 14 .. 7 of a half (5 bits of exponent, 3 of mantissa, no sign), K4_TOP at most, so that 6 of them are a half; K4_NAN stands for 16 NaN. A number times its
// scale has 6 significant bits and no more than a half's exponents: exact as a half and as bfloat16.
constexpr int K4_GROUP = 16;
constexpr uint32_t K4_TOP = 226u, K4_NAN = 255u;   // 10240; what is written

// (a cache in 4 bits has the same structure, whose scales are bytes)
__device__ __forceinline__ const uint8_t* scales4(const float* p) { return reinterpret_cast<const uint8_t*>(p); }
__device__ __forceinline__ uint32_t both_halves(uint32_t scale) { return scale * 0x00800080u; }
// the halves of two scales that stand for NaN, or for nothing that is ever written (they may lie behind the last token), as ones
__device__ __forceinline__ uint32_t nan_scales(uint32_t two) { return __vcmpgtu2(two, K4_TOP * 0x00800080u); }
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Byte i of a word: two numbers as halves, the one in the low bits first. kWhole: the caller converts all four bytes of the word. Of a word that is unpacked into four bytes at once the compiler (CUDA 12.9) converts zeros where
// only one half of it is used, and of one that is unpacked by halves in place of the third byte; the third and fourth byte by a shift ahead of the halves are right, and all four at once are
// (tests/e2m1_words_check.cu goes through sets of bytes and ways to load them). The shift everywhere would cost 128 x 8192 tokens of 8 heads of 128 220 us in place of 183.
template <bool kWhole>
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t w, int i) {
  uint32_t r;
  if constexpr (kWhole) {
    if (i == 0) asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, a;\n}\n" : "=r"(r) : "r"(w));
    else if (i == 1) asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(r) : "r"(w));
    else if (i == 2) asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, c;\n}\n" : "=r"(r) : "r"(w));
    else asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, d;\n}\n" : "=r"(r) : "r"(w));
  } else {
    if (i >= 2) w >>= 16;
    if (i % 2 == 0) asm("{\n.reg .b16 l, h;\n.reg .b8 a, b;\nmov.b32 {l, h}, %1;\nmov.b16 {a, b}, l;\ncvt.rn.f16x2.e2m1x2 %0, a;\n}\n" : "=r"(r) : "r"(w));
    else asm("{\n.reg .b16 l, h;\n.reg .b8 a, b;\nmov.b32 {l, h}, %1;\nmov.b16 {a, b}, l;\ncvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(r) : "r"(w));
  }
  return r;
}
// eight numbers, nearest, ties to even, 6 at most, as a word
__device__ __forceinline__ uint32_t f32x8_to_e2m1x8(const float* f) {
  uint32_t r;
  asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\nmov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}
// half `half` of a word: four numbers times their scale (twice in a word)
template <bool kWhole>
__device__ __forceinline__ HalfPairs e2m1x4_to_f16x4(uint32_t w, int half, uint32_t scale) {
  return HalfPairs{times(e2m1x2_to_f16x2<kWhole>(w, 2 * half), scale), times(e2m1x2_to_f16x2<kWhole>(w, 2 * half + 1), scale)};
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
// 16 numbers of a row as they came: two 16-byte words of a 16-bit type, four of float
template <int kType>
struct Raw16 {
  static constexpr int WORDS = kType == KD_F32 ? 4 : 2;
  uint4 v[WORDS];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v[i] = __ldg(static_cast<const uint4*>(p) + i);
  }
  // The largest finite magnitude as the bits of a float, and whether there is a number that is not finite. 16-bit types two at a time: magnitudes
  // are ordered as their bits are.
  __device__ __forceinline__ uint32_t amax(bool& special) const {
    uint32_t top = 0, out = 0;
    constexpr uint32_t kInf = kType == KD_F32 ? 0x7F800000u : kType == KD_BF16 ? 0x7F807F80u : 0x7C007C00u;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kType == KD_F32) {
          const uint32_t u = w[j] & 0x7FFFFFFFu;
          out |= u >= kInf ? 1u : 0u;
          top = max(top, u >= kInf ? 0u : u);
        } else {
          const uint32_t u = w[j] & 0x7FFF7FFFu, beyond = __vcmpgeu2(u, kInf);
          out |= beyond;
          top = __vmaxu2(top, u & ~beyond);
        }
      }
    }
    special = special || out != 0u;
    if constexpr (kType == KD_F32) return top;
    const uint32_t one = max(top & 0xFFFFu, top >> 16);
    return kType == KD_BF16 ? one << 16 : __float_as_uint(unpack2<false>(one).x);
  }
  __device__ __forceinline__ void floats(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kType == KD_F32) {
          f[4 * i + j] = __uint_as_float(w[j]);
        } else {
          const float2 x = unpack2<kType == KD_BF16>(w[j]);
          f[8 * i + 2 * j] = x.x;
          f[8 * i + 2 * j + 1] = x.y;
        }
      }
    }
  }
};

constexpr int KC_THREADS = 256, KC_CHUNKS = KC_PAGE * 128 / 16 / KC_THREADS;   // chunks of 16 numbers of a block that a thread holds, at most

int launch_cache_append(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_tokens& t, cudaStream_t stream);
int launch_cache_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k,
                      const kd_tensor& v, cudaStream_t stream);
// bits: 8, or 4 with c standing for a kd_cache4
size_t cache_attention_workspace(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& q, int bits);
int launch_cache_attention(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& q, int bits, cudaStream_t stream);
int launch_cache_evict(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, int bits, cudaStream_t stream);
// kv_cache4.cu
cudaError_t launch_cache4_gather(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_eviction& e, unsigned grid, int W, cudaStream_t stream);
int launch_cache4_append(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_tokens& t, cudaStream_t stream);
int launch_cache4_read(const kd_cache& c, const kd_cache_seqs& s, const int32_t* start, int count, int dtype, const kd_tensor& k, const kd_tensor& v, cudaStream_t stream);

}  // namespace kd
