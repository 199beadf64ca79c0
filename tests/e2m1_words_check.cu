// The conversions of 4-bit numbers (kerneldev_b200/csrc/kv_cache.cuh) for every byte of a word, in code that uses each set of a word's bytes, from words that are loaded as 8, 16 or 32 bits, from shared or global
// memory, masked or as they are; and the way back for numbers on, between and beyond the levels, in each place. Prints "bad=0" where all are right.
#include <cstdio>
#include <utility>

#include "../kerneldev_b200/csrc/kv_cache.cuh"

using namespace kd;

template <int N>
__device__ __forceinline__ uint32_t load(const uint8_t* p) {
  return N == 1 ? *p : N == 2 ? *reinterpret_cast<const uint16_t*>(p) : *reinterpret_cast<const uint32_t*>(p);
}

// Thread t of 256 has word t of the table, of which it converts the bytes of kSet.
template <bool kWhole, int N, int kSet, int kForm>
__global__ void unpack_kernel(const uint8_t* in, uint32_t one, uint32_t* out) {
  __shared__ __align__(16) uint8_t s[1024];
  for (int i = threadIdx.x; i < 1024; i += 256) s[i] = in[i];
  __syncthreads();
  uint32_t w = load<N>(((kForm & 1) != 0 ? s : in) + 4 * threadIdx.x);
  if ((kForm & 2) != 0) w &= 0x0F0F0F0Fu;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((kSet >> i & 1) != 0) {
      const uint32_t r = e2m1x2_to_f16x2<kWhole>(w, i);
      out[threadIdx.x * 4 + i] = (kForm & 4) != 0 ? times(r, one) : r;
    }
}

__global__ void pack_kernel(const float* in, uint32_t* out, int only) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = in[threadIdx.x * 8 + i];
  const uint32_t w = f32x8_to_e2m1x8(f);
  out[threadIdx.x] = only >= 0 ? w >> (8 * only) & 0xFFu : w;
}

static const float kLevels[8] = {0.f, 0.5f, 1.f, 1.5f, 2.f, 3.f, 4.f, 6.f};
static uint32_t half_of(uint32_t code) {   // as bits
  static const uint32_t bits[8] = {0x0000u, 0x3800u, 0x3C00u, 0x3E00u, 0x4000u, 0x4200u, 0x4400u, 0x4600u};
  return bits[code & 7u] | (code & 8u) << 12;
}

static long bad = 0;
static uint8_t table[1024];
static uint8_t* d_in;
static uint32_t *d_out, h_out[1024];

template <bool kWhole, int N, int kSet, int kForm>
static void unpack() {
  unpack_kernel<kWhole, N, kSet, kForm><<<1, 256>>>(d_in, 0x3C003C00u, d_out);
  if (cudaMemcpy(h_out, d_out, sizeof h_out, cudaMemcpyDeviceToHost) != cudaSuccess) ++bad;
  long here = 0;
  for (int t = 0; t < 256; ++t)
    for (int i = 0; i < 4; ++i) {
      const uint32_t byte = table[4 * t + i] & ((kForm & 2) != 0 ? 0x0Fu : 0xFFu);
      here += (kSet >> i & 1) != 0 && h_out[4 * t + i] != (half_of(byte & 15u) | half_of(byte >> 4) << 16);
    }
  if (here != 0) printf("whole %d, load of %d bytes, set %x, form %d: %ld wrong\n", kWhole, N, kSet, kForm, here);
  bad += here;
}
template <bool kWhole, int N, int kSet, int... kForms>
static void forms(std::integer_sequence<int, kForms...>) {
  (unpack<kWhole, N, kSet, kForms>(), ...);
}
template <bool kWhole, int N, int kFirst, int... kSets>
static void sets(std::integer_sequence<int, kSets...>) {
  (forms<kWhole, N, kFirst + kSets>(std::make_integer_sequence<int, 8>()), ...);
}

int main() {
  for (int i = 0; i < 1024; ++i) table[i] = static_cast<uint8_t>(i / 4 * (2 * (i & 3) + 1) + 77 * (i & 3));   // each byte of the words takes every value
  if (cudaMalloc(&d_in, 1024) != cudaSuccess || cudaMalloc(&d_out, 4096) != cudaSuccess || cudaMemcpy(d_in, table, 1024, cudaMemcpyHostToDevice) != cudaSuccess) return 1;
  sets<false, 1, 1>(std::make_integer_sequence<int, 1>());
  sets<false, 2, 1>(std::make_integer_sequence<int, 3>());
  sets<false, 4, 1>(std::make_integer_sequence<int, 15>());
  sets<true, 4, 15>(std::make_integer_sequence<int, 1>());

  // levels, the middles of two (to even), what is a little off them, and beyond the largest, in all eight places
  static float f[128 * 8];
  static uint32_t want[128];
  uint32_t seed = 1;
  for (int i = 0; i < 1024; ++i) {
    seed = seed * 1664525u + 1013904223u;
    const int a = static_cast<int>(seed >> 29), kind = static_cast<int>(seed >> 20 & 3u);
    const uint32_t sign = seed >> 28 & 1u;
    uint32_t code = static_cast<uint32_t>(a);
    float x = kLevels[a];
    if (a == 7 && kind == 3) x = 1e30f;
    if (a < 7 && kind != 0) {
      const float middle = (kLevels[a] + kLevels[a + 1]) * 0.5f;
      x = kind == 1 ? middle : kind == 2 ? middle * (1.f - 0x1p-22f) : middle * (1.f + 0x1p-22f);
      code = kind == 1 ? static_cast<uint32_t>(a + (a & 1)) : static_cast<uint32_t>(kind == 2 ? a : a + 1);
    }
    f[i] = sign != 0u ? -x : x;
    want[i / 8] |= (code | sign << 3) << (4 * (i % 8));
  }
  float* d_f;
  if (cudaMalloc(&d_f, sizeof f) != cudaSuccess || cudaMemcpy(d_f, f, sizeof f, cudaMemcpyHostToDevice) != cudaSuccess) return 1;
  for (int only = -1; only < 4; ++only) {
    pack_kernel<<<1, 128>>>(d_f, d_out, only);
    if (cudaMemcpy(h_out, d_out, 128 * 4, cudaMemcpyDeviceToHost) != cudaSuccess) ++bad;
    long here = 0;
    for (int t = 0; t < 128; ++t) here += h_out[t] != (only >= 0 ? want[t] >> (8 * only) & 0xFFu : want[t]);
    if (here != 0) printf("eight numbers to a word, byte %d: %ld wrong\n", only, here);
    bad += here;
  }
  printf("bad=%ld %s\n", bad, cudaGetErrorString(cudaGetLastError()));
  return bad != 0;
}
