// Norms of the queries and keys of each head and their rotation by position, in one pass, and the gradients of both.
//
// A row x of D numbers (one head of one token): y = w x r with r = 1 / sqrt(mean(x^2) + eps) where there is a weight, else x. Pair p of R / 2 turns by the angle
// position * step[p]: (a, b) -> (a cos - b sin, b cos + a sin). Backward, with g the gradient turned back: dx = g, or r (g w - x r^2 mean(g w x)), and
// dw = the sum of g x r over all rows. All in 32 bits, rounded once.
//
// Angles. A step is kept as a 64-bit fraction of a turn, so that position * step modulo 2^64 is the fraction of a turn that is left, exact to position / 2^64 turns
// whatever the position: its upper 32 bits are the angle. For 16-bit types sine and cosine are the hardware's (off by 2^-21, beside 2^-9 or 2^-12 of the output), for float sincospif's.
//
// Bound by memory: each number is read and written once. A row has a group of L lanes, 16 numbers to each: the pairs of a lane are its own, and a lane keeps its
// sines and cosines for all heads of its token.
#include <algorithm>

#include "common.cuh"
#include "sm100_prims.cuh"

namespace kd {

constexpr int RT_THREADS = 256, RT_GRAD_BLOCKS = 148 * 2;

// eight numbers of a row as they came
template <int kType>
struct Chunk8 {
  static constexpr int WORDS = kType == KD_F32 ? 2 : 1;
  uint4 v[WORDS];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kType == KD_F32) {
          f[4 * i + j] = __uint_as_float(w[j]);
        } else {
          const float2 x = unpack2<kType == KD_BF16>(w[j]);
          f[2 * j] = x.x;
          f[2 * j + 1] = x.y;
        }
      }
    }
  }
  static __device__ __forceinline__ void store(char* p, const float* f) {
    if constexpr (kType == KD_F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    } else {
      constexpr bool kBf16 = kType == KD_BF16;
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<kBf16>(f[0], f[1]), pack2<kBf16>(f[2], f[3]), pack2<kBf16>(f[4], f[5]), pack2<kBf16>(f[6], f[7]));
    }
  }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == KD_F32) return static_cast<const float*>(w)[i];
  const uint32_t u = static_cast<const uint16_t*>(w)[i];
  return dtype == KD_BF16 ? unpack2<true>(u).x : unpack2<false>(u).x;
}

// sine and cosine of a fraction of a turn, in 2^-32 turns
template <int kType>
__device__ __forceinline__ void turn(int32_t fraction, float& c, float& s) {
  if constexpr (kType == KD_F32) {
    // the nearest quarter first, in whole numbers: what is left is a float that is off by 2^-27
    const int32_t quarter = static_cast<int32_t>(static_cast<uint32_t>(fraction) + (1u << 29)) >> 30;   // -2 .. 1, modulo a turn
    const int32_t rest = static_cast<int32_t>(static_cast<uint32_t>(fraction) - (static_cast<uint32_t>(quarter) << 30));
    float x, y;
    sincospif(static_cast<float>(rest) * 0x1p-31f, &y, &x);
    c = (quarter & 1) != 0 ? -y : x;
    s = (quarter & 1) != 0 ? x : y;
    if ((quarter & 2) != 0) {
      c = -c;
      s = -s;
    }
  } else {
    const float angle = static_cast<float>(fraction) * (3.14159265358979f * 0x1p-31f);
    c = __cosf(angle);
    s = __sinf(angle);
  }
}

// 16 numbers of a lane; kBack: by the negative angles
template <bool kBack>
__device__ __forceinline__ void rotate16(float (&f)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = f[2 * i], b = f[2 * i + 1], y = kBack ? -s[i] : s[i];
      f[2 * i] = fmaf(a, c[i], -(b * y));
      f[2 * i + 1] = fmaf(b, c[i], a * y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = f[i], b = f[i + 8], y = kBack ? -s[i] : s[i];
      f[i] = fmaf(a, c[i], -(b * y));
      f[i + 8] = fmaf(b, c[i], a * y);
    }
  }
}

// sum over a row's lanes
template <int L>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// How the work is cut: blockIdx.y a run of heads of q (the first splits_q) or k, blockIdx.x tiles of 256 / L tokens.
struct RotateShape {
  int splits_q, heads, tiles;
  float* partial;   // backward with weights: (gridDim.y, gridDim.x, D) sums of a CTA
};

template <int kType, int L, bool kGrad>
__global__ void __launch_bounds__(RT_THREADS) rotate_kernel(const __grid_constant__ kd_rotation p, const __grid_constant__ RotateShape shape) {
  constexpr int GROUPS = RT_THREADS / L, kSize = kType == KD_F32 ? 4 : 2;
  constexpr int BATCH = (kGrad ? 2 : 4) / (kType == KD_F32 ? 2 : 1);   // heads that a lane has on their way
  pdl_wait();
  pdl_launch_dependents();
  const int u = threadIdx.x & (L - 1), group = threadIdx.x / L;
  const bool is_k = static_cast<int>(blockIdx.y) >= shape.splits_q, mine = u < p.D / 16, turns = 16 * u < p.R;
  const int split = blockIdx.y - (is_k ? shape.splits_q : 0), h0 = split * shape.heads, h1 = min(h0 + shape.heads, is_k ? p.Hk : p.Hq);
  const kd_tensor& x = is_k ? p.k : p.q;
  const kd_tensor& y = is_k ? p.k_out : p.q_out;
  const kd_tensor& dx = is_k ? p.dk : p.dq;
  const void* weight = is_k ? p.k_weight : p.q_weight;
  // the lane's two pieces of eight
  const int first = p.interleaved != 0 || !turns ? 16 * u : 8 * u, second = p.interleaved != 0 || !turns ? first + 8 : p.R / 2 + first;
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = mine && weight != nullptr ? weight_at(weight, p.w_dtype, (i < 8 ? first : second - 8) + i) : 1.f;
    dw[i] = 0.f;
  }
  const float inv_d = 1.f / static_cast<float>(p.D);
  const int tokens = p.B * p.T;
#pragma unroll 1
  for (int tile = blockIdx.x; tile < shape.tiles; tile += gridDim.x) {
    const int token = tile * GROUPS + group;
    const bool live = token < tokens && mine;
    const int b = min(token, tokens - 1) / p.T, t = min(token, tokens - 1) - b * p.T;
    float c[8], s[8];
    if (turns && mine) {
      int64_t at[3];
#pragma unroll
      for (int a = 0; a < 3; ++a) {
        at[a] = t;
        if (a < p.axes && p.positions != nullptr) {
          const int64_t i = a * p.pos_stride_a + b * p.pos_stride_b + t * p.pos_stride_t;
          at[a] = p.pos_is_64 != 0 ? static_cast<const int64_t*>(p.positions)[i] : static_cast<const int32_t*>(p.positions)[i];
        }
      }
      if (p.offsets != nullptr) at[0] += p.offsets[b];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = 8 * u + i;
        const int64_t n = p.positions == nullptr || pair < p.ends[0] ? at[0] : pair < p.ends[1] ? at[1] : at[2];
        turn<kType>(static_cast<int32_t>((static_cast<uint64_t>(n) * p.steps[pair]) >> 32), c[i], s[i]);
      }
    }
    const int64_t from = b * x.stride_b + t * x.stride_t, to_y = b * y.stride_b + t * y.stride_t, to_dx = kGrad ? b * dx.stride_b + t * dx.stride_t : 0;
#pragma unroll 1
    for (int h = h0; h < h1; h += BATCH) {
      Chunk8<kType> rx[BATCH][2], rg[kGrad ? BATCH : 1][2];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (!live || h + i >= h1) continue;
        if (!kGrad || weight != nullptr) {
          const char* row = static_cast<const char*>(x.ptr) + (from + (h + i) * x.stride_h) * kSize;
          rx[i][0].load(row + first * kSize);
          rx[i][1].load(row + second * kSize);
        }
        if constexpr (kGrad) {
          const char* row = static_cast<const char*>(y.ptr) + (to_y + (h + i) * y.stride_h) * kSize;
          rg[i][0].load(row + first * kSize);
          rg[i][1].load(row + second * kSize);
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const bool here = live && h + i < h1;
        float f[16];
        if constexpr (!kGrad) {
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = 0.f;
          if (here) {
            rx[i][0].floats(f);
            rx[i][1].floats(f + 8);
          }
          if (weight != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) sum = fmaf(f[j], f[j], sum);
            const float r = __frsqrt_rn(fmaf(row_sum<L>(sum), inv_d, p.eps));
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = f[j] * r * w[j];
          }
          if (turns) rotate16<false>(f, c, s, p.interleaved != 0);
          if (here) {
            char* row = static_cast<char*>(y.ptr) + (to_y + (h + i) * y.stride_h) * kSize;
            Chunk8<kType>::store(row + first * kSize, f);
            Chunk8<kType>::store(row + second * kSize, f + 8);
          }
        } else {
          float g[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = g[j] = 0.f;
          if (here) {
            rg[i][0].floats(g);
            rg[i][1].floats(g + 8);
          }
          if (turns) rotate16<true>(g, c, s, p.interleaved != 0);
          if (weight != nullptr) {
            if (here) {
              rx[i][0].floats(f);
              rx[i][1].floats(f + 8);
            }
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              sum = fmaf(f[j], f[j], sum);
              dot = fmaf(g[j] * w[j], f[j], dot);
            }
            const float r = __frsqrt_rn(fmaf(row_sum<L>(sum), inv_d, p.eps)), back = row_sum<L>(dot) * inv_d * r * r;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              dw[j] = fmaf(g[j], f[j] * r, dw[j]);
              g[j] = r * fmaf(-f[j], back, g[j] * w[j]);
            }
          }
          if (here) {
            char* row = static_cast<char*>(dx.ptr) + (to_dx + (h + i) * dx.stride_h) * kSize;
            Chunk8<kType>::store(row + first * kSize, g);
            Chunk8<kType>::store(row + second * kSize, g + 8);
          }
        }
      }
    }
  }
  if constexpr (kGrad) {
    if (weight == nullptr || shape.partial == nullptr) return;
    // the CTA's sums, in a fixed order: over the groups of a warp, then over the warps
    __shared__ float sums[RT_THREADS / 32][16 * L];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int o = L; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane < L && mine)
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[warp][(j < 8 ? first : second - 8) + j] = dw[j];
    __syncthreads();
    float* out = shape.partial + (static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x) * p.D;
    for (int d = threadIdx.x; d < p.D; d += RT_THREADS) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < RT_THREADS / 32; ++i) total += sums[i][d];
      out[d] = total;
    }
  }
}

// The weights' gradients from the sums of the CTAs: eight elements of one of them a CTA, in a fixed order.
constexpr int RW_COLS = 8, RW_ROWS = RT_THREADS / RW_COLS;
__global__ void __launch_bounds__(RT_THREADS) rotate_weight_kernel(const __grid_constant__ kd_rotation p, const float* partial, int rows_q, int rows_k) {
  __shared__ float sums[RW_ROWS][RW_COLS];
  const int groups = p.D / RW_COLS;
  const bool is_k = static_cast<int>(blockIdx.x) >= groups;
  const int d = (blockIdx.x - (is_k ? groups : 0)) * RW_COLS + threadIdx.x % RW_COLS, lane = threadIdx.x / RW_COLS;
  void* out = is_k ? p.dk_weight : p.dq_weight;
  pdl_wait();
  pdl_launch_dependents();
  if (out == nullptr) return;
  const int rows = is_k ? rows_k : rows_q;
  const float* from = partial + (is_k ? static_cast<size_t>(rows_q) * p.D : 0) + d;
  float total = 0.f;
#pragma unroll 4
  for (int r = lane; r < rows; r += RW_ROWS) total += from[static_cast<size_t>(r) * p.D];
  sums[lane][threadIdx.x % RW_COLS] = total;
  __syncthreads();
  if (lane != 0) return;
  total = 0.f;
#pragma unroll
  for (int r = 0; r < RW_ROWS; ++r) total += sums[r][threadIdx.x];
  if (p.w_dtype == KD_F32) static_cast<float*>(out)[d] = total;
  else static_cast<uint16_t*>(out)[d] = static_cast<uint16_t>(p.w_dtype == KD_BF16 ? pack2<true>(total, 0.f) : pack2<false>(total, 0.f));
}

struct RotateGrid {
  int lanes, blocks, splits_q, splits_k, heads, tiles;
};
// Heads are cut until there are CTAs for all SMs; a lane's sines and cosines are for all heads of a run.
static RotateGrid grid_of(const kd_rotation& p, bool grad) {
  RotateGrid g;
  const int units = p.D / 16;
  g.lanes = units > 4 ? 8 : units > 2 ? 4 : units;
  const int64_t tokens = static_cast<int64_t>(p.B) * p.T, groups = RT_THREADS / g.lanes;
  g.tiles = static_cast<int>((tokens + groups - 1) / groups);
  const int wanted = grad ? RT_GRAD_BLOCKS : 148 * 8, most = std::max(p.Hq, p.Hk);
  const int64_t cuts = std::max<int64_t>(1, (wanted + 2 * static_cast<int64_t>(g.tiles) - 1) / (2 * static_cast<int64_t>(g.tiles)));
  g.heads = static_cast<int>(std::max<int64_t>(1, most / std::min<int64_t>(cuts, most)));
  g.splits_q = (p.Hq + g.heads - 1) / g.heads;
  g.splits_k = (p.Hk + g.heads - 1) / g.heads;
  g.blocks = grad ? std::min(g.tiles, std::max(1, RT_GRAD_BLOCKS / (g.splits_q + g.splits_k))) : g.tiles;
  return g;
}

size_t rotate_grad_workspace(const kd_rotation& p) {
  if (p.dq_weight == nullptr && p.dk_weight == nullptr) return 0;
  const RotateGrid g = grid_of(p, true);
  return static_cast<size_t>(g.splits_q + g.splits_k) * g.blocks * p.D * sizeof(float);
}

template <int kType, bool kGrad>
static cudaError_t launch_lanes(const kd_rotation& p, const RotateGrid& g, const RotateShape& s, cudaStream_t stream) {
  const dim3 grid(g.blocks, g.splits_q + g.splits_k);
  switch (g.lanes) {
    case 1: return launch(rotate_kernel<kType, 1, kGrad>, grid, RT_THREADS, 0, stream, p, s);
    case 2: return launch(rotate_kernel<kType, 2, kGrad>, grid, RT_THREADS, 0, stream, p, s);
    case 4: return launch(rotate_kernel<kType, 4, kGrad>, grid, RT_THREADS, 0, stream, p, s);
    default: return launch(rotate_kernel<kType, 8, kGrad>, grid, RT_THREADS, 0, stream, p, s);
  }
}

template <bool kGrad>
static cudaError_t launch_type(const kd_rotation& p, const RotateGrid& g, const RotateShape& s, cudaStream_t stream) {
  switch (p.dtype) {
    case KD_F16: return launch_lanes<KD_F16, kGrad>(p, g, s, stream);
    case KD_BF16: return launch_lanes<KD_BF16, kGrad>(p, g, s, stream);
    default: return launch_lanes<KD_F32, kGrad>(p, g, s, stream);
  }
}

int launch_rotate(const kd_rotation& p, bool grad, cudaStream_t stream) {
  const RotateGrid g = grid_of(p, grad);
  const bool weights = grad && (p.dq_weight != nullptr || p.dk_weight != nullptr);
  if (g.splits_q + g.splits_k > 65535) return set_error(KD_ERR_LIMIT, "%d and %d heads are too many for one call", p.Hq, p.Hk);
  const RotateShape s{g.splits_q, g.heads, g.tiles, weights ? static_cast<float*>(p.workspace) : nullptr};
  cudaError_t e = grad ? launch_type<true>(p, g, s, stream) : launch_type<false>(p, g, s, stream);
  if (e == cudaSuccess && weights)
    e = launch(rotate_weight_kernel, 2 * (p.D / RW_COLS), RT_THREADS, 0, stream, p, static_cast<const float*>(p.workspace), g.splits_q * g.blocks, g.splits_k * g.blocks);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "rotate_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace kd
