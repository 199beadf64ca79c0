// Norms of the queries and keys of each head and their rotation by position, in one pass, and the gradients of both.
//
// A row x of D numbers (one head of one token): y = w x r with r = 1 / sqrt(mean(x^2) + eps) where there is a weight, else x. Pair p of R / 2 turns by the angle
// position * step[p]: (a, b) -> (a cos - b sin, b cos + a sin). Backward, with g the gradient turned back: dx = g, or r (g w - x r^2 mean(g w x)), and
// dw = the sum of g x r over all rows. All in 32 bits, rounded once.
//
// Angles. A step is kept as a 64-bit fraction of a turn, so that position * step modulo 2^64 is the fraction of a turn that is left, exact to position / 2^65 turns
// whatever the position: rounded to 32 bits it is the angle. For 16-bit types sine and cosine are the hardware's (off by 2^-21.4 and 2^-21.2 for what it is given, an angle that is off by 2^-21.7 as a float: 2^-20 together,
// beside 2^-9 or 2^-12 of the output), for float polynomials (2^-23.2).
//
// Bound by memory: each number is read and written once. A row has a group of D / 16 lanes, 16 numbers to each: the pairs of a lane are its own, and a lane keeps its
// sines and cosines for all heads of a run. Rows are asked for ahead by asynchronous copies into shared memory, so that what is in flight takes no registers: with loads into registers a backward of
// 16 x 4096 tokens of 32 heads of 64 (bf16) took 235 us, so 133 (805 MB, 6.0 TB/s; the forward 87 us, 6.1 TB/s, 106 before); instructions come next, of which addresses formed anew and zeros for rows that
// are not there cost 22 us. A lane's pieces lie a part of the row apart, so that a copy of all lanes takes whole
// sectors: with 32 bytes side by side to a lane, interleaved pairs of 16384 tokens of 40 heads of 128 took 79 us, so 57.
#include <algorithm>
#include <numeric>

#include "attn_common.cuh"
#include "common.cuh"
#include "sm100_prims.cuh"

namespace kd {

// CTAs of an SM (registers allow two of the backward's; three of the forward's were 3 to 8 % slower), and bytes that a thread has in its ring: rows in flight are what reaches the memory's rate. 128 bytes
// for the forward cost 16 x 4096 tokens of 32 heads of 64 nothing and 2 x 2945 of 16 of 80 (float) 14 %, 384 gained nothing.
constexpr int RT_THREADS = 256, RT_WARPS = RT_THREADS / 32, RT_CTAS = 2, RT_RING = 256;
// Lanes of a row, 16 numbers to each, and rows of a warp (whose last two or four lanes may be idle).
constexpr __host__ __device__ int lanes_of(int D) { return D / 16; }
constexpr __host__ __device__ int tokens_of(int D) { return RT_WARPS * (32 / lanes_of(D)); }

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == KD_F32) return static_cast<const float*>(w)[i];
  const uint32_t u = static_cast<const uint16_t*>(w)[i];
  return dtype == KD_BF16 ? unpack2<true>(u).x : unpack2<false>(u).x;
}

// sine and cosine of a fraction of a turn, in 2^-32 turns
template <int kType>
__device__ __forceinline__ void turn(int32_t fraction, float& c, float& s) {
  if constexpr (kType == KD_F32) {
    // The nearest quarter first, in whole numbers; of the rest, an angle t of pi / 4 at most, the Taylor polynomials of sine and cosine to t^9 and t^10 (the next terms are below 2^-29). sincospif took
    // three times the instructions, which with few heads to a token was half of the time.
    const int32_t quarter = static_cast<int32_t>(static_cast<uint32_t>(fraction) + (1u << 29)) >> 30;   // -2 .. 1, modulo a turn
    const int32_t rest = static_cast<int32_t>(static_cast<uint32_t>(fraction) - (static_cast<uint32_t>(quarter) << 30));
    const float a = static_cast<float>(rest) * (6.28318530717958648f * 0x1p-32f), q = a * a;
    const float x = fmaf(q, fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const float y = fmaf(a * q, fmaf(q, fmaf(q, fmaf(q, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), a);
    const float even = (quarter & 1) != 0 ? -y : x, odd = (quarter & 1) != 0 ? x : y;
    c = (quarter & 2) != 0 ? -even : even;
    s = (quarter & 2) != 0 ? -odd : odd;
  } else {
    const float angle = static_cast<float>(fraction) * (3.14159265358979f * 0x1p-31f);
    c = __cosf(angle);
    s = __sinf(angle);
  }
}

// 16 numbers of a lane, eight pairs; kBack: by the negative angles
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

// Sum over the L lanes of a row that begins at lane `base`; i: this lane's number in it. All lanes of the warp call it.
template <int L>
__device__ __forceinline__ float row_sum(float x, int base, int i) {
  if constexpr ((L & (L - 1)) == 0) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  } else {   // pairs first where L is even, then the sums in a ring
    constexpr int RING = L % 2 == 0 ? L / 2 : L;
    if (L % 2 == 0) x += __shfl_sync(0xffffffffu, x, base + (i + L / 2) % L);
    float sum = x;
#pragma unroll
    for (int o = 1; o < RING; ++o) sum += __shfl_sync(0xffffffffu, x, base + (i + o) % L);
    return sum;
  }
}

// How the work is cut: `heads` heads of q (the first runs_q runs) or k, and tiles of tokens, which `ctas` CTAs share.
struct RotateShape {
  int runs_q, heads, tiles, ctas;
  float* partial;   // backward with weights: (runs, ctas, D) sums of a CTA
};

// A lane's 16 numbers of one tensor's row, in pieces of 16 bytes: piece i of a row's lanes lies side by side, so that a load takes whole sectors. A run of elements (those that turn, or those that do
// not) is cut into as many parts as a lane has pieces; with that, both elements of a pair are the same lane's in either order of pairs.
template <int kType>
struct Lane16 {
  static constexpr int SIZE = kType == KD_F32 ? 4 : 2, PIECES = SIZE, EACH = 16 / SIZE;   // numbers of a piece
  int start, part;   // the first piece's first element; elements of a part
  __device__ __forceinline__ Lane16(int u, int R, int D) : start(16 * u < R ? EACH * u : R + EACH * (u - R / 16)), part((16 * u < R ? R : D - R) / PIECES) {}
  __device__ __forceinline__ int element(int j) const { return start + j / EACH * part + j % EACH; }   // of number j
  static __device__ __forceinline__ void floats(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kType == KD_F32) {
        f[j] = __uint_as_float(w[j]);
      } else {
        const float2 x = unpack2<kType == KD_BF16>(w[j]);
        f[2 * j] = x.x;
        f[2 * j + 1] = x.y;
      }
    }
  }
  // row: of the first piece
  __device__ __forceinline__ void store(char* row, const float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      uint4 v;
      if constexpr (kType == KD_F32) {
        v = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
      } else {
        constexpr bool kBf16 = kType == KD_BF16;
        v = make_uint4(pack2<kBf16>(f[8 * i], f[8 * i + 1]), pack2<kBf16>(f[8 * i + 2], f[8 * i + 3]), pack2<kBf16>(f[8 * i + 4], f[8 * i + 5]), pack2<kBf16>(f[8 * i + 6], f[8 * i + 7]));
      }
      *reinterpret_cast<uint4*>(row + i * part * SIZE) = v;
    }
  }
};

// The rows on their way: a ring of each thread's own, in shared memory. Nobody else reads its places, so that no barrier is needed; what is in flight costs no registers.
template <int kType, bool kGrad>
struct RotateRing {
  static constexpr int PIECES = Lane16<kType>::PIECES * (kGrad ? 2 : 1);   // of a row: x, then the gradient
  static constexpr int STAGES = RT_RING / (16 * PIECES), BYTES = STAGES * PIECES * 16 * RT_THREADS;
  static __device__ __forceinline__ uint32_t place(uint32_t ring, int stage, int piece) { return ring + ((stage * PIECES + piece) * RT_THREADS + threadIdx.x) * 16; }
};

template <int N>
__device__ __forceinline__ void await_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

template <int kType, int D, bool kGrad>
__global__ void __launch_bounds__(RT_THREADS, RT_CTAS) rotate_kernel(const __grid_constant__ kd_rotation p, const __grid_constant__ RotateShape shape) {
  using Row = Lane16<kType>;
  using Ring = RotateRing<kType, kGrad>;
  constexpr int L = lanes_of(D), ROWS = 32 / L, kSize = Row::SIZE;
  extern __shared__ __align__(16) char smem[];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t ring = smem_u32(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane / L, u = lane - group * L, base = group * L;
  const int run = blockIdx.x / shape.ctas, cta = blockIdx.x - run * shape.ctas;
  const bool is_k = run >= shape.runs_q, mine = group < ROWS, turns = 16 * u < p.R;
  const int h0 = (run - (is_k ? shape.runs_q : 0)) * shape.heads;
  const kd_tensor& x = is_k ? p.k : p.q;
  const kd_tensor& y = is_k ? p.k_out : p.q_out;
  const kd_tensor& dx = is_k ? p.dk : p.dq;
  const void* weight = is_k ? p.k_weight : p.q_weight;
  const bool reads_x = !kGrad || weight != nullptr;
  const Row mine16(u, p.R, D);
  const int tokens = p.B * p.T;
  struct Place {
    int b, t;
    bool live;
  };
  auto place_of = [&](int tile) {
    const int token = tile * tokens_of(D) + warp * ROWS + group, at = min(token, tokens - 1), b = at / p.T;
    return Place{b, at - b * p.T, token < tokens && mine};
  };
  // the lane's first piece in the first head of the run; further heads are a step apart
  auto row_of = [&](const kd_tensor& z, const Place& at) { return static_cast<char*>(z.ptr) + (at.b * z.stride_b + h0 * z.stride_h + at.t * z.stride_t + mine16.start) * kSize; };

  // the next row to ask for
  int ask_tile = cta, ask_h = 0, ask_stage = 0;   // ask_h: of the run
  bool ask_live;
  const char *ask_x, *ask_y = nullptr;
  auto open = [&]() {
    const Place at = place_of(ask_tile);
    ask_live = at.live;
    ask_x = row_of(x, at);
    if (kGrad) ask_y = row_of(y, at);
  };
  open();
  // (Pointers that move on from head to head in the backward; in the forward, where they were 3 to 4 % slower, products with the head.)
  auto ask = [&]() {
    if (ask_tile < shape.tiles) {
      const char* row = kGrad ? ask_x : ask_x + ask_h * x.stride_h * kSize;
      if (ask_live) {
        if (reads_x)
#pragma unroll
          for (int i = 0; i < Row::PIECES; ++i) cp_async16(Ring::place(ring, ask_stage, i), row + i * mine16.part * kSize);
        if constexpr (kGrad)
#pragma unroll
          for (int i = 0; i < Row::PIECES; ++i) cp_async16(Ring::place(ring, ask_stage, Row::PIECES + i), ask_y + i * mine16.part * kSize);
      }
      if (kGrad) {
        ask_x += x.stride_h * kSize;
        ask_y += y.stride_h * kSize;
      }
      if (++ask_h == shape.heads) {
        ask_h = 0;
        ask_tile += shape.ctas;
        open();
      }
    }
    ask_stage = ask_stage + 1 == Ring::STAGES ? 0 : ask_stage + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Ring::STAGES - 1; ++i) ask();

  float w[16], dw[kGrad ? 16 : 1];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = mine && weight != nullptr ? weight_at(weight, p.w_dtype, mine16.element(i)) : 1.f;
    if (kGrad) dw[i] = 0.f;
  }
  int stage = 0;
#pragma unroll 1
  for (int tile = cta; tile < shape.tiles; tile += shape.ctas) {
    const Place at = place_of(tile);
    float c[8], s[8];
    if (turns && mine) {
      int64_t n[3];
#pragma unroll
      for (int a = 0; a < 3; ++a) {
        n[a] = at.t;
        if (a < p.axes && p.positions != nullptr) {
          const int64_t i = a * p.pos_stride_a + at.b * p.pos_stride_b + at.t * p.pos_stride_t;
          n[a] = p.pos_is_64 != 0 ? static_cast<const int64_t*>(p.positions)[i] : static_cast<const int32_t*>(p.positions)[i];
        }
      }
      if (p.offsets != nullptr) n[0] += p.offsets[at.b];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = p.interleaved != 0 ? mine16.element(2 * i) / 2 : mine16.element(i);
        const int64_t here = p.positions == nullptr || pair < p.ends[0] ? n[0] : pair < p.ends[1] ? n[1] : n[2];
        turn<kType>(static_cast<int32_t>((static_cast<uint64_t>(here) * p.steps[pair] + (1ull << 31)) >> 32), c[i], s[i]);
      }
    }
    char* to = row_of(kGrad ? dx : y, at);
    const int64_t to_step = (kGrad ? dx : y).stride_h * kSize;
#pragma unroll 1
    for (int h = 0; h < shape.heads; ++h) {
      await_copies<Ring::STAGES - 2>();
      float f[16];
      auto take = [&](int from, float (&into)[16]) {   // (a row that is not there is whatever its place holds, and stays in its lanes)
#pragma unroll
        for (int i = 0; i < Row::PIECES; ++i) Row::floats(lds16(Ring::place(ring, stage, from + i)), into + i * Row::EACH);
      };
      if constexpr (!kGrad) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = 0.f;   // (without these, and loads for dead rows too, the forward is 5 % slower)
        if (at.live) take(0, f);
        if (weight != nullptr) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) sum = fmaf(f[j], f[j], sum);
          const float r = __frsqrt_rn(fmaf(row_sum<L>(sum, base, u), 1.f / D, p.eps));
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = f[j] * r * w[j];
        }
        if (turns) rotate16<false>(f, c, s, p.interleaved != 0);
        if (at.live) mine16.store(to + h * to_step, f);
      } else {
        float g[16];
        take(Row::PIECES, g);
        if (turns) rotate16<true>(g, c, s, p.interleaved != 0);
        if (weight != nullptr) {
          take(0, f);
          float sum = 0.f, dot = 0.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            sum = fmaf(f[j], f[j], sum);
            dot = fmaf(g[j] * w[j], f[j], dot);
          }
          const float r = __frsqrt_rn(fmaf(row_sum<L>(sum, base, u), 1.f / D, p.eps)), back = row_sum<L>(dot, base, u) * (1.f / D) * r * r;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (at.live) dw[j] = fmaf(g[j], f[j] * r, dw[j]);
            g[j] = r * fmaf(-f[j], back, g[j] * w[j]);
          }
        }
        if (at.live) mine16.store(to + h * to_step, g);
      }
      ask();   // (into the place of the row before: its numbers have been used)
      stage = stage + 1 == Ring::STAGES ? 0 : stage + 1;
    }
  }
  await_copies<0>();
  if constexpr (kGrad) {
    if (weight == nullptr || shape.partial == nullptr) return;
    // the CTA's sums, in a fixed order: over the rows of its warps
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    if (mine)
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(warp * ROWS + group) * D + mine16.element(j)] = dw[j];
    __syncthreads();
    if (threadIdx.x < D) {
      float total = 0.f;
#pragma unroll 8
      for (int i = 0; i < RT_WARPS * ROWS; ++i) total += sums[i * D + threadIdx.x];
      shape.partial[static_cast<size_t>(blockIdx.x) * D + threadIdx.x] = total;
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
  int runs_q, runs_k, heads, tiles, ctas;
};
// Runs of as many heads as q and k have equal ones of, so that all CTAs of one wave have the same; the run that has the least to do, by heads and by what the sines and cosines of a tile cost beside a head.
static RotateGrid grid_of(const kd_rotation& p) {
  const int64_t tokens = static_cast<int64_t>(p.B) * p.T, tile = tokens_of(p.D), tiles = (tokens + tile - 1) / tile, room = 148 * RT_CTAS;
  const int both = p.Hk > 0 ? std::gcd(p.Hq, p.Hk) : p.Hq;
  const float angles = p.dtype == KD_F32 ? 1.5f : 0.7f;
  RotateGrid best{};
  float least = 0.f;
  for (int heads = 1; heads <= std::min(both, 64); ++heads) {
    if (both % heads != 0) continue;
    const int64_t runs = (p.Hq + p.Hk) / heads, each = (tiles * runs + room - 1) / room;
    const float cost = static_cast<float>(each) * (static_cast<float>(heads) + angles);
    if (best.heads != 0 && cost > least) continue;
    least = cost;
    best = RotateGrid{p.Hq / heads, p.Hk / heads, heads, static_cast<int>(tiles), static_cast<int>((tiles + each - 1) / each)};
  }
  return best;
}

size_t rotate_grad_workspace(const kd_rotation& p) {
  if (p.dq_weight == nullptr && p.dk_weight == nullptr) return 0;
  const RotateGrid g = grid_of(p);
  return static_cast<size_t>(g.runs_q + g.runs_k) * g.ctas * p.D * sizeof(float);
}

template <int kType, int D, bool kGrad>
static cudaError_t launch_of(const kd_rotation& p, const RotateGrid& g, const RotateShape& s, cudaStream_t stream) {
  constexpr int kShared = RotateRing<kType, kGrad>::BYTES;
  static_assert(!kGrad || kShared >= tokens_of(D) * D * 4, "the weights' sums take the ring's place");
  static SmemOptIn opt_in;
  const cudaError_t e = opt_in(rotate_kernel<kType, D, kGrad>, kShared);
  return e != cudaSuccess ? e : launch(rotate_kernel<kType, D, kGrad>, static_cast<unsigned>((g.runs_q + g.runs_k) * g.ctas), RT_THREADS, kShared, stream, p, s);
}

template <int kType, bool kGrad>
static cudaError_t launch_dim(const kd_rotation& p, const RotateGrid& g, const RotateShape& s, cudaStream_t stream) {
  switch (p.D) {
    case 16: return launch_of<kType, 16, kGrad>(p, g, s, stream);
    case 32: return launch_of<kType, 32, kGrad>(p, g, s, stream);
    case 48: return launch_of<kType, 48, kGrad>(p, g, s, stream);
    case 64: return launch_of<kType, 64, kGrad>(p, g, s, stream);
    case 80: return launch_of<kType, 80, kGrad>(p, g, s, stream);
    case 96: return launch_of<kType, 96, kGrad>(p, g, s, stream);
    case 112: return launch_of<kType, 112, kGrad>(p, g, s, stream);
    default: return launch_of<kType, 128, kGrad>(p, g, s, stream);
  }
}

template <bool kGrad>
static cudaError_t launch_type(const kd_rotation& p, const RotateGrid& g, const RotateShape& s, cudaStream_t stream) {
  switch (p.dtype) {
    case KD_F16: return launch_dim<KD_F16, kGrad>(p, g, s, stream);
    case KD_BF16: return launch_dim<KD_BF16, kGrad>(p, g, s, stream);
    default: return launch_dim<KD_F32, kGrad>(p, g, s, stream);
  }
}

int launch_rotate(const kd_rotation& p, bool grad, cudaStream_t stream) {
  const RotateGrid g = grid_of(p);
  const bool weights = grad && (p.dq_weight != nullptr || p.dk_weight != nullptr);
  if (static_cast<int64_t>(g.runs_q + g.runs_k) * g.ctas > INT32_MAX) return set_error(KD_ERR_LIMIT, "%d and %d heads are too many for one call", p.Hq, p.Hk);
  const RotateShape s{g.runs_q, g.heads, g.tiles, g.ctas, weights ? static_cast<float*>(p.workspace) : nullptr};
  cudaError_t e = grad ? launch_type<true>(p, g, s, stream) : launch_type<false>(p, g, s, stream);
  if (e == cudaSuccess && weights)
    e = launch(rotate_weight_kernel, 2 * (p.D / RW_COLS), RT_THREADS, 0, stream, p, static_cast<const float*>(p.workspace), g.runs_q * g.ctas, g.runs_k * g.ctas);
  if (e != cudaSuccess) return set_error(KD_ERR_DEVICE, "rotate_kernel launch: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace kd
