// Attention of the newest tokens over the cache, and the weight that each cached token receives: the kernels for few query rows, for both number formats (kBits).
//
// One key head at a time has few query rows (its group's heads times the new tokens), so what bounds these kernels is reading the cache: 2 D bytes
// a token. Every warp walks units of 32 tokens on its own, from asynchronous copies of its own, with no tile shared between warps and no barrier:
//   S^T = K Q^T    mma m16n8k16: the cache's tokens are the wide operand, 8 query rows the narrow one (with the rows in the wide one, half of it would be
//                  empty for most models). A lane's 16 bytes of a key row are its part of four steps: the order of the head dims inside a step is free as
//                  long as Q's registers have the same.
//   P = exp2(S)    each 8 x 8 block transposed between the lanes (movmatrix), as the operand of
//   O^T += V^T P^T A lane's 16 bytes of four tokens are its parts of all tiles of 16 head dims: the rows g and g + 8 of tile m are the bytes 2 m and 2 m + 1 of the
//                  eight lanes' pieces, so that loads stay 16 bytes wide.
// Both on halves: they hold every e4m3 number, and one instruction converts four. Rounded are P (2^-11, beside the output's 2^-8 or 2^-11) and the output; bfloat16
// queries become halves exactly, after a power of two for each row. (mma on e4m3 itself is made of conversions and products of halves on this
// chip: with it, and queries in three e4m3 terms, a unit took 740 instructions in place of 510.)
//
// Scales. A page's K scale multiplies its scores. Its V scale 2^ev goes into the exponent, p' = 2^(s + ev - ref + 8), and no product of its own is spent on it:
// O = sum p' v / sum p' 2^-ev. A half has 30 exponents for p', the scales of two pages may lie 63 apart, and what a page of small values brings must not
// get lost beside a page that has one large number: its other channels may be all zeros. So ref follows the maximum of s + ev, in steps of 6 or more; the offset of 8 keeps
// probabilities down to 2^-22 of the largest out of the half's subnormals, so that long tails keep their weight. And where a unit's scale is more than 2^4 below one that came before it, ref follows
// the unit's own maximum down (below_reference): its largest p' is 2^-4 at least. A half is off by 2^-25 at most below 2^-14: in
// probabilities that is 2^-28 of the row's largest, or 2^-20 of the unit's.
//
// Numbers of 4 bits have a scale for each 16 of a row: K = e2m1 times scale in one multiplication of two halves behind the conversion of two numbers, exact, V too; nothing of it is in the exponents, whose reference goes
// up only. A unit is 4.6 KB and 560 to 640 instructions, and what bounds it is that they wait for one another: at 32 x 4096 tokens of 8 heads of 128 an instruction is 5.0 cycles in its warp's hands (1.1 of them for a result
// at a fixed distance, 0.7 for the other warps, 0.5 for a pipe, 0.4 at barriers, 0.2 for memory), and 2.8 warps a scheduler cover 56 % of the issue slots. So each instruction counts, though slots are free: 128 x 8192 tokens
// take 183 us (907 MB, 5.0 TB/s), 164 without the multiplications, 158 without the conversions too, 220 with a shift for each word, and no less with the input in L2.
//
// NaN. A masked token has p' = 0, and 0 * NaN of a masked value would be NaN. A warp that ends with a NaN walks its units once more, with NaN values
// taken as zeros and, beside the product, one of indicators (row sees token, value is NaN) that puts NaN where it belongs. So does one that has met scores beyond KA_FAR.
#pragma once
#include "attn_common.cuh"
#include "kv_attn.cuh"

namespace kd {

// ---- a unit in shared memory --------------------------------------------------------------------------------------

template <int N>
__device__ __forceinline__ void lds(uint32_t at, uint32_t* w) {
  if constexpr (N == 16) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  } else if constexpr (N == 8) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  } else if constexpr (N == 4) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.u16 %0, [%1];" : "=r"(w[0]) : "r"(at));
  } else {
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(w[0]) : "r"(at));
  }
}
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// How a row of ROW bytes is spread over lanes. K: the four lanes t of a quad own pieces of KU bytes, 4 KU apart; V: the eight lanes g pieces of VU bytes.
template <int kBits, int D>
struct Spread {
  static constexpr int ROW = D * kBits / 8, PER = 8 / kBits;   // PER: numbers of a byte
  static constexpr int KU = ROW % 64 == 0 ? 16 : ROW % 32 == 0 ? 8 : ROW % 16 == 0 ? 4 : 2, KN = KU * PER, K_PIECES = ROW / 4 / KU, K_WORDS = K_PIECES * (KU > 4 ? KU / 4 : 1);
  static constexpr int VU = ROW == 128 ? 16 : ROW == 64 ? 8 : ROW % 32 == 0 ? 4 : ROW % 16 == 0 ? 2 : 1, VN = VU * PER, V_PIECES = ROW / 8 / VU, V_WORDS = V_PIECES * (VU > 4 ? VU / 4 : 1);
  // the first of the four head dims that lane t has of step s
  static __device__ __forceinline__ int k_dim(int s, int t) { return 4 * KN * (s / (KN / 4)) + KN * t + 4 * (s % (KN / 4)); }
  // ... and the inverse: dims d .. d + 3, d a multiple of 4
  static __device__ __forceinline__ int k_word(int d) { return d / (4 * KN) * (KN / 4) + d % KN / 4; }
  static __device__ __forceinline__ int k_lane(int d) { return d % (4 * KN) / KN; }
  // the head dim that number m of lane g's pieces of V is
  static __device__ __forceinline__ int v_dim(int m, int g) { return 8 * VN * (m / VN) + VN * g + m % VN; }
};

// A warp's copy of a unit: K, V, descriptors, scales. Rows of 128 or 64 bytes would put all rows into the same banks: the 16-byte pieces of a
// row change places, so that the eight lanes of a part of a load (two g, four t) find theirs in eight different ones: for K by the row's lowest bit,
// for V by the two above it.
template <int kBits, int D>
struct Stage {
  static constexpr int ROW = Spread<kBits, D>::ROW, GROUPS = D / K4_GROUP, SCALES = kBits == 4 ? KA_UNIT * GROUPS : 0;   // SCALES: bytes of the groups' scales, behind their numbers
  static constexpr int K4_AT = KA_UNIT * ROW, V_AT = K4_AT + SCALES, V4_AT = V_AT + KA_UNIT * ROW, DESC_AT = V4_AT + SCALES, SCALE_AT = DESC_AT + KA_UNIT * 4, BYTES = SCALE_AT + 128;
  static __device__ __forceinline__ uint32_t k_place(uint32_t o) { return ROW == 128 ? o ^ ((o >> 1) & 64u) : o; }
  static __device__ __forceinline__ uint32_t v_place(uint32_t o) { return ROW == 128 ? o ^ ((o >> 3) & 96u) : ROW == 64 ? o ^ ((o >> 2) & 96u) : o; }
};
// Where a lane finds things in its stage. The places of later steps and tokens are at fixed distances: the bits that a place depends on are the lane's own, but
// for every second step of V's copy at 128 bytes (bit 9) and V's odd tokens at 64 (bit 6).
template <int kBits, int D>
struct Lane {
  uint32_t copy_k, copy_v[2], k[Spread<kBits, D>::K_PIECES], v[2];
  __device__ __forceinline__ Lane() {
    using S = Stage<kBits, D>;
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    copy_k = S::k_place(lane * 16);
    copy_v[0] = S::V_AT + S::v_place(lane * 16);
    copy_v[1] = S::V_AT + S::v_place(lane * 16 + 512);
#pragma unroll
    for (int i = 0; i < Spread<kBits, D>::K_PIECES; ++i) k[i] = S::k_place(g * S::ROW + 4 * Spread<kBits, D>::KU * i + Spread<kBits, D>::KU * t);
    v[0] = S::V_AT + S::v_place(2 * t * S::ROW + Spread<kBits, D>::VU * g);
    v[1] = S::V_AT + S::v_place((2 * t + 1) * S::ROW + Spread<kBits, D>::VU * g);
  }
  // one operand's bytes, 16 a lane and step
  template <bool kV>
  __device__ __forceinline__ void copy(uint32_t stage, const uint8_t* from) const {
    using S = Stage<kBits, D>;
#pragma unroll
    for (int i = 0; i < (KA_UNIT * S::ROW + 511) / 512; ++i)
      if (512 * (i + 1) <= KA_UNIT * S::ROW || (threadIdx.x & 31) * 16 + 512 * i < KA_UNIT * S::ROW)
        cp_async16(stage + (!kV ? copy_k + 512 * i : copy_v[i & 1] + 512 * (i & ~1)), from + (threadIdx.x & 31) * 16 + 512 * i);
  }
  // lane (g, t): its pieces of an 8-token tile of K
  __device__ __forceinline__ void load_keys(uint32_t stage, int j, uint32_t* w) const {
    using S = Spread<kBits, D>;
#pragma unroll
    for (int i = 0; i < S::K_PIECES; ++i) lds<S::KU>(stage + k[i] + 8 * S::ROW * j, &w[i * (S::KU > 4 ? S::KU / 4 : 1)]);
  }
  // ... its pieces of the tokens 2t, 2t + 1, 2t + 8, 2t + 9 of 16
  __device__ __forceinline__ void load_values(uint32_t stage, int half, uint32_t (&w)[4][Spread<kBits, D>::V_WORDS]) const {
    using S = Spread<kBits, D>;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < S::V_PIECES; ++i) lds<S::VU>(stage + v[r & 1] + (16 * half + 8 * (r >> 1)) * S::ROW + 8 * S::VU * i, &w[r][i * (S::VU > 4 ? S::VU / 4 : 1)]);
  }
};

// Scales of 4-bit numbers as pairs of halves, and the numbers times them.
template <int D>
struct Scales4 {
  using S = Spread<4, D>;
  using St = Stage<4, D>;
  static constexpr int STEPS = S::KN < 16 ? S::KN / 4 : 4, K_COUNT = D / 16 / STEPS;   // steps of K that share a scale; scales of a lane's part of a key row
  // lane (g, t), its row of an 8-token tile of K: each twice
  static __device__ __forceinline__ void keys(uint32_t stage, int j, uint32_t (&w)[K_COUNT]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t row = stage + St::K4_AT + (8 * j + g) * St::GROUPS;
    if constexpr (S::KN == 32) {   // two groups, side by side
      uint32_t two;
      lds<2>(row + 2 * t, &two);
      w[0] = both_halves(two & 0xFFu);
      w[1] = both_halves(two >> 8);
    } else {
#pragma unroll
      for (int i = 0; i < K_COUNT; ++i) {
        uint32_t one;
        lds<1>(row + S::k_dim(i * STEPS, t) / K4_GROUP, &one);
        w[i] = both_halves(one);
      }
    }
  }
  // ... piece i of the tokens 2t, 2t + 1 (low, high) and 2t + 8, 2t + 9 of 16
  static __device__ __forceinline__ void values(uint32_t stage, int half, uint32_t (&w)[S::V_PIECES][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < S::V_PIECES; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t at = stage + St::V4_AT + (16 * half + 8 * x + 2 * t) * St::GROUPS + S::v_dim(i * S::VN, g) / K4_GROUP;
        uint32_t a, b;
        lds<1>(at, &a);
        lds<1>(at + St::GROUPS, &b);
        w[i][x] = (a | b << 16) << 7;
      }
  }
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// c = a b
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
// an 8 x 8 block of halves, lane (g, t) with row g and columns 2 t, 2 t + 1, transposed
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Query rows in shared memory: the operands of every step and what the mask needs. NT tiles of 8 rows.
template <int D, int NT>
struct QueryTile {
  uint2 frag[NT][D / 16][32];
  RowMask mask[NT * KA_TILE];
  float factor[NT * KA_TILE];   // what a row's products are to be multiplied with, sm_scale and log2(e) among it
  int min_limit;                // of the rows that see anything
};

// S^T of a unit: c[n][i][x] of lane (g, t): token 16 i + g + 8 (x >> 1), row 2 t + (x & 1) of tile n
// ... query(n, s): the operands of step s of tile n
template <int kBits, int D, int NT, typename F>
__device__ __forceinline__ void scores_of(uint32_t stage, const Lane<kBits, D>& at, F query, float (&c)[NT][2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    using S = Spread<kBits, D>;
    uint32_t k[2][S::K_WORDS];
    at.load_keys(stage, 2 * i, k[0]);
    at.load_keys(stage, 2 * i + 1, k[1]);
    uint32_t scale[2][Scales4<D>::K_COUNT];
    if constexpr (kBits == 4) {
      Scales4<D>::keys(stage, 2 * i, scale[0]);
      Scales4<D>::keys(stage, 2 * i + 1, scale[1]);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      HalfPairs lo, hi;
      if constexpr (kBits == 4) {
        constexpr int PIECE = S::KN / 4, WORDS = S::KU > 4 ? S::KU / 4 : 1;   // steps and words of a piece
        const int word = s / PIECE * WORDS + s % PIECE / 2, half = s % PIECE & 1;
        lo = e2m1x4_to_f16x4<(S::KU > 2)>(k[0][word], half, scale[0][s / Scales4<D>::STEPS]);
        hi = e2m1x4_to_f16x4<(S::KU > 2)>(k[1][word], half, scale[1][s / Scales4<D>::STEPS]);
      } else {
        lo = e4m3x4_to_f16x4(k[0][s]);
        hi = e4m3x4_to_f16x4(k[1][s]);
      }
      const uint4 a = make_uint4(lo.lo, hi.lo, lo.hi, hi.hi);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint2 b = query(n, s);
        if (s == 0) mma_f16_first(c[n][i], a, b.x, b.y);
        else mma_f16(c[n][i], a, b.x, b.y);
      }
    }
  }
}
template <int kBits, int D, int NT>
__device__ __forceinline__ void scores(uint32_t stage, const Lane<kBits, D>& at, const QueryTile<D, NT>& q, float (&c)[NT][2][4]) {
  const int lane = threadIdx.x & 31;
  scores_of<kBits, D, NT>(stage, at, [&](int n, int s) { return q.frag[n][s][lane]; }, c);
}

// bytes 0 and 1 (2 and 3) of two words in turn: for two tokens' values of two head dims
__device__ __forceinline__ uint32_t interleave(uint32_t a, uint32_t b, bool high) { return __byte_perm(a, b, high ? 0x7362 : 0x5140); }
// the bytes that are NaN, as bytes of ones
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// O^T += V^T P^T for 16 tokens. p: the tiles' operands (two words a tile). kSafe: see the head of the file; vis: the operands of indicators
template <int D, int NT, bool kSafe>
__device__ __forceinline__ void add_values(float (&o)[NT][D / 16][4], const uint32_t (&p)[NT][2], const uint32_t (&vis)[NT][2], const uint32_t (&v)[4][Spread<8, D>::V_WORDS]) {
  using S = Spread<8, D>;
  constexpr int PER = S::VU >= 4 ? 2 : 1;   // tiles of a word
#pragma unroll
  for (int w = 0; w < S::V_WORDS; ++w) {
#pragma unroll
    for (int half = 0; half < PER; ++half) {
      uint32_t b0 = interleave(v[0][w], v[1][w], half != 0), b1 = interleave(v[2][w], v[3][w], half != 0);
      const int m = w * PER + half;
      if constexpr (kSafe) {
        const uint32_t n0 = nan_bytes(b0), n1 = nan_bytes(b1);
        b0 &= ~n0;
        b1 &= ~n1;
        const HalfPairs one0 = e4m3x4_to_f16x4(n0 & 0x38383838u), one1 = e4m3x4_to_f16x4(n1 & 0x38383838u);   // 0x38: 1 in e4m3
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float hit[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(hit, make_uint4(one0.lo, one0.hi, one1.lo, one1.hi), vis[n][0], vis[n][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) o[n][m][i] = __uint_as_float(0x7FC00000u);
        }
      }
      const HalfPairs h0 = e4m3x4_to_f16x4(b0), h1 = e4m3x4_to_f16x4(b1);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(o[n][m], make_uint4(h0.lo, h0.hi, h1.lo, h1.hi), p[n][0], p[n][1]);
    }
  }
}

// ... for numbers of 4 bits. scale: of the pieces' tokens (see Scales4)
template <int D, int NT, bool kSafe>
__device__ __forceinline__ void add_values4(float (&o)[NT][D / 16][4], const uint32_t (&p)[NT][2], const uint32_t (&vis)[NT][2], const uint32_t (&v)[4][Spread<4, D>::V_WORDS],
                                            const uint32_t (&scale)[Spread<4, D>::V_PIECES][2]) {
  using S = Spread<4, D>;
  constexpr int WORDS = S::VU > 4 ? S::VU / 4 : 1, BYTES = S::VU > 4 ? 4 : S::VU;   // words of a piece, bytes of a word: a tile each
#pragma unroll
  for (int w = 0; w < S::V_WORDS; ++w) {
    const uint32_t (&sc)[2] = scale[w / WORDS];
    [[maybe_unused]] uint32_t gone[2];
    if constexpr (kSafe) {
      gone[0] = nan_scales(sc[0]);
      gone[1] = nan_scales(sc[1]);
    }
    // two tokens' numbers of one head dim side by side: the even dims', then the odd ones'
    uint32_t b[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint32_t a = v[2 * x][w], c = v[2 * x + 1][w];
      b[x][0] = (a & 0x0F0F0F0Fu) | (c << 4 & 0xF0F0F0F0u);
      b[x][1] = (a >> 4 & 0x0F0F0F0Fu) | (c & 0xF0F0F0F0u);
    }
#pragma unroll
    for (int i = 0; i < BYTES; ++i) {
      const int m = w * BYTES + i;
      uint32_t s0 = sc[0], s1 = sc[1];
      if constexpr (kSafe) {
        s0 &= ~gone[0];
        s1 &= ~gone[1];
        const uint32_t one0 = gone[0] & 0x3C003C00u, one1 = gone[1] & 0x3C003C00u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float hit[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(hit, make_uint4(one0, one0, one1, one1), vis[n][0], vis[n][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (hit[j] > 0.f) o[n][m][j] = __uint_as_float(0x7FC00000u);
        }
      }
      auto numbers = [&](int x, int y, uint32_t by) { return times(e2m1x2_to_f16x2<BYTES == 4>(b[x][y], i), by); };
      const uint4 a = make_uint4(numbers(0, 0, s0), numbers(0, 1, s0), numbers(1, 0, s1), numbers(1, 1, s1));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(o[n][m], a, p[n][0], p[n][1]);
    }
  }
}

// ---- query rows ---------------------------------------------------------------------------------------------------

// The query tiles of an item. fetch: loads, ahead of the item's first copies of the cache (behind them, with the copies of all CTAs on their way, they took
// 2 us); store: into shared memory, all threads of the CTA, ends with a barrier. bfloat16 rows are multiplied with the power of two that brings their largest finite number to 2^14
// (what falls below a half's subnormals is 2^-38 of it).
template <int kBits, int D, int NT>
struct QueryLoad {
  static constexpr int ROWS = NT * KA_TILE, PER = ROWS / KA_WARPS;   // rows of a warp, four numbers of each to a lane
  uint2 v[PER];
  RowMask mask;   // of thread r < ROWS: row r

  __device__ __forceinline__ void fetch(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const Item& it, int G, int rows) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = 4 * lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = it.tile * ROWS + warp * PER + i;
      v[i] = make_uint2(0u, 0u);
      if (row < rows && d < D) {
        const int n = row / G, hq = it.h * G + row - n * G;
        v[i] = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q.ptr) + it.b * p.q.stride_b + hq * p.q.stride_h + n * p.q.stride_t + d);
      }
    }
    if (threadIdx.x < ROWS) mask = row_mask(c, s, p, it, it.tile * ROWS + threadIdx.x, G, rows, query_count(c, p, it.b));
  }
  __device__ __forceinline__ void store(const kd_cache_queries& p, QueryTile<D, NT>& q) {
    using S = Spread<kBits, D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = 4 * lane;
    const bool bf16 = p.dtype == KD_BF16;
    if (threadIdx.x < ROWS) {
      q.mask[threadIdx.x] = mask;
      const int low = __reduce_min_sync(ROWS == 32 ? 0xFFFFFFFFu : (1u << ROWS) - 1u, mask.limit > 0 ? mask.limit : INT_MAX);
      if (threadIdx.x == 0) q.min_limit = low;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = warp * PER + i;
      int e = 0;
      if (bf16) e = row_to_halves(v[i]);
      if (lane == 0) q.factor[r] = row_factor(p.sm_scale, e);
      if (d < D) q.frag[r / KA_TILE][S::k_word(d)][(r % KA_TILE) * 4 + S::k_lane(d)] = v[i];
    }
    __syncthreads();
  }
};

// masks the scores of a unit (c as above); rows: the masks of a tile's rows
__device__ __forceinline__ void mask_scores(float (&c)[2][4], const uint32_t* desc, int j0, int g, int t, int end, const RowMask* rows) {
  const RowMask m[2] = {rows[2 * t], rows[2 * t + 1]};
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int at = 16 * i + 8 * y + g, token = j0 + at;
      const uint32_t kd = desc != nullptr ? desc[at] : TD_CTX;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bool see = token < end && ((kd & (token < m[x].limit ? m[x].sees | m[x].causal : m[x].sees)) != 0u || span_match_key(m[x].span_key, kd) != 0u);
        if (!see) c[i][2 * y + x] = -INFINITY;
      }
    }
}

// ---- the walk -----------------------------------------------------------------------------------------------------

// A warp's share of units first, first + KA_WARPS, ... below `last` of one head of a sequence, through two copies of its own: while
// one unit is worked on, the next is on its way. Accumulators: rows 2 t + {0, 1} of a tile (registers x & 1), head dims v_dim(2 m + (x >> 1), g); maxima and sums: rows 2 t and 2 t + 1.
template <int kBits, int D, int NT>
struct Walker {
  float o[NT][D / 16][4];
  float ref[NT][2], sum[NT][2];
  Scales scales;

  // starts the copies of a unit (nothing at or beyond `last`)
  static __device__ __forceinline__ void fetch(const kd_cache& c, const Lane<kBits, D>& place, int h, int unit, int last, int page, char* stage) {
    const int lane = threadIdx.x & 31;
    if (unit < last) {
      const uint32_t to = smem_u32(stage);
      page = checked_page(c, page);
      if (page >= 0) {
        const size_t at = block_index(c, page, h), token = at * KC_PAGE + (unit & 1) * KA_UNIT;
        place.template copy<false>(to, static_cast<const uint8_t*>(c.k) + token * Stage<kBits, D>::ROW);
        place.template copy<true>(to, static_cast<const uint8_t*>(c.v) + token * Stage<kBits, D>::ROW);
        if constexpr (kBits == 4) {
          const int piece = (lane & 15) * 16;
          if (piece < KA_UNIT * Stage<4, D>::GROUPS)
            cp_async16(to + (lane < 16 ? Stage<4, D>::K4_AT : Stage<4, D>::V4_AT) + piece, (lane < 16 ? scales4(c.k_scale) : scales4(c.v_scale)) + token * Stage<4, D>::GROUPS + piece);
        }
        if (c.desc != nullptr && lane < 8) cp_async16(to + Stage<kBits, D>::DESC_AT + lane * 16, c.desc + token + lane * 4);
        if (kBits == 8 && lane < 2) cp_async4(to + Stage<kBits, D>::SCALE_AT + lane * 4, (lane == 0 ? c.k_scale : c.v_scale) + at);
      } else if (kBits == 8 && lane < 2) {
        reinterpret_cast<float*>(stage + Stage<kBits, D>::SCALE_AT)[lane] = 1.f;   // (any bytes: all of it is masked)
      }
      if (lane == 0) *reinterpret_cast<int*>(stage + Stage<kBits, D>::SCALE_AT + 8) = page;
    }
    cp_async_commit();
  }
  // the first copy, and the page of the unit behind it
  static __device__ __forceinline__ int begin(const kd_cache& c, const kd_cache_seqs& s, const Lane<kBits, D>& place, const Item& it, int first, int last, char* ring) {
    const int32_t* table = s.table + it.b * s.table_stride;
    const int page = first < last ? table[first >> 1] : -1, next = first + KA_WARPS < last ? table[(first + KA_WARPS) >> 1] : -1;
    fetch(c, place, it.h, first, last, page, ring);
    return next;
  }

  // next_page: what begin returned
  // scores: of the item's first token, or null: they are not wanted
  // far: a second pass over rows that are (see KA_FAR). Scores are rounded first, ref is the largest and no more, and V's scale goes into the units of O instead.
  template <bool kSafe>
  __device__ __forceinline__ void walk(const kd_cache& c, const kd_cache_seqs& s, const Lane<kBits, D>& place, const Item& it, const QueryTile<D, NT>& q, int first, int last, int next_page,
                                       char* ring, float* all_scores, int score_rows, bool far) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      ref[n][0] = ref[n][1] = -INFINITY;
      sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][m][x] = 0.f;
    }
    const int32_t* table = s.table + it.b * s.table_stride;
    const int free_end = c.desc != nullptr ? 0 : q.min_limit;   // units below it need no mask
    scales = Scales{};
    int o_unit = 0;
    const float slack = kSafe && far ? 0.f : KA_SLACK;
    char* stage = ring;
    // One tile of rows over numbers of 4 bits: instructions are what bounds it, and what does not change from unit to unit stays in registers.
    constexpr bool kHold = kBits == 4 && NT == 1;
    [[maybe_unused]] uint2 held[kHold ? D / 16 : 1];
    [[maybe_unused]] float held_factor[2], held_add[2] = {0.f, 0.f};
    if constexpr (kHold) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) held[i] = q.frag[0][i][lane];
#pragma unroll
      for (int x = 0; x < 2; ++x) held_factor[x] = score_factor(1.f, q.factor[2 * t + x]);
    }
    for (int unit = first; unit < last; unit += KA_WARPS) {
      cp_async_wait<0>();
      __syncwarp();   // everyone's copies of this unit are there, and everyone is done with the one before it, whose place the next one takes
      char* other = stage == ring ? ring + Stage<kBits, D>::BYTES : ring;
      const int ahead = unit + KA_WARPS;
      fetch(c, place, it.h, ahead, last, next_page, other);
      if (ahead + KA_WARPS < last) next_page = table[(ahead + KA_WARPS) >> 1];
      const uint32_t at = smem_u32(stage);
      const float* scale = reinterpret_cast<const float*>(stage + Stage<kBits, D>::SCALE_AT);
      const uint32_t* desc = c.desc != nullptr ? reinterpret_cast<const uint32_t*>(stage + Stage<kBits, D>::DESC_AT) : nullptr;
      const int page = reinterpret_cast<const int*>(scale)[2], j0 = unit * KA_UNIT;
      const float ks = kBits == 4 ? 1.f : scale[0];   // (numbers of 4 bits have their scales in them)
      const int ev_page = kBits == 4 ? 0 : scale_exponent(scale[1]), ev = kSafe && far ? 0 : ev_page;   // (of far rows: nothing of it in the exponent)
      if (kBits == 8) scales.see(ev, ev);
      else scales.apart = false;
      if (kBits == 8 && kSafe && far && ev_page != o_unit) {
        const float to = exp2i(o_unit - ev_page);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < D / 16; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[n][m][x] *= to;
        o_unit = ev_page;
      }
      float sc[NT][2][4];
      if constexpr (kHold) scores_of<kBits, D, NT>(at, place, [&](int, int i) { return held[i]; }, sc);
      else scores<kBits, D, NT>(at, place, q, sc);
      uint32_t p[2][NT][2], vis[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (page < 0 || j0 + KA_UNIT > free_end) mask_scores(sc[n], desc, j0, g, t, page < 0 ? 0 : it.len, &q.mask[n * KA_TILE]);
        float k[2], add[2];
        if (NT == 1 && all_scores != nullptr && 2 * t < score_rows) {
          const float k0 = score_factor(ks, q.factor[2 * t]), k1 = score_factor(ks, q.factor[2 * t + 1]);
#pragma unroll
          for (int y = 0; y < 4; ++y)
            *reinterpret_cast<float2*>(all_scores + static_cast<size_t>(j0 + 8 * y + g) * score_rows + 2 * t) = make_float2(sc[n][y >> 1][2 * (y & 1)] * k0, sc[n][y >> 1][2 * (y & 1) + 1] * k1);
        }
        if constexpr (kHold) {
          // A row's reference stays while no lane has a score beyond it: the maximum over the lanes is formed only then.
          float top[2];
          bool moves = false;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            k[x] = held_factor[x];
            top[x] = fmaxf(fmaxf(sc[n][0][x], sc[n][0][2 + x]), fmaxf(sc[n][1][x], sc[n][1][2 + x])) * k[x];
            moves = moves | (top[x] > ref[n][x] + slack);
          }
          if (__any_sync(0xffffffffu, moves)) {
            float shrink[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 4));
              top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 8));
              top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 16));
              const float to = top[x] > ref[n][x] + slack ? top[x] : ref[n][x];
              shrink[x] = to == ref[n][x] ? 1.f : fast_exp2(ref[n][x] - to);
              ref[n][x] = to;
              held_add[x] = to == -INFINITY ? 0.f : KA_OFFSET - to;
              sum[n][x] *= shrink[x];
              scales.look(to);
            }
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[n][m][x] *= shrink[x & 1];
          }
          add[0] = held_add[0];
          add[1] = held_add[1];
        } else {
          float high[2], old[2];
          bool moves = false;
          auto set_add = [&](int x) { add[x] = ref[n][x] == -INFINITY ? 0.f : static_cast<float>(ev) + KA_OFFSET - ref[n][x]; };
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            k[x] = score_factor(ks, q.factor[n * KA_TILE + 2 * t + x]);
            // the row's maximum, over the lanes of its tokens
            float top = fmaxf(fmaxf(sc[n][0][x], sc[n][0][2 + x]), fmaxf(sc[n][1][x], sc[n][1][2 + x]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            high[x] = fmaf(top, k[x], static_cast<float>(ev));
            old[x] = ref[n][x];
            const bool up = high[x] > old[x] + slack;
            moves = moves | up | (scales.apart & (high[x] < old[x] - KA_DEPTH));   // (no branch here: it costs 4 % of the time with 32 rows; -inf is seen to below)
            ref[n][x] = up ? high[x] : old[x];   // (ahead of the vote: the exponentials wait for it)
            set_add(x);
          }
          if (__any_sync(0xffffffffu, moves)) {
            float shrink[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) shrink[x] = ref[n][x] == old[x] ? 1.f : fast_exp2(old[x] - ref[n][x]);
            if (kBits == 8 && scales.ever())
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                float total = sum[n][x];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                if (ref[n][x] != old[x]) ref[n][x] = rintf(high[x]);
                else if (scales.apart && below_reference(high[x], old[x])) ref[n][x] = reference_below(high[x], old[x], total);
                set_add(x);
                shrink[x] = rescale(old[x], ref[n][x]);
              }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              sum[n][x] *= shrink[x];
              scales.look(ref[n][x]);
            }
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[n][m][x] *= shrink[x & 1];
          }
        }
        if constexpr (kSafe) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              vis[i][n][y] = transpose8x8((sc[n][i][2 * y] == -INFINITY ? 0u : 0x3C00u) | (sc[n][i][2 * y + 1] == -INFINITY ? 0u : 0x3C000000u));
        }
        if (kSafe && far)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              float& v = sc[n][y >> 1][2 * (y & 1) + x];
              v = __fsub_rn(__fmul_rn(v, k[x]), ref[n][x] == -INFINITY ? 0.f : ref[n][x]);
            }
            k[x] = 1.f;
            add[x] = KA_OFFSET;
          }
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float a = fast_exp2(fmaf(sc[n][i][2 * y], k[0], add[0])), b = fast_exp2(fmaf(sc[n][i][2 * y + 1], k[1], add[1]));
            part[0] += a;
            part[1] += b;
            p[i][n][y] = transpose8x8(pack2<false>(a, b));
          }
        const float unscale = exp2i(-ev);
        sum[n][0] = kBits == 4 ? sum[n][0] + part[0] : fmaf(part[0], unscale, sum[n][0]);
        sum[n][1] = kBits == 4 ? sum[n][1] + part[1] : fmaf(part[1], unscale, sum[n][1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t v[4][Spread<kBits, D>::V_WORDS];
        place.load_values(at, i, v);
        if constexpr (kBits == 4) {
          uint32_t scale4[Spread<4, D>::V_PIECES][2];
          Scales4<D>::values(at, i, scale4);
          add_values4<D, NT, kSafe>(o, p[i], kSafe ? vis[i] : p[i], v, scale4);
        } else {
          add_values<D, NT, kSafe>(o, p[i], kSafe ? vis[i] : p[i], v);
        }
      }
      stage = other;
    }
    cp_async_wait<0>();
    __syncwarp();
    if (kBits == 8 && kSafe && far) {
      const float to = exp2i(o_unit);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][m][x] *= to;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[n][x] += __shfl_xor_sync(0xffffffffu, sum[n][x], o);
  }

  __device__ __forceinline__ bool any_nan() const {
    bool bad = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int x = 0; x < 4; ++x) bad = bad || is_nan(o[n][m][x]);
    return __any_sync(0xffffffffu, bad);
  }
};

// Shared memory of the kernel. A warp's rows of O take the place of its second copy (and more, with many rows) when it is through; the first one belongs to the next item by then.
template <int kBits, int D, int NT>
struct AttnShared {
  static constexpr int ROWS = NT * KA_TILE, O_BYTES = ROWS * (D + 4) * 4;
  struct Warp {
    char stage[2 * Stage<kBits, D>::BYTES + (O_BYTES > Stage<kBits, D>::BYTES ? O_BYTES - Stage<kBits, D>::BYTES + 127 & ~127 : 0)];
    __device__ __forceinline__ float* o(int row) { return reinterpret_cast<float*>(stage + Stage<kBits, D>::BYTES) + row * (D + 4); }
  } warp[KA_WARPS];
  QueryTile<D, NT> q;
  ItemShare next;
  float2 ml[KA_WARPS][ROWS];      // the warps' maxima and sums
  float scale[KA_WARPS][ROWS];    // what a warp's rows are multiplied with: all on one maximum, and divided by the sum where the item is whole
};

template <int kBits, int D, int NT>
__global__ void __launch_bounds__(KA_THREADS, ctas_of(NT))
cache_attention_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                       const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  touch_parameters(c, s, p, shape, ws);
  pdl_wait();
  pdl_launch_dependents();
  constexpr int ROWS = NT * KA_TILE;
  extern __shared__ __align__(1024) char smem[];
  AttnShared<kBits, D, NT>& sh = *reinterpret_cast<AttnShared<kBits, D, NT>*>(smem);
  const Lane<kBits, D> place;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  ItemShare share = share_of_cta(c, s, p, shape, 0);
  if (share.here < 0) return;
  char* ring = sh.warp[warp].stage;
  QueryLoad<kBits, D, NT> queries;
  int first, last, next_page;
  auto begin = [&]() {   // an item's first loads
    first = 2 * share.page0 + warp;
    last = min(2 * (share.page0 + share.here), (share.it.len + KA_UNIT - 1) / KA_UNIT);
    queries.fetch(c, s, p, share.it, shape.G, shape.rows);
    next_page = Walker<kBits, D, NT>::begin(c, s, place, share.it, first, last, ring);
  };
  begin();
#pragma unroll 1
  for (uint32_t done = share.here;;) {   // (with even pages an item has at least one: `done` grows)
    const Item it = share.it;
    const bool whole = share.here == share.pages;
    queries.store(p, sh.q);
    if (shape.even && warp == 0) {   // what comes next is looked up while this item's copies are on their way
      const ItemShare next = share_of_cta(c, s, p, shape, done);
      if (lane == 0) sh.next = next;
    }
    Walker<kBits, D, NT> w;
    float* scores = shape.score_rows > 0 ? ws.scores + (static_cast<size_t>(it.b) * c.H + it.h) * s.blocks * KC_PAGE * shape.score_rows : nullptr;
    w.template walk<false>(c, s, place, it, sh.q, first, last, next_page, ring, scores, shape.score_rows, false);
    const bool far = __any_sync(0xffffffffu, w.scales.met_far());
    if (w.any_nan() || far) {
      next_page = Walker<kBits, D, NT>::begin(c, s, place, it, first, last, ring);
      w.template walk<true>(c, s, place, it, sh.q, first, last, next_page, ring, nullptr, 0, far);
    }
    if (g == 0)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) sh.ml[warp][n * KA_TILE + 2 * t + x] = make_float2(w.ref[n][x], w.sum[n][x]);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int m = 0; m < D / 16; ++m)
#pragma unroll
        for (int x = 0; x < 4; ++x) sh.warp[warp].o(n * KA_TILE + 2 * t + (x & 1))[Spread<kBits, D>::v_dim(2 * m + (x >> 1), g)] = w.o[n][m][x];
    const size_t part = share.part;
    __syncthreads();
    if (shape.even) {   // its first copies run while this one's rows are put together
      share = sh.next;
      if (share.here >= 0) begin();
    }
    auto place_of_row = [&](int row, int& hq, int& i) {   // of the key head
      i = row / shape.G;
      hq = it.h * shape.G + row - i * shape.G;
    };
    if (tid < ROWS && it.tile * ROWS + tid < shape.rows) {
      float ref = -INFINITY, sum = 0.f, scale[KA_WARPS];
#pragma unroll
      for (int k = 0; k < KA_WARPS; ++k) ref = fmaxf(ref, sh.ml[k][tid].x);
#pragma unroll
      for (int k = 0; k < KA_WARPS; ++k) {
        scale[k] = sh.ml[k][tid].x == -INFINITY ? 0.f : fast_exp2(sh.ml[k][tid].x - ref);
        sum = fmaf(sh.ml[k][tid].y, scale[k], sum);
      }
      const bool live = sh.q.mask[tid].limit > 0;
      const float inv = whole ? (live && sum != 0.f ? 1.f / sum : -1.f) : 1.f;   // -1: nothing is seen
#pragma unroll
      for (int k = 0; k < KA_WARPS; ++k) sh.scale[k][tid] = inv < 0.f ? -1.f : scale[k] * inv;
      if (whole) {
        int hq, i;
        place_of_row(it.tile * ROWS + tid, hq, i);
        write_stats(p, ws, shape.stats, (static_cast<size_t>(it.b) * p.H + hq) * p.T + i, live, ref, sum);
      } else {
        ws.part_ml[part * ROWS + tid] = make_float2(ref, sum);
      }
    }
    __syncthreads();
    const int rows = min(ROWS, shape.rows - it.tile * ROWS);
    for (int x = tid; x < rows * (D / 4); x += KA_THREADS) {
      const int r = x / (D / 4), d = (x - r * (D / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (sh.scale[0][r] >= 0.f || is_nan(sh.scale[0][r])) {
#pragma unroll
        for (int k = 0; k < KA_WARPS; ++k) {
          const float f = sh.scale[k][r];
          const float4 y = *reinterpret_cast<const float4*>(sh.warp[k].o(r) + d);
          v.x = fmaf(y.x, f, v.x);
          v.y = fmaf(y.y, f, v.y);
          v.z = fmaf(y.z, f, v.z);
          v.w = fmaf(y.w, f, v.w);
        }
      }
      if (whole) {
        int hq, i;
        place_of_row(it.tile * ROWS + r, hq, i);
        uint16_t* out = static_cast<uint16_t*>(p.o.ptr) + it.b * p.o.stride_b + hq * p.o.stride_h + i * p.o.stride_t + d;
        *reinterpret_cast<uint2*>(out) = p.dtype == KD_BF16 ? make_uint2(pack2<true>(v.x, v.y), pack2<true>(v.z, v.w)) : make_uint2(pack2<false>(v.x, v.y), pack2<false>(v.z, v.w));
      } else {
        *reinterpret_cast<float4*>(ws.part_o + (part * ROWS + r) * D + d) = v;
      }
    }
    if (!shape.even || share.here < 0) return;
    done += share.here;
    __syncthreads();   // shared memory is free for the next item
  }
}

// no more than 1 (the statistics of many rows are from scores that were added up in another order: in far rows that can be many powers of two), and NaN stays NaN
__device__ __forceinline__ float at_most_one(float x) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(1.f));
  return y;
}

// weights[j] += sum over the query rows of the head of softmax_j, from the rows' maxima and sums. A warp has a unit of tokens for all
// rows, so that nothing is added twice and the order is fixed; a CTA kPages pages of one head: 8, and 2 where those would be CTAs for less than half
// of the SMs (8 x 2000 tokens of one head, 1024 rows: 203 us with 2, 301 with 8; 2 x 8192 tokens of 8 heads, 512 rows: 284 and 223; now 206 and 231: each CTA goes through all query rows). The queries of the next tile of rows are asked for before the tile in hand is worked on.
template <int kBits, int D>
constexpr int KW_STAGE = Stage<kBits, D>::V_AT + KA_UNIT * 4;   // K and descriptors
template <int kBits, int D, int NT, int kPages>
__global__ void __launch_bounds__(KA_THREADS)
cache_weights_kernel(const __grid_constant__ kd_cache c, const __grid_constant__ kd_cache_seqs s, const __grid_constant__ kd_cache_queries p,
                     const __grid_constant__ AttnShape shape, const __grid_constant__ AttnWorkspace ws) {
  touch_parameters(c, s, p, shape, ws);
  pdl_wait();
  pdl_launch_dependents();
  constexpr int UNITS = 2 * kPages, MINE = UNITS / KA_WARPS, ROWS = NT * KA_TILE;
  extern __shared__ __align__(1024) char smem[];
  char* stages = smem + (threadIdx.x >> 5) * MINE * KW_STAGE<kBits, D>;
  QueryTile<D, NT>& q = *reinterpret_cast<QueryTile<D, NT>*>(smem + UNITS * KW_STAGE<kBits, D>);
  __shared__ float2 s_stat[ROWS];
  const Lane<kBits, D> place;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, groups = (s.blocks + kPages - 1) / kPages;
  uint32_t item = blockIdx.x;
  const int first = static_cast<int>(item % static_cast<uint32_t>(groups)) * UNITS + warp;
  item /= static_cast<uint32_t>(groups);
  Item it;
  it.h = static_cast<int>(item % static_cast<uint32_t>(c.H));
  it.b = static_cast<int>(item / static_cast<uint32_t>(c.H));
  it.len = sequence_length(c, s, it.b);
  if ((first - warp) * KA_UNIT >= it.len) return;
  int page[MINE];
  float ks[MINE], sums[MINE][4];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int unit = first + i * KA_WARPS;
    page[i] = unit * KA_UNIT < it.len ? page_of(c, s, it.b, unit >> 1) : -1;
    ks[i] = 1.f;
    if (page[i] >= 0) {
      const size_t at = block_index(c, page[i], it.h), token = at * KC_PAGE + (unit & 1) * KA_UNIT;
      const uint32_t to = smem_u32(stages + i * KW_STAGE<kBits, D>);
      place.template copy<false>(to, static_cast<const uint8_t*>(c.k) + token * Stage<kBits, D>::ROW);
      if (kBits == 4 && lane * 16 < KA_UNIT * Stage<4, D>::GROUPS) cp_async16(to + Stage<4, D>::K4_AT + lane * 16, scales4(c.k_scale) + token * Stage<4, D>::GROUPS + lane * 16);
      if (c.desc != nullptr && lane < 8) cp_async16(to + Stage<kBits, D>::V_AT + lane * 16, c.desc + token + lane * 4);
      if (kBits == 8) ks[i] = c.k_scale[at];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) sums[i][x] = 0.f;
  }
  cp_async_commit();
  QueryLoad<kBits, D, NT> queries;
  it.tile = 0;
  queries.fetch(c, s, p, it, shape.G, shape.rows);
  for (int tile = 0; tile < shape.tiles; ++tile) {
    queries.store(p, q);
    it.tile = tile + 1;
    if (it.tile < shape.tiles) queries.fetch(c, s, p, it, shape.G, shape.rows);
    if (tid < ROWS) {
      const int r = tile * ROWS + tid, i = r / shape.G;
      s_stat[tid] = r < shape.rows ? ws.stats[(static_cast<size_t>(it.b) * p.H + it.h * shape.G + r - i * shape.G) * p.T + i] : make_float2(0.f, 0.f);
    }
    cp_async_wait<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (page[i] < 0) continue;
      const char* stage = stages + i * KW_STAGE<kBits, D>;
      const int j0 = (first + i * KA_WARPS) * KA_UNIT;
      float sc[NT][2][4];
      scores<kBits, D, NT>(smem_u32(stage), place, q, sc);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (c.desc != nullptr || j0 + KA_UNIT > q.min_limit)
          mask_scores(sc[n], c.desc != nullptr ? reinterpret_cast<const uint32_t*>(stage + Stage<kBits, D>::V_AT) : nullptr, j0, g, t, it.len, &q.mask[n * KA_TILE]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = n * KA_TILE + 2 * t + x;
          const float2 st = s_stat[r];
          const float f = score_factor(ks[i], q.factor[r]);
#pragma unroll
          for (int y = 0; y < 4; ++y) {   // (from rounded scores, as the statistics of far rows are)
            const float v = sc[n][y >> 1][2 * (y & 1) + x], pr = at_most_one(fast_exp2(__fsub_rn(__fmul_rn(v, f), st.x) + KA_OFFSET) * st.y);
            if (st.y != 0.f && v != -INFINITY) sums[i][y] += pr;   // rows that exist, tokens that they see
          }
        }
      }
    }
    __syncthreads();   // the tile in shared memory is free
  }
#pragma unroll
  for (int i = 0; i < MINE; ++i)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      sums[i][y] += __shfl_xor_sync(0xffffffffu, sums[i][y], 1);
      sums[i][y] += __shfl_xor_sync(0xffffffffu, sums[i][y], 2);
      const int j = (first + i * KA_WARPS) * KA_UNIT + 8 * y + g;
      if (t == 0 && page[i] >= 0 && j < it.len && j < p.w_len) p.weights[it.b * p.w_stride_b + it.h * p.w_stride_h + j] += sums[i][y];
    }
}

// the weights from the rows' statistics
template <int kBits, int D, int NT, int kPages>
static cudaError_t launch_weights_of(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, AttnShape a, const AttnWorkspace& ws, cudaStream_t stream) {
  const int64_t groups = static_cast<int64_t>(s.B) * c.H * ((s.blocks + kPages - 1) / kPages);
  constexpr size_t kShared = 2 * kPages * KW_STAGE<kBits, D> + sizeof(QueryTile<D, NT>);
  static SmemOptIn opt_in;
  static SharedFirst shared_first;
  a.item_rows = NT * KA_TILE;
  a.tiles = (a.rows + a.item_rows - 1) / a.item_rows;
  cudaError_t e = opt_in(cache_weights_kernel<kBits, D, NT, kPages>, kShared);
  if (e == cudaSuccess) e = shared_first(cache_weights_kernel<kBits, D, NT, kPages>);
  return e != cudaSuccess ? e : launch(cache_weights_kernel<kBits, D, NT, kPages>, static_cast<unsigned>(groups), KA_THREADS, kShared, stream, c, s, p, a, ws);
}

template <int kBits, int D, int NT>
static cudaError_t launch_weights(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  if (!a.stats || s.blocks == 0) return cudaSuccess;
  const bool few = static_cast<int64_t>(s.B) * c.H * s.blocks < 148 / 2 * 8;
  return few ? launch_weights_of<kBits, D, NT, 2>(c, s, p, a, ws, stream) : launch_weights_of<kBits, D, NT, 8>(c, s, p, a, ws, stream);
}

template <int kBits, int D, int NT>
static cudaError_t launch_rows(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  constexpr size_t kShared = sizeof(AttnShared<kBits, D, NT>);
  static SmemOptIn opt_in;
  static SharedFirst shared_first;
  cudaError_t e = opt_in(cache_attention_kernel<kBits, D, NT>, kShared);
  if (e == cudaSuccess) e = shared_first(cache_attention_kernel<kBits, D, NT>);
  const int64_t items = static_cast<int64_t>(s.B) * c.H * a.tiles;
  return e != cudaSuccess ? e : launch_shares(a.ctas > 0 && a.even, cache_attention_kernel<kBits, D, NT>, static_cast<unsigned>(a.ctas > 0 ? a.ctas : items), KA_THREADS, kShared, stream, c, s, p, a, ws);
}

template <int kBits, int D>
static cudaError_t launch_rows_dim(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  return a.item_rows == KA_TILE ? launch_rows<kBits, D, 1>(c, s, p, a, ws, stream) : a.item_rows == 2 * KA_TILE ? launch_rows<kBits, D, 2>(c, s, p, a, ws, stream) : launch_rows<kBits, D, 4>(c, s, p, a, ws, stream);
}
template <int kBits, int D>
static cudaError_t launch_weights_dim(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  return a.item_rows <= 2 * KA_TILE ? launch_weights<kBits, D, 2>(c, s, p, a, ws, stream) : launch_weights<kBits, D, 4>(c, s, p, a, ws, stream);   // (one tile of rows: beyond scores_limit)
}

}  // namespace kd
