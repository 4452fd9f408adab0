// Device pieces of the gated delta rule's chunked kernels.
//
// Products on the matrix cores take bf16 operands.  An fp32 value goes in as
// the sum of three bf16 planes (x = b0 + b1 + b2 exactly up to 2^-24: each
// plane takes 8 bits of what the planes before left), and a product of two
// such values as the six plane products b_i b_j with i + j <= 2, whose
// rejects are below 2^-24.  A bf16 input is one plane, exactly.  Three planes
// cost 3 (against a bf16 operand) or 6 matrix instructions where the fp32
// matrix instruction takes the time of 16.
//
// Layout.  v_mfma_f32_16x16x32_bf16: lane (j, c) = (lane / 16, lane % 16) holds
// A[c][8 j + e], B[8 j + e][c], e < 8, and the result's rows 4 j + r, r < 4, of
// column c.  A 32-row operand X (steps of a chunk, or 32 rows of the state)
// lives in two result tiles, tile h row 4 j + r holding X's row 8 j + 4 h + r:
// the two tiles' registers of a lane are then X[8 j + 4 h + r][c] =
// X[8 j + e][c], the B operand of the next product as they stand.  Nothing
// crosses lanes between the products of a chunk.
#pragma once

#include "delta.h"

namespace tssm {
namespace {

constexpr int kC = 32;            // steps of a chunk
constexpr int kTld = 40;          // bf16 elements of a row of T or P in LDS

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

__device__ inline f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ inline f32x4 zero4() { return f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }

// The first NP planes of 8 values, as operands.
template <int NP>
__device__ inline void split8(const float* x, u32x4* p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const uint32_t w = pk_bf16(a, b);
      p[n][i] = w;
      if (n + 1 < NP) {
        a -= __uint_as_float(w << 16);
        b -= __uint_as_float(w & 0xffff0000u);
      }
    }
  }
}

// Planes of two result tiles (one 32-row operand) as a B operand.
template <int NP>
__device__ inline void split_tiles(const f32x4& lo, const f32x4& hi, u32x4* p) {
  const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  split8<NP>(x, p);
}

// acc += A B over the plane pairs (i, j) with i + j < MAXP.
template <int NA, int NB, int MAXP>
__device__ inline f32x4 mfma_planes(const u32x4* a, const u32x4* b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < MAXP) acc = mfma32(a[i], b[j], acc);
  return acc;
}

// Eight consecutive elements of a row as they lie in memory, and as planes.
template <typename T, bool VEC>
struct Piece {
  static constexpr int NP = sizeof(T) == 2 && std::is_same<T, bf16_t>::value ? 1 : 3;
  static constexpr int kW = VEC ? 8 * (int)sizeof(T) / 16 : 8;
  typedef std::conditional_t<VEC, u32x4,
                             std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>> word;
  union {
    word w[kW];
    T e[8];
  };
  // lim: elements that exist (the others read p[0], which does)
  __device__ inline void load(const T* p, int lim) {
#pragma unroll
    for (int i = 0; i < kW; ++i)
      w[i] = reinterpret_cast<const word*>(p)[VEC || i < lim ? i : 0];
  }
  __device__ inline void planes(int lim, u32x4* out) const {
    if constexpr (NP == 1 && VEC) {
      out[0] = lim > 0 ? w[0] : u32x4{0, 0, 0, 0};
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < lim ? ldf(&e[i]) : 0.0f;
      split8<NP>(x, out);
    }
  }
};

// LDS reads of A operands.
__device__ inline u32x4 lds16(const uint16_t* p) { return *reinterpret_cast<const u32x4*>(p); }
// Four elements of column lane % 16 from the rows that the quads of each
// 16-lane group point at.
__device__ inline u32x2v lds_tr(const uint16_t* p) {
  auto q = (__attribute__((address_space(3))) s16x4*)(p);
  return __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q));
}
// The A operand M^T for the row-major M [32][ld] in LDS: rows of the result are
// the columns col + 8 (ρ / 4) + ρ % 4 (ρ < 16) of M, the sum runs over M's rows.
__device__ inline u32x4 lds_col(const uint16_t* m, int ld, int col, int lane) {
  const int j = lane >> 4, i = lane & 15;
  const uint16_t* p = m + (8 * j + (i >> 2)) * ld + col + 8 * (i & 3);
  const u32x2v a = lds_tr(p), b = lds_tr(p + 4 * ld);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// What the preparing pass leaves for each chunk and value head, in the
// workspace.  Rows past the sequence's end count as k = q = 0, g = beta = 0.
template <int NPP>
struct ChunkWs {
  uint16_t T[3][kC][kC];    // planes of (I + A)^-1
  uint16_t P[NPP][kC][kC];  // planes of scale (Q K^T) o D
  float fac[4][kC];         // e^{G_t}, beta_t, e^{G_last - G_t}, g_t
};

}  // namespace
}  // namespace tssm
