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

// What the bf16 values in w leave of (a, b): one v_dot2c each, which takes the
// plane as it is packed; every intermediate is exact.  The constants (-1 in
// one half) come through asm: folded as literals they reach the instruction
// in the wrong half.
__device__ inline void take_plane(uint32_t w, float& a, float& b) {
  uint32_t lo, hi;
  asm("s_mov_b32 %0, 0xbf80" : "=s"(lo));
  asm("s_mov_b32 %0, 0xbf800000" : "=s"(hi));
  const hw_bf16x2 p = __builtin_bit_cast(hw_bf16x2, w);
  a = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(hw_bf16x2, lo), a, false);
  b = __builtin_amdgcn_fdot2_f32_bf16(p, __builtin_bit_cast(hw_bf16x2, hi), b, false);
}

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
      if (n + 1 < NP) take_plane(w, a, b);
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
  // through a buffer descriptor, whose end bounds the access
  __device__ inline void load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      if constexpr (VEC) w[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, 0, 0);
      else if constexpr (sizeof(T) == 4) w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, off + 4 * i, 0, 0);
      else w[i] = __builtin_amdgcn_raw_buffer_load_b16(r, off + 2 * i, 0, 0);
    }
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

// The rows of a tensor for one batch and head: at(n) is a buffer descriptor of
// chunk n whose end is the chunk's last row's, so that rows past the sequence
// read zero and drop stores.  (Rows must not overlap, and their offsets within
// a chunk take 31 bits: delta.hip sees to it.)  A chunk outside the sequence
// is taken for the nearest one in it: loads ahead need no branch.
struct ChunkRows {
  const char* p;
  int64_t step;             // bytes of 32 rows
  int row, full, end, last; // bytes of a row, a full chunk, the last chunk; its number
  template <typename T>
  __device__ inline void init(const T* base, int64_t stride, int cols, int64_t L) {
    p = reinterpret_cast<const char*>(base);
    row = (int)(stride * (int64_t)sizeof(T));
    step = stride * (int64_t)sizeof(T) * kC;
    last = (int)((L - 1) / kC);
    full = (kC - 1) * row + cols * (int)sizeof(T);
    end = (int)((L - 1) % kC) * row + cols * (int)sizeof(T);
  }
  __device__ inline __amdgpu_buffer_rsrc_t at(int n) const {
    const int m = n < 0 ? 0 : (n < last ? n : last);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p + m * step), (short)0,
                                             m < last ? full : end, 0x00020000);
  }
};
constexpr uint32_t kPast = 0x7ffffff0u;  // an offset past every descriptor's end

template <typename T>
__device__ inline T buf_elem(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (sizeof(T) == 4)
    return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
  else
    return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
}
template <typename T>
__device__ inline void buf_put(__amdgpu_buffer_rsrc_t r, uint32_t off, float x) {
  T y;
  stf(&y, x);
  if constexpr (sizeof(T) == 4)
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, y), r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, y), r, off, 0, 0);
}

// A workgroup's waves meet; what they wrote to LDS is there for all.  (Global
// loads and stores stay in flight, unlike with __syncthreads.)
__device__ inline void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ inline __amdgpu_buffer_rsrc_t rsrc_of(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
}

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

// The same for the 16 columns from col on.
__device__ inline u32x4 lds_col16(const uint16_t* m, int ld, int col, int lane) {
  const int j = lane >> 4, i = lane & 15;
  const uint16_t* p = m + (8 * j + (i >> 2)) * ld + col + 4 * (i & 3);
  const u32x2v a = lds_tr(p), b = lds_tr(p + 4 * ld);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// What the preparing pass leaves for each chunk and value head, in the
// workspace.  Steps past the sequence's end count as k = q = 0, g = beta = 0.
// With G the sums of g within the chunk:
//   fac: e^{G_t}, beta_t, e^{G_last - G_t}, g_t, and G_t log2(e) in two parts
enum { kEg, kBeta, kEnd, kG, kGhi, kGlo, kFac = 8 };
//   T: planes of (I + A)^-1, which is 0 above the diagonal: rows 16 to 31, then
//   the left half of rows 0 to 15
struct ChunkWs {
  struct {
    uint16_t below[16][32], first[16][16];
  } T[3];
  float fac[kFac][kC];
};
constexpr int kPlane = 16 * 48 * 2;  // bytes of a plane of T

// The offset in ChunkWs of 8 elements of a plane from row id / 4, column
// 8 (id % 4) on, or one past the end, where zeros are read.
__device__ inline uint32_t t_at(int plane, int id) {
  const int at = id >= 64 ? 16 * (id - 64) : 1024 + 16 * (id >> 2) * 2 + 16 * (id & 1);
  return id < 64 && (id & 2) ? kPast : plane * kPlane + at;
}

__device__ inline const ChunkWs* chunk_at(const ChunkWs* ws, int n, int nch) {
  return ws + (n < 0 ? 0 : (n < nch ? n : nch - 1));
}

// The state (or its gradient) of one value head in the workspace: [Vp][KP]
// fp32, column by column, Vp = V rounded up to 16, zero past K and V.  A lane's
// rows 8 j .. 8 j + 7 of 32 are 32 bytes.
template <int NS>
__device__ inline void put_cols(float* m, const f32x4 (&S)[2 * NS], int64_t col, int j) {
  float* p = m + col * 32 * NS + 8 * j;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
    *reinterpret_cast<f32x4*>(p + 32 * (i >> 1) + 4 * (i & 1)) = S[i];
}
template <int NS>
__device__ inline void get_cols(const float* m, f32x4 (&S)[2 * NS], int64_t col, int j) {
  const float* p = m + col * 32 * NS + 8 * j;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
    S[i] = *reinterpret_cast<const f32x4*>(p + 32 * (i >> 1) + 4 * (i & 1));
}
// The same from and to a caller's [K][V] state.
template <int NS>
__device__ inline void get_state(const float* m, f32x4 (&S)[2 * NS], int64_t col, int64_t V, int K,
                                 int j) {
  const bool on = m && col < V;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
      const float x = m ? m[(int64_t)(k < K ? k : 0) * V + (on ? col : 0)] : 0.0f;
      S[i][r] = on && k < K ? x : 0.0f;
    }
}
template <int NS>
__device__ inline void put_state(float* m, const f32x4 (&S)[2 * NS], int64_t col, int64_t V, int K,
                                 int j) {
  if (!m || col >= V) return;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
      if (k < K) m[(int64_t)k * V + col] = S[i][r];
    }
}

}  // namespace
}  // namespace tssm
