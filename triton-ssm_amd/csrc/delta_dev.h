// Device pieces of the gated delta rule's chunked kernels (planes.h: the products).
#pragma once

#include "delta.h"
#include "planes.h"

namespace tssm {
namespace {

constexpr int kC = 32;            // steps of a chunk
constexpr int kTld = 40;          // bf16 elements of a row of T or P in LDS

typedef RowsOf<kC> ChunkRows;

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
