// Device pieces of linear attention's chunked kernels (planes.h: the products).
#pragma once

#include "linattn.h"
#include "planes.h"

namespace tssm {
namespace {

// Planes of an input (fp32 three, fp16 two, bf16 one: exactly), and of what is
// formed on the way to the outputs alone (two, each 2^-17 of a term of sums that are
// rounded to 2^-8 or 2^-11 at the end: with the planes' products left out 2^-16, which
// counts where terms cancel by more than 2^8 or 2^5; three where nothing is rounded).
// What reaches the state always has three.
template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : (std::is_same<T, bf16_t>::value ? 1 : 2);
template <typename T>
constexpr int kOutPlanes = sizeof(T) == 4 ? 3 : 2;

// A state in the workspace lies as the waves hold it: tiles [Vp / 16][KP / 16] of
// 64 lanes x 4, tile (vt, 2 s + x) lane (j, c) register r holding S[32 s + 8 j + 4 x
// + r][16 vt + c]; Vp is V rounded up to 32, zero past K and V.
__host__ __device__ inline int64_t lin_state_elems(int64_t KP, int64_t V) {
  return KP * ((V + 31) / 32 * 32);
}

// A tile's lane of a caller's [K][V] state, zero past K and V or without one.
__device__ inline f32x4 get_tile(const float* m, int kt, int64_t col, int64_t V, int K, int j) {
  const bool on = m && col < V;
  f32x4 S;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int k = 32 * (kt >> 1) + 8 * j + 4 * (kt & 1) + r;
    const float x = m ? m[(int64_t)(k < K ? k : 0) * V + (on ? col : 0)] : 0.0f;
    S[r] = on && k < K ? x : 0.0f;
  }
  return S;
}
__device__ inline void put_tile(float* m, const f32x4& S, int kt, int64_t col, int64_t V, int K,
                                int j) {
  if (!m || col >= V) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int k = 32 * (kt >> 1) + 8 * j + 4 * (kt & 1) + r;
    if (k < K) m[(int64_t)k * V + col] = S[r];
  }
}

// Decays of a chunk of C steps.  With G the sums of g from the chunk's start in
// units of log 2, formed in 64 bits: hi + lo = G_t in two parts, whose differences
// keep 24 bits where the decay between two steps counts, and u = e^(G_end - G_t),
// end being the last of the step's 32; w is the step's weight in the state, e^(G_last -
// G_t), or on the way back scale e^(G_t).  g below -200 counts as -200 (e^-200 is 0 in
// fp32, and sums stay finite).
template <int C>
struct Decays {
  float hi[C], lo[C], u[C], w[C];
};

__device__ inline float diff2(float hi, float lo, float hi0, float lo0) {
  return exp2_fast((hi - hi0) + (lo - lo0));
}

// Inclusive sums over the wave's lanes: row shifts within 16 lanes, then the rows'
// last lanes (scan_incl() of common.h, in 64 bits).
template <int CTRL, int ROWS>
__device__ inline double dpp_in64(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double wave_scan(double v) {
  v += dpp_in64<0x111, 0xf>(v);
  v += dpp_in64<0x112, 0xf>(v);
  v += dpp_in64<0x114, 0xf>(v);
  v += dpp_in64<0x118, 0xf>(v);
  v += dpp_in64<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_in64<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

// g of a lane's steps: steps lane E .. lane E + E - 1, E = max(C / 64, 1).
template <int C>
struct Gaps {
  static constexpr int E = C > 64 ? C / 64 : 1;
  float g[E];
  int rows;  // steps past these count as 0: when they are used, not here (a load whose
             // value is looked at in a branch is waited for in it)
  __device__ inline void load(const float* p, int64_t stride, int lane, int n) {
    rows = n;
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = p[lane * E + e < n ? (lane * E + e) * stride : 0];
  }
  // One wave forms a chunk's decays.
  template <bool REV = false>
  __device__ inline void decays(Decays<C>& d, int lane, float scale = 1.0f) const {
    double s[E], sum = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = lane * E + e < rows ? (g[e] < -200.0f ? -200.0f : g[e]) : 0.0f;
      sum += (double)x;
      s[e] = sum;
    }
    // of the lanes before (wave_shr:1): subtracting the lane's own would carry a later
    // step's NaN to an earlier one
    const double before = dpp_in64<0x138, 0xf>(wave_scan(sum));
    float hi[E], lo[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double G = (before + s[e]) * 1.4426950408889634;
      hi[e] = (float)G;
      lo[e] = (float)(G - (double)hi[e]);
    }
    constexpr int kBlock = 32 / E;  // lanes of 32 steps
    const int end = lane | (kBlock - 1);
    const float hE = __shfl(hi[E - 1], end), lE = __shfl(lo[E - 1], end);
    constexpr int kLast = C / E - 1;  // lane of the last step
    const float hL = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(hi[E - 1]), kLast));
    const float lL = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lo[E - 1]), kLast));
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int t = lane * E + e;
      if (t < C) {
        d.hi[t] = hi[e];
        d.lo[t] = lo[e];
        d.u[t] = diff2(hE, lE, hi[e], lo[e]);
        d.w[t] = REV ? scale * exp2_fast(hi[e] + lo[e]) : diff2(hL, lL, hi[e], lo[e]);
      }
    }
  }
};

// The planes of a piece of q, k or v.  (Pieces of whole vectors are zero past the row's
// end as they were read.)  Channels must not meet: take_plane() takes the planes of a
// pair together, where a value that is not finite would reach its neighbour.
template <typename T, bool VEC, int NP>
__device__ inline void planes_apart(const Piece<T, VEC, NP>& x, int lim, u32x4* out) {
  if constexpr (NP == 1 && VEC) {
    out[0] = x.w[0];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a = VEC || 2 * i < lim ? ldf(&x.e[2 * i]) : 0.0f;
      float b = VEC || 2 * i + 1 < lim ? ldf(&x.e[2 * i + 1]) : 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const uint32_t w = pk_bf16(a, b);
        out[n][i] = w;
        a -= __uint_as_float(w << 16);
        b -= __uint_as_float(w & 0xffff0000u);
      }
    }
  }
}

// Eight floats of a table in LDS, 8 j and up, for the 16 lanes of each j: a lane reads one
// of them and eight() hands them round, which takes LDS an eighth of the time that two
// 16-byte reads of every lane do (gradients 85 -> 84 us, and 8 to 16 registers less).
__device__ inline float one_of8(const float* table, int lane) {
  return table[8 * (lane >> 4) + (lane & 7)];
}
template <int E>
__device__ inline float row_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + E, 0xf, 0xf,
                                                    true));  // row_newbcast:E
}
__device__ inline void eight(float x, float* out) {
  out[0] = row_lane<0>(x);
  out[1] = row_lane<1>(x);
  out[2] = row_lane<2>(x);
  out[3] = row_lane<3>(x);
  out[4] = row_lane<4>(x);
  out[5] = row_lane<5>(x);
  out[6] = row_lane<6>(x);
  out[7] = row_lane<7>(x);
}

// The values of an operand's planes.
template <int NP>
__device__ inline void operand_values(const u32x4 (&f)[NP], float* x) {
#pragma unroll
  for (int p = NP - 1; p >= 0; --p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = __uint_as_float(f[p][e] << 16), b = __uint_as_float(f[p][e] & 0xffff0000u);
      x[2 * e] = p == NP - 1 ? a : x[2 * e] + a;
      x[2 * e + 1] = p == NP - 1 ? b : x[2 * e + 1] + b;
    }
}

}  // namespace
}  // namespace tssm
