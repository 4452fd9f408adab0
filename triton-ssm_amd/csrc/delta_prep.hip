// Gated delta rule, preparing pass: per chunk of 32 steps and value head, what
// the walks need of the keys, decays and step sizes alone.
//
// With G the running sums of g within the chunk:
//   A[t][i] = beta_t e^(G_t - G_i) k_t.k_i (i < t),   T = (I + A)^-1.
// One wave per chunk and head.  The Gram product runs on the matrix cores (3
// of the 4 tiles of 16 x 16).  T's diagonal blocks come from forward
// substitution (a lane per column: stable where keys repeat, unlike products
// of powers of A), the block below from -T22 A21 T11 in fp32.  G is summed in
// 64 bits: its differences are what counts, and a reset may put -6400 before a
// slow step; a decay below e^-200 is 0 in fp32 either way.
//
// Bound by memory: 4 KiB of keys and 0.25 of g and beta in, 5.25 out a chunk (B=8
// L=4096 H=16 K=64 bf16: 172 MB in 34 to 36 us, 5 TB/s; 43 us with T's zeros stored
// and 16 bytes of every 32 written at a time).  T in fp32 would be less to write
// (36 us with its zeros), but the walks' loaders then split it into planes, and
// the chain waves on their SIMDs lose more to that than is gained here.
#include "delta_dev.h"

namespace tssm {
namespace {

constexpr int kLd = 36;  // floats of a row of A or T in LDS

__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// T into planes, a KiB of one after the other at a time.
__device__ inline void put_planes(const float* m, ChunkWs& out, int lane) {
  auto put = [&](int row, int col, auto dst) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(m + row * kLd + col + 4 * q);
      v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
    }
    u32x4 p[3];
    split8<3>(v, p);
#pragma unroll
    for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x4*>(dst(n)) = p[n];
  };
  const int r4 = lane >> 2, c4 = 8 * (lane & 3), r2 = lane >> 1, c2 = 8 * (lane & 1);
  put(16 + r4, c4, [&](int n) { return &out.T[n].below[r4][c4]; });
  if (lane < 32) put(r2, c2, [&](int n) { return &out.T[n].first[r2][c2]; });
}

template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(256) void delta_prep_kernel(DeltaArgs a, ChunkWs* ws, uint32_t nch,
                                                         uint32_t units) {
  constexpr int NP = Piece<T, VEC>::NP;
  __shared__ __attribute__((aligned(16))) float mat[4][2][kC * kLd];
  __shared__ __attribute__((aligned(16))) float sums[4][2][kC], bet[4][kC];  // G log2(e) in two parts, beta
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t unit = block_of() * 4 + wv;
  if (unit >= units) return;
  // units run over the value heads of one chunk first: a group shares its keys
  const uint32_t Hv = (uint32_t)a.Hv, bn = unit / Hv, nth = bn / nch;
  const int64_t n = bn - nth * nch, t0 = n * kC;
  const auto [b, h, hk] = head_of(a, nth * Hv + (unit - bn * Hv));
  const int rows = a.L - t0 < kC ? (int)(a.L - t0) : kC;
  ChunkWs& out = ws[(b * a.Hv + h) * nch + n];
  float *mA = mat[wv][0], *mT = mat[wv][1];

  // running sums of g, per step
  const int t = lane & 31;
  const bool on = t < rows;
  const int64_t tt = t0 + (on ? t : 0);
  const float g0 = a.g[b * a.g_b + tt * a.g_l + h * a.g_h];
  const float b0 = a.beta[b * a.be_b + tt * a.be_l + h * a.be_h];
  const float g = on ? (g0 < -200.0f ? -200.0f : g0) : 0.0f, beta = on ? b0 : 0.0f;
  double G = g;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    const double up = __shfl_up(G, s, 32);
    if (t >= s) G += up;
  }
  const double Gl = __shfl(G, 31, 32);
  if (lane < kC) {
    const double log2e = 1.4426950408889634074, G2 = G * log2e;
    const float hi = (float)G2, lo = (float)(G2 - (double)hi);
    sums[wv][0][t] = hi;
    sums[wv][1][t] = lo;
    bet[wv][t] = beta;
    out.fac[kEg][t] = exp2_fast(hi);
    out.fac[kBeta][t] = beta;
    out.fac[kEnd][t] = exp2_fast((float)((Gl - G) * log2e));
    out.fac[kG][t] = on ? g0 : 0.0f;
    out.fac[kGhi][t] = hi;
    out.fac[kGlo][t] = lo;
  }

  // Gram product: tiles (0,0), (1,0), (1,1)
  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_b + t0 * a.k_l + hk * a.k_h;
  f32x4 kk[3] = {zero4(), zero4(), zero4()};
  Piece<T, VEC> pk[2];
#pragma unroll
  for (int s = 0; s < KP / 32; ++s) {
    const int col = 32 * s + 8 * j, clim = (int)a.K - col;
    u32x4 fk[2][NP];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 16 * x + c, lim = r < rows ? clim : 0;
      const int64_t kr = (r < rows ? r : 0) * a.k_l + (clim > 0 ? col : 0);
      pk[x].load(kb + kr, lim);
      pk[x].planes(lim, fk[x]);
    }
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      const int ro = x > 0, co = x > 1;
      kk[x] = mfma_planes<NP, NP, 3>(fk[ro], fk[co], kk[x]);
    }
  }
  wave_order();
#pragma unroll
  for (int x = 0; x < 3; ++x) {
    const int i = 16 * (x > 1) + c;
    const float hi = sums[wv][0][i], lo = sums[wv][1][i];
    const int at = 16 * (x > 0) + 4 * j;
    const float4 h4 = *reinterpret_cast<const float4*>(&sums[wv][0][at]);
    const float4 l4 = *reinterpret_cast<const float4*>(&sums[wv][1][at]);
    const float4 b4 = *reinterpret_cast<const float4*>(&bet[wv][at]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float d = exp2_fast(((&h4.x)[r] - hi) + ((&l4.x)[r] - lo));
      mA[(at + r) * kLd + i] = i < at + r ? (&b4.x)[r] * d * kk[x][r] : 0.0f;
    }
  }
  wave_order();
  // diagonal blocks: lane (d, c) solves for column c of block d
  {
    const int d = (lane >> 4) & 1;
    const float* A = mA + 16 * d * kLd + 16 * d;
    float X[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float row[16];
#pragma unroll
      for (int q = 0; q < (i + 3) / 4; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(A + i * kLd + 4 * q);
        row[4 * q] = f.x; row[4 * q + 1] = f.y; row[4 * q + 2] = f.z; row[4 * q + 3] = f.w;
      }
      float s0 = i == c ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
      for (int m = 0; m < i; ++m) {
        if (m & 1) s1 = __builtin_fmaf(-row[m], X[m], s1);
        else s0 = __builtin_fmaf(-row[m], X[m], s0);
      }
      X[i] = s0 + s1;
    }
    if (lane < kC) {
#pragma unroll
      for (int i = 0; i < 16; ++i) mT[(16 * d + i) * kLd + 16 * d + c] = X[i];
    }
  }
  wave_order();
  {
    f32x4 x = zero4(), y = zero4();
#pragma unroll
    for (int m = 0; m < 4; ++m)
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(mA[(16 + c) * kLd + 4 * m + j],
                                               mT[(4 * m + j) * kLd + c], x, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      y = __builtin_amdgcn_mfma_f32_16x16x4f32(mT[(16 + c) * kLd + 16 + 4 * j + r], x[r], y, 0, 0,
                                               0);
#pragma unroll
    for (int r = 0; r < 4; ++r) mT[(16 + 4 * j + r) * kLd + c] = -y[r];
  }
  wave_order();
  put_planes(mT, out, lane);
}

template <typename T, int KP>
void launch(const DeltaArgs& a, bool vec, ChunkWs* ws, hipStream_t s) {
  const int64_t nch = cdiv64(a.L, kC), units = a.B * a.Hv * nch;
  const dim3 wgs = grid_of(cdiv64(units, 4));
  if (vec) delta_prep_kernel<T, KP, true><<<wgs, 256, 0, s>>>(a, ws, (uint32_t)nch, (uint32_t)units);
  else delta_prep_kernel<T, KP, false><<<wgs, 256, 0, s>>>(a, ws, (uint32_t)nch, (uint32_t)units);
}

template <typename T>
void prep(const DeltaArgs& a, bool vec, ChunkWs* ws, hipStream_t s) {
  if (a.K <= 32) launch<T, 32>(a, vec, ws, s);
  else if (a.K <= 64) launch<T, 64>(a, vec, ws, s);
  else launch<T, 128>(a, vec, ws, s);
}

}  // namespace

int delta_prep_launch(int dtype, const DeltaArgs& a, bool vec, void* workspace, hipStream_t s) {
  ChunkWs* ws = reinterpret_cast<ChunkWs*>(workspace);
  switch (dtype) {
    case TSSM_F32: prep<float>(a, vec, ws, s); break;
    case TSSM_BF16: prep<bf16_t>(a, vec, ws, s); break;
    default: prep<f16_t>(a, vec, ws, s); break;
  }
  return launch_status();
}

}  // namespace tssm
