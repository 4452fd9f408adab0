// Gated delta rule, chunked: the walk over the chunks.
//
// Per chunk of 32 steps, with S the state before it and T, P, G from the
// preparing pass:
//   R = beta (V - e^G K S),  U = T R,  O = scale e^G Q S + P U,
//   S' = e^(G_last) S + K^T (e^(G_last - G) U).
// Columns of V never meet, so a wave owns 16 of them: S^T's columns stay in its
// registers for the whole sequence and every product's result is the next
// one's B operand in place (delta_dev.h).  The A operands K, Q, T and P come
// through LDS, shared by the waves of a workgroup and double-buffered: the
// next chunk's loads are in flight while this one is multiplied.
//
// A chunk whose U is not finite is done again step by step from S: zero
// weights would otherwise carry a later step's NaN to earlier outputs.
#include "delta_dev.h"

namespace tssm {
namespace {

template <typename T, int KP, bool VEC, int NPP, int NW>
struct Walk {
  static constexpr int NT = 64 * NW, NP = Piece<T, VEC>::NP;
  static constexpr int kLd = KP + 8;               // bf16 elements of a row of K or Q in LDS
  static constexpr int kPieces = kC * KP / 8;      // 8-element pieces of K
  static constexpr int kNk = (kPieces + NT - 1) / NT;
  static constexpr int kTp = (3 + NPP) * kC * kC / 8;  // 16-byte pieces of T and P
  static constexpr int kNt = (kTp + NT - 1) / NT;
  struct Buf {
    uint16_t K[NP][kC * kLd], Q[NP][kC * kLd], M[3 + NPP][kC * kTld];  // M: T, then P
    float fac[4][kC];
  };
  Piece<T, VEC> rk[kNk], rq[kNk];
  u32x4 rt[kNt];
  float rf;

  __device__ inline void load(const DeltaArgs& a, const T* kp, const T* qp,
                              const ChunkWs<NPP>* ws, int64_t n) {
    const int64_t t0 = n * kC;
    const int rows = a.L - t0 < kC ? (int)(a.L - t0) : kC;
#pragma unroll
    for (int i = 0; i < kNk; ++i) {
      const int id = threadIdx.x + NT * i, r0 = id / (KP / 8) % kC, col = id % (KP / 8) * 8;
      const int r = r0 < rows ? r0 : 0, cc = col < a.K ? col : 0;
      rk[i].load(kp + (t0 + r) * a.k_l + cc, (int)a.K - col);
      rq[i].load(qp + (t0 + r) * a.q_l + cc, (int)a.K - col);
    }
    const u32x4* tp = reinterpret_cast<const u32x4*>(ws + n);  // T and P are adjacent
#pragma unroll
    for (int i = 0; i < kNt; ++i) {
      const int id = threadIdx.x + NT * i;
      rt[i] = tp[id < kTp ? id : 0];
    }
    rf = (&ws[n].fac[0][0])[threadIdx.x & 127];
  }
  __device__ inline void store(const DeltaArgs& a, Buf& b, int64_t n) const {
    const int64_t t0 = n * kC;
    const int rows = a.L - t0 < kC ? (int)(a.L - t0) : kC;
#pragma unroll
    for (int i = 0; i < kNk; ++i) {
      const int id = threadIdx.x + NT * i, r = id / (KP / 8), col = id % (KP / 8) * 8;
      if (kPieces % NT && id >= kPieces) continue;
      const int lim = r < rows ? (int)a.K - col : 0;
      u32x4 p[NP];
      rk[i].planes(lim, p);
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&b.K[x][r * kLd + col]) = p[x];
      rq[i].planes(lim, p);
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&b.Q[x][r * kLd + col]) = p[x];
    }
#pragma unroll
    for (int i = 0; i < kNt; ++i) {
      const int id = threadIdx.x + NT * i;
      if (kTp % NT && id >= kTp) continue;
      const int r = id / (kC / 8), col = id % (kC / 8) * 8;  // r: row of all planes
      *reinterpret_cast<u32x4*>(&b.M[r / kC][r % kC * kTld + col]) = rt[i];
    }
    if (threadIdx.x < 128) (&b.fac[0][0])[threadIdx.x] = rf;
  }
};

template <typename T, int KP, bool VEC, int NPP, int NW>
__global__ __launch_bounds__(64 * NW) void delta_walk_kernel(DeltaArgs a, const ChunkWs<NPP>* ws,
                                                             int64_t nch, uint32_t nvb) {
  typedef Walk<T, KP, VEC, NPP, NW> W;
  constexpr int NP = W::NP, NS = KP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  typename W::Buf* buf = reinterpret_cast<typename W::Buf*>(lds);
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t bh = blockIdx.x / nvb, b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int64_t vw = ((blockIdx.x - bh * nvb) * NW + wv) * 16, vc = vw + c;
  const bool act = vw < a.V, on = vc < a.V;  // the wave, the lane has columns
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h;
  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h;
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + (on ? vc : 0);
  T* op = reinterpret_cast<T*>(a.o) + b * a.o_b + h * a.o_h + vc;
  const ChunkWs<NPP>* cw = ws + bh * nch;

  // S[k][c], k = 32 s + 8 j + 4 x + r, in tile 2 s + x register r
  f32x4 S[2 * NS];
  const int64_t sbase = bh * a.K * a.V + vc;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
      S[i][r] = a.h0 && on && k < a.K ? a.h0[sbase + (int64_t)k * a.V] : 0.0f;
    }

  W w;
  float nv[8], v[8];
  auto fetch_v = [&](int64_t n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t t = n * kC + 8 * j + e;
      nv[e] = ldf(vp + (t < a.L ? t : 0) * a.v_l);
    }
  };
  w.load(a, kp, qp, cw, 0);
  if (act) fetch_v(0);
  w.store(a, buf[0], 0);
  __syncthreads();
  for (int64_t n = 0; n < nch; ++n) {
    const typename W::Buf& B = buf[n & 1];
    const int rows = a.L - n * kC < kC ? (int)(a.L - n * kC) : kC;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 8 * j + e < rows && on ? nv[e] : 0.0f;
    if (n + 1 < nch) {
      w.load(a, kp, qp, cw, n + 1);
      if (act) fetch_v(n + 1);
    }
    if (act) {
      float eg[8], be[8], en[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        *reinterpret_cast<float4*>(eg + 4 * q) =
            *reinterpret_cast<const float4*>(&B.fac[0][8 * j + 4 * q]);
        *reinterpret_cast<float4*>(be + 4 * q) =
            *reinterpret_cast<const float4*>(&B.fac[1][8 * j + 4 * q]);
        *reinterpret_cast<float4*>(en + 4 * q) =
            *reinterpret_cast<const float4*>(&B.fac[2][8 * j + 4 * q]);
      }
      const float last = B.fac[0][kC - 1];
      // row of tile x that this lane holds of an A operand
      const int ar = 8 * (c >> 2) + (c & 3);
      f32x4 ks[2] = {zero4(), zero4()}, qs[2] = {zero4(), zero4()};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        u32x4 sp[3], f[NP];
        split_tiles<3>(S[2 * s], S[2 * s + 1], sp);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int at = (ar + 4 * x) * W::kLd + 32 * s + 8 * j;
#pragma unroll
          for (int p = 0; p < NP; ++p) f[p] = lds16(&B.K[p][at]);
          ks[x] = mfma_planes<NP, 3, 3>(f, sp, ks[x]);
#pragma unroll
          for (int p = 0; p < NP; ++p) f[p] = lds16(&B.Q[p][at]);
          qs[x] = mfma_planes<NP, 3, NPP>(f, sp, qs[x]);
        }
      }
      f32x4 R[2], U[2] = {zero4(), zero4()};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 4 * x + r;
          R[x][r] = be[e] * __builtin_fmaf(-eg[e], ks[x][r], v[e]);
          qs[x][r] *= eg[e] * a.scale;
        }
      u32x4 rp[3];
      split_tiles<3>(R[0], R[1], rp);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4 f[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) f[p] = lds16(&B.M[p][(ar + 4 * x) * kTld + 8 * j]);
        U[x] = mfma_planes<3, 3, 3>(f, rp, U[x]);
      }
      float big = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) big += __builtin_fabsf(U[e >> 2][e & 3]);
      if (__builtin_expect(__ballot(!(big < __builtin_inff())) == 0, 1)) {
        u32x4 up[NPP];
        split_tiles<NPP>(U[0], U[1], up);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 f[NPP];
#pragma unroll
          for (int p = 0; p < NPP; ++p) f[p] = lds16(&B.M[3 + p][(ar + 4 * x) * kTld + 8 * j]);
          qs[x] = mfma_planes<NPP, NPP, NPP>(f, up, qs[x]);
        }
        f32x4 E[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) E[e >> 2][e & 3] = en[e] * U[e >> 2][e & 3];
        u32x4 ep[3];
        split_tiles<3>(E[0], E[1], ep);
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) {
          u32x4 f[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p)
            f[p] = lds_col(B.K[p], W::kLd, 32 * (i >> 1) + 4 * (i & 1), lane);
#pragma unroll
          for (int r = 0; r < 4; ++r) S[i][r] *= last;
          S[i] = mfma_planes<NP, 3, 3>(f, ep, S[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (on && 8 * j + e < rows) stf(op + (n * kC + 8 * j + e) * a.o_l, qs[e >> 2][e & 3]);
      } else {
        for (int t = 0; t < rows; ++t) {
          const float al = exp_acc(B.fac[3][t]), bt = B.fac[1][t];
          const float vt = on ? ldf(vp + (n * kC + t) * a.v_l) : 0.0f;
          auto row = [&](const uint16_t (&m)[NP][kC * W::kLd], int i, int r) {
            const int at = t * W::kLd + 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
            float x = 0.0f;
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) x += bf16_bits_to_f32(m[p][at]);
            return x;
          };
          float s = 0.0f, y = 0.0f;
#pragma unroll
          for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              S[i][r] *= al;
              s = __builtin_fmaf(row(B.K, i, r), S[i][r], s);
            }
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
          const float u = bt * (vt - s);
#pragma unroll
          for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              S[i][r] = __builtin_fmaf(row(B.K, i, r), u, S[i][r]);
              y = __builtin_fmaf(row(B.Q, i, r), S[i][r], y);
            }
          y += __shfl_xor(y, 16);
          y += __shfl_xor(y, 32);
          if (on && j == 0) stf(op + (n * kC + t) * a.o_l, a.scale * y);
        }
      }
    }
    if (n + 1 < nch) w.store(a, buf[(n + 1) & 1], n + 1);
    __syncthreads();
  }
  if (!a.h_last || !on) return;
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
      if (k < a.K) a.h_last[sbase + (int64_t)k * a.V] = S[i][r];
    }
}

template <typename T, int KP, bool VEC, int NPP, int NW>
int launch(const DeltaArgs& a, const void* ws, hipStream_t s) {
  typedef Walk<T, KP, VEC, NPP, NW> W;
  const int64_t nvb = cdiv64(a.V, 16 * NW), wgs = a.B * a.Hv * nvb;
  if (wgs > 0x7fffffff) return TSSM_ERR_UNSUPPORTED;
  constexpr int bytes = 2 * (int)sizeof(typename W::Buf);
  static_assert(bytes <= 160 * 1024, "two chunks in LDS");
  auto* f = delta_walk_kernel<T, KP, VEC, NPP, NW>;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return (int)e;
  }
  f<<<(unsigned)wgs, 64 * NW, bytes, s>>>(a, reinterpret_cast<const ChunkWs<NPP>*>(ws),
                                          cdiv64(a.L, kC), (uint32_t)nvb);
  return launch_status();
}

template <typename T, int NPP>
int walk(const DeltaArgs& a, bool vec, const void* ws, hipStream_t s) {
  if (a.K <= 32)
    return vec ? launch<T, 32, true, NPP, 4>(a, ws, s) : launch<T, 32, false, NPP, 4>(a, ws, s);
  if (a.K <= 64)
    return vec ? launch<T, 64, true, NPP, 4>(a, ws, s) : launch<T, 64, false, NPP, 4>(a, ws, s);
  return vec ? launch<T, 128, true, NPP, 4>(a, ws, s) : launch<T, 128, false, NPP, 4>(a, ws, s);
}

}  // namespace

int delta_walk_launch(int dtype, const DeltaArgs& a, bool vec, const void* ws, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return walk<float, 3>(a, vec, ws, s);
    case TSSM_BF16: return walk<bf16_t, 2>(a, vec, ws, s);
    default: return walk<f16_t, 3>(a, vec, ws, s);
  }
}

int64_t delta_chunk_ws_bytes(int dtype) {
  return dtype == TSSM_BF16 ? (int64_t)sizeof(ChunkWs<2>) : (int64_t)sizeof(ChunkWs<3>);
}

}  // namespace tssm
