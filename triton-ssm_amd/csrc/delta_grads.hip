// Gated delta rule, chunked: the gradients of the inputs, per chunk in parallel,
// from the state S before the chunk and the gradient G' of the state after it.
//
// With D[t][i] = e^(G_t - G_i), qk = Q K^T, kk = K K^T, A = beta D kk (i < t),
// P = D qk (i <= t), Y = V - e^G K S, R = beta Y, U = T R,
// dU = scale P^T dO + e^(G_last - G) K G', dR = T^T dU:
//   dV = beta dR,   dP = scale dO U^T,   dA = -dR U^T,
//   M = dP D (i <= t),   E = dA D beta (i < t),
//   X1 = scale dO S^T,   X2 = U G'^T,   X3 = dR S^T,
//   dQ = e^G X1 + M K,
//   dK = M^T Q + (E + E^T) K + e^(G_last - G) X2 - beta e^G X3,
//   dbeta = sum_v dR Y + sum_i dA D kk,
//   dG_t = e^G q.X1 - beta e^G k.X3 - b_t + sum_i F[t][i] - sum_i F[i][t],
//     F = dP P + dA A,  b_t = e^(G_last - G_t) k.X2,
//   dG_last += sum_t b_t + e^(G_last) <S, G'>,   dg_t = sum of dG from t on.
// A workgroup of four waves takes one chunk of one key head and goes through
// its value heads (whose gradients of q and k add up in registers, in order),
// and through V in slices of 64 columns: first column by column as the walks
// do (U, dR), then the sums over v, whose results are the tiles of 32 x K and
// 32 x 32 a wave keeps.  All products that reach dg and dbeta take three
// planes.
#include "delta_dev.h"

namespace tssm {
namespace {

struct GradArgs {
  DeltaArgs a;                // o: unused
  const void* dout;           // dO
  int64_t d_b, d_l, d_h;
  const ChunkWs* ws;
  const float *states, *grads;  // [bh][nch][Vp][KP]
  void *dq, *dk, *dv;         // contiguous
  float *dg, *dbeta;
  int nch;
};

template <typename T, int KP, bool VEC>
struct Grad {
  static constexpr int NP = Piece<T, VEC>::NP;
  static constexpr int NO = NP == 1 ? 2 : 3;  // planes of M and E: they reach dq and dk only
  static constexpr int NS = KP / 32, NK = NS < 2 ? 1 : NS / 2;  // tiles of 16 keys a wave keeps
  static constexpr int kLd = KP + 8, kVld = 64 + 8;
  static constexpr int kWaves = NP * KP <= 64 ? 2 : 1;
  struct Lds {
    uint16_t K[NP][kC * kLd], Q[NP][kC * kLd];
    uint16_t Tm[3][kC * kTld], PT[3][kC * kTld];  // T[t][i]; P[t][i] at [i][t]
    uint16_t D[NP][kC * kVld], V[NP][kC * kVld];
    union {
      struct {
        uint16_t U[3][64 * kTld], R[3][64 * kTld];  // of step t and column v at [v][t]
      } c;
      struct {
        uint16_t M[NO][kC * kTld], E[NO][kC * kTld];  // [i][t]
      } m;
    };
    float fac[kFac][kC];
    float row[4][5][kC];  // a wave's sums for each step: F, dA D kk, dR Y, q.X1 and k.X3, k.X2
    float col[4][kC];     // and of F over t
    float dot[4];
  };
};

// Four values of a column (rows t .. t + 3 of one [i][t] row) as planes.
template <int NP>
__device__ inline void put4(uint16_t (*m)[kC * kTld], int at, const f32x4& x) {
  float a = x[0], b = x[1], c = x[2], d = x[3];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const uint32_t lo = pk_bf16(a, b), hi = pk_bf16(c, d);
    *reinterpret_cast<u32x2v*>(&m[p][at]) = u32x2v{lo, hi};
    if (p + 1 < NP) {
      take_plane(lo, a, b);
      take_plane(hi, c, d);
    }
  }
}

template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(256, (Grad<T, KP, VEC>::kWaves)) void delta_grads_kernel(GradArgs g) {
  typedef Grad<T, KP, VEC> W;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, NK = W::NK;
  extern __shared__ __attribute__((aligned(16))) char raw[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(raw);
  const DeltaArgs& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, j = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), tx = w >> 1, ty = w & 1;
  const int ar = 8 * (c >> 2) + (c & 3);
  const int K = (int)a.K, per = (int)(a.Hv / a.Hk);
  const int64_t Vp = (a.V + 15) / 16 * 16;
  // the chunks of one head follow each other; heads go round the XCDs
  const int64_t n = blockIdx.x % g.nch, bk = blockIdx.x / g.nch, b = bk / a.Hk, hk = bk - b * a.Hk;
  const int64_t t0 = n * kC;
  const int rows = a.L - t0 < kC ? (int)(a.L - t0) : kC;

  {  // K and Q
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h + t0 * a.k_l;
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h + t0 * a.q_l;
#pragma unroll
    for (int i = 0; i < (kC * KP / 8 + 255) / 256; ++i) {
      const int id = tid + 256 * i, r = id / (KP / 8), col = id % (KP / 8) * 8;
      if (kC * KP / 8 % 256 && r >= kC) continue;
      const int lim = r < rows ? K - col : 0;
      Piece<T, VEC> x, y;
      x.load(kp + (r < rows ? r : 0) * a.k_l + (col < K ? col : 0), lim);
      y.load(qp + (r < rows ? r : 0) * a.q_l + (col < K ? col : 0), lim);
      u32x4 p[NP];
      x.planes(lim, p);
#pragma unroll
      for (int m = 0; m < NP; ++m) *reinterpret_cast<u32x4*>(&lds.K[m][r * W::kLd + col]) = p[m];
      y.planes(lim, p);
#pragma unroll
      for (int m = 0; m < NP; ++m) *reinterpret_cast<u32x4*>(&lds.Q[m][r * W::kLd + col]) = p[m];
    }
  }
  f32x4 aq[NK][2], ak[NK][2];  // dQ and dK, rows 8 j + 4 x + r, keys 32 s + 4 h + ar of tile (s, h)
#pragma unroll
  for (int m = 0; m < NK; ++m)
#pragma unroll
    for (int x = 0; x < 2; ++x) aq[m][x] = ak[m][x] = zero4();

  for (int hh = 0; hh < per; ++hh) {
    const int64_t h = hk * per + hh, bh = b * a.Hv + h, unit = bh * g.nch + n;
    const ChunkWs& cw = g.ws[unit];
    __syncthreads();
    for (int i = tid; i < 3 * kC * 4; i += 256)
      *reinterpret_cast<u32x4*>(&lds.Tm[i / 128][i % 128 / 4 * kTld + i % 4 * 8]) =
          *reinterpret_cast<const u32x4*>(&cw.T[i / 128][i % 128 / 4][i % 4 * 8]);
    (&lds.fac[0][0])[tid] = (&cw.fac[0][0])[tid];
    __syncthreads();
    float eg[8], be[8], en[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      eg[e] = lds.fac[kEg][8 * j + e];
      be[e] = lds.fac[kBeta][8 * j + e];
      en[e] = lds.fac[kEnd][8 * j + e];
    }
    // this wave's tile of D, P and D kk: rows t = 8 j + 4 tx + r, column i = ar + 4 ty
    f32x4 dd, pp = zero4(), dkk = zero4();
    const int ti = ar + 4 * ty;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      u32x4 fk[NP], fa[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fk[p] = lds16(&lds.K[p][ti * W::kLd + 32 * s + 8 * j]);
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fa[p] = lds16(&lds.Q[p][(ar + 4 * tx) * W::kLd + 32 * s + 8 * j]);
      pp = mfma_planes<NP, NP, 3>(fa, fk, pp);
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fa[p] = lds16(&lds.K[p][(ar + 4 * tx) * W::kLd + 32 * s + 8 * j]);
      dkk = mfma_planes<NP, NP, 3>(fa, fk, dkk);
    }
    {
      const float hi = lds.fac[kGhi][ti], lo = lds.fac[kGlo][ti];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 8 * j + 4 * tx + r;
        const float d = exp2_fast((lds.fac[kGhi][t] - hi) + (lds.fac[kGlo][t] - lo));
        dd[r] = ti <= t ? d : 0.0f;
        pp[r] = ti <= t ? d * pp[r] : 0.0f;
        dkk[r] = ti < t ? d * dkk[r] : 0.0f;
      }
      put4<3>(lds.PT, ti * kTld + 8 * j + 4 * tx, pp);
    }
    f32x4 X1[NK][2], X2[NK][2], X3[NK][2], dP = zero4(), dA = zero4();
    float db[8], ss = 0.0f;
#pragma unroll
    for (int m = 0; m < NK; ++m)
#pragma unroll
      for (int x = 0; x < 2; ++x) X1[m][x] = X2[m][x] = X3[m][x] = zero4();
#pragma unroll
    for (int e = 0; e < 8; ++e) db[e] = 0.0f;

    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + t0 * a.v_l;
    const T* dp = reinterpret_cast<const T*>(g.dout) + b * g.d_b + h * g.d_h + t0 * g.d_l;
    T* dvp = reinterpret_cast<T*>(g.dv) + ((b * a.L + t0) * a.Hv + h) * a.V;
    const float* Sp = g.states + unit * Vp * KP;
    const float* Gp = g.grads + unit * Vp * KP;
    for (int64_t v0 = 0; v0 < a.V; v0 += 64) {
      {
        const int r = tid / 8, col = tid % 8 * 8;
        const int64_t left = a.V - v0 - col;
        const int lim = r < rows ? (left < 0 ? 0 : (left < 8 ? (int)left : 8)) : 0;
        Piece<T, VEC> x, y;
        x.load(vp + (r < rows ? r : 0) * a.v_l + (left > 0 ? v0 + col : 0), lim);
        y.load(dp + (r < rows ? r : 0) * g.d_l + (left > 0 ? v0 + col : 0), lim);
        u32x4 p[NP];
        x.planes(lim, p);
#pragma unroll
        for (int m = 0; m < NP; ++m) *reinterpret_cast<u32x4*>(&lds.V[m][r * W::kVld + col]) = p[m];
        y.planes(lim, p);
#pragma unroll
        for (int m = 0; m < NP; ++m) *reinterpret_cast<u32x4*>(&lds.D[m][r * W::kVld + col]) = p[m];
      }
      __syncthreads();
      const int64_t vc = v0 + 16 * w + c;
      if (v0 + 16 * w < Vp) {
        f32x4 ks[2] = {zero4(), zero4()}, kg[2] = {zero4(), zero4()};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          f32x4 S[2], G[2];
          u32x4 sp[3], gp[3];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            S[x] = *reinterpret_cast<const f32x4*>(Sp + vc * KP + 32 * s + 8 * j + 4 * x);
            G[x] = *reinterpret_cast<const f32x4*>(Gp + vc * KP + 32 * s + 8 * j + 4 * x);
#pragma unroll
            for (int r = 0; r < 4; ++r) ss = __builtin_fmaf(S[x][r], G[x][r], ss);
          }
          split_tiles<3>(S[0], S[1], sp);
          split_tiles<3>(G[0], G[1], gp);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            u32x4 f[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p)
              f[p] = lds16(&lds.K[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
            ks[x] = mfma_planes<NP, 3, 3>(f, sp, ks[x]);
            kg[x] = mfma_planes<NP, 3, 3>(f, gp, kg[x]);
          }
        }
        float v[8];
        u32x4 dop[NP], pl[3];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int at = (8 * j + (c >> 2)) * W::kVld + 16 * w + 4 * (c & 3);
          const u32x2v v0_ = lds_tr(&lds.V[p][at]), v1_ = lds_tr(&lds.V[p][at + 4 * W::kVld]);
          const u32x2v d0_ = lds_tr(&lds.D[p][at]), d1_ = lds_tr(&lds.D[p][at + 4 * W::kVld]);
          dop[p] = u32x4{d0_[0], d0_[1], d1_[0], d1_[1]};
          const uint32_t u[4] = {v0_[0], v0_[1], v1_[0], v1_[1]};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t x = e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16;
            v[e] = p == 0 ? __uint_as_float(x) : v[e] + __uint_as_float(x);
          }
        }
        f32x4 R[2], U[2] = {zero4(), zero4()}, Z[2] = {zero4(), zero4()};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = __builtin_fmaf(-eg[e], ks[e >> 2][e & 3], v[e]);  // Y
          R[e >> 2][e & 3] = be[e] * v[e];
        }
        split_tiles<3>(R[0], R[1], pl);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 f[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) f[p] = lds16(&lds.Tm[p][(ar + 4 * x) * kTld + 8 * j]);
          U[x] = mfma_planes<3, 3, 3>(f, pl, U[x]);
#pragma unroll
          for (int p = 0; p < 3; ++p) f[p] = lds16(&lds.PT[p][(ar + 4 * x) * kTld + 8 * j]);
          Z[x] = mfma_planes<3, NP, 3>(f, dop, Z[x]);
        }
        split_tiles<3>(U[0], U[1], pl);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<u32x4*>(&lds.c.U[p][(16 * w + c) * kTld + 8 * j]) = pl[p];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          Z[e >> 2][e & 3] = __builtin_fmaf(en[e], kg[e >> 2][e & 3], a.scale * Z[e >> 2][e & 3]);
        split_tiles<3>(Z[0], Z[1], pl);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 f[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) f[p] = lds_col(lds.Tm[p], kTld, 4 * x, lane);
          R[x] = mfma_planes<3, 3, 3>(f, pl, zero4());  // dR
        }
        split_tiles<3>(R[0], R[1], pl);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<u32x4*>(&lds.c.R[p][(16 * w + c) * kTld + 8 * j]) = pl[p];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float r = R[e >> 2][e & 3];
          db[e] = __builtin_fmaf(r, v[e], db[e]);
          if (8 * j + e < rows && vc < a.V) stf(dvp + (8 * j + e) * a.Hv * a.V + vc, be[e] * r);
        }
      } else {
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          *reinterpret_cast<u32x4*>(&lds.c.U[p][(16 * w + c) * kTld + 8 * j]) = u32x4{0, 0, 0, 0};
          *reinterpret_cast<u32x4*>(&lds.c.R[p][(16 * w + c) * kTld + 8 * j]) = u32x4{0, 0, 0, 0};
        }
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (v0 + 32 * q >= Vp) continue;
        u32x4 fd[2][NP], fu[2][3], fr[2][3];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int p = 0; p < NP; ++p)
            fd[x][p] = lds16(&lds.D[p][(ar + 4 * x) * W::kVld + 32 * q + 8 * j]);
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            fu[x][p] = lds_col(&lds.c.U[p][32 * q * kTld], kTld, 4 * x, lane);
            fr[x][p] = lds_col(&lds.c.R[p][32 * q * kTld], kTld, 4 * x, lane);
          }
        }
        // (uniform selections: a register array has no runtime index)
        u32x4 da[NP], ra[3], ub[3];
#pragma unroll
        for (int p = 0; p < NP; ++p) da[p] = tx ? fd[1][p] : fd[0][p];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          ra[p] = tx ? fr[1][p] : fr[0][p];
          ub[p] = ty ? fu[1][p] : fu[0][p];
        }
        dP = mfma_planes<NP, 3, 3>(da, ub, dP);
        dA = mfma_planes<3, 3, 3>(ra, ub, dA);
#pragma unroll
        for (int m = 0; m < NK; ++m) {
          const int tile = w + 4 * m;
          if (tile >= 2 * NS) continue;
          const int key = 32 * (tile >> 1) + 4 * (tile & 1) + ar;
          float s8[8], g8[8];
          u32x4 sp[3], gp[3];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t r = v0 + 32 * q + 8 * j + e, rr = r < Vp ? r : Vp - 1;
            s8[e] = Sp[rr * KP + key];
            g8[e] = Gp[rr * KP + key];
          }
          split8<3>(s8, sp);
          split8<3>(g8, gp);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            X1[m][x] = mfma_planes<NP, 3, 3>(fd[x], sp, X1[m][x]);
            X2[m][x] = mfma_planes<3, 3, 3>(fu[x], gp, X2[m][x]);
            X3[m][x] = mfma_planes<3, 3, 3>(fr[x], sp, X3[m][x]);
          }
        }
      }
      __syncthreads();
    }

    // the 32 x 32 tiles: M, E and the sums of F
    {
      f32x4 M, E;
      float fcol = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 8 * j + 4 * tx + r;
        const float bt = lds.fac[kBeta][t];
        const float p = a.scale * dP[r], q = -dA[r];
        M[r] = p * dd[r];
        E[r] = ti < t ? q * dd[r] * bt : 0.0f;
        const float f = __builtin_fmaf(p, pp[r], q * bt * dkk[r]);
        fcol += f;
        const float frow = group_sum<16>(f), kb = group_sum<16>(q * dkk[r]);
        if (c == 0) {
          lds.row[w][0][t] = frow;
          lds.row[w][1][t] = kb;
        }
      }
      fcol += __shfl_xor(fcol, 16);
      fcol += __shfl_xor(fcol, 32);
      if (j == 0) lds.col[w][ti] = fcol;
      put4<NO>(lds.m.M, ti * kTld + 8 * j + 4 * tx, M);
      put4<NO>(lds.m.E, ti * kTld + 8 * j + 4 * tx, E);
    }
    // products with q and k over the keys, step by step
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 8 * j + e;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int m = 0; m < NK; ++m) {
        const int tile = w + 4 * m;
        if (tile >= 2 * NS) continue;
        const int at = t * W::kLd + 32 * (tile >> 1) + 4 * (tile & 1) + ar;
        float kv = 0.0f, qv = 0.0f;
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {
          kv += bf16_bits_to_f32(lds.K[p][at]);
          qv += bf16_bits_to_f32(lds.Q[p][at]);
        }
        s1 += a.scale * qv * X1[m][e >> 2][e & 3] - be[e] * kv * X3[m][e >> 2][e & 3];
        s2 = __builtin_fmaf(kv, X2[m][e >> 2][e & 3], s2);
      }
      s1 = group_sum<16>(s1);
      s2 = group_sum<16>(s2);
      const float s3 = group_sum<16>(db[e]);
      if (c == 0) {
        lds.row[w][2][t] = s3;
        lds.row[w][3][t] = eg[e] * s1;
        lds.row[w][4][t] = en[e] * s2;
      }
    }
    ss = group_sum<64>(ss);
    if (lane == 0) lds.dot[w] = ss;
    __syncthreads();
    if (w == 0) {
      const int t = lane & 31, x = t >> 2 & 1;  // the tiles of row t: waves 2 x, 2 x + 1
      const auto sum4 = [&](int i) {
        return (lds.row[0][i][t] + lds.row[1][i][t]) + (lds.row[2][i][t] + lds.row[3][i][t]);
      };
      const float f = lds.row[2 * x][0][t] + lds.row[2 * x + 1][0][t];
      const float kb = lds.row[2 * x][1][t] + lds.row[2 * x + 1][1][t];
      const float fc = lds.col[x][t] + lds.col[2 + x][t];  // column t: waves x and 2 + x
      const float bt = sum4(4);
      double G = (double)(f - fc) + (double)(sum4(3) - bt), B = bt;
#pragma unroll
      for (int s = 1; s < 32; s *= 2) B += __shfl_xor(B, s, 32);
      if (t == 31)
        G += B + (double)lds.fac[kEg][31] *
                     (double)((lds.dot[0] + lds.dot[1]) + (lds.dot[2] + lds.dot[3]));
#pragma unroll
      for (int s = 1; s < 32; s *= 2) {
        const double y = __shfl_down(G, s, 32);
        if (t + s < 32) G += y;
      }
      if (lane < rows) {
        const int64_t at = (b * a.L + t0 + t) * a.Hv + h;
        g.dg[at] = (float)G;
        g.dbeta[at] = sum4(2) + kb;
      }
    }
#pragma unroll
    for (int m = 0; m < NK; ++m) {
      const int tile = w + 4 * m;
      if (tile >= 2 * NS) continue;
      const int at = 32 * (tile >> 1) + 4 * (tile & 1);
      u32x4 kc[NP], qc[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kc[p] = lds_col(lds.K[p], W::kLd, at, lane);
        qc[p] = lds_col(lds.Q[p], W::kLd, at, lane);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 4 * x + r;
          aq[m][x][r] = __builtin_fmaf(a.scale * eg[e], X1[m][x][r], aq[m][x][r]);
          ak[m][x][r] += en[e] * X2[m][x][r] - be[e] * eg[e] * X3[m][x][r];
        }
        u32x4 f[NO];
#pragma unroll
        for (int p = 0; p < NO; ++p) f[p] = lds_col(lds.m.M[p], kTld, 4 * x, lane);
        aq[m][x] = mfma_planes<NO, NP, NO>(f, kc, aq[m][x]);
#pragma unroll
        for (int p = 0; p < NO; ++p) f[p] = lds16(&lds.m.M[p][(ar + 4 * x) * kTld + 8 * j]);
        ak[m][x] = mfma_planes<NO, NP, NO>(f, qc, ak[m][x]);
#pragma unroll
        for (int p = 0; p < NO; ++p) f[p] = lds_col(lds.m.E[p], kTld, 4 * x, lane);
        ak[m][x] = mfma_planes<NO, NP, NO>(f, kc, ak[m][x]);
#pragma unroll
        for (int p = 0; p < NO; ++p) f[p] = lds16(&lds.m.E[p][(ar + 4 * x) * kTld + 8 * j]);
        ak[m][x] = mfma_planes<NO, NP, NO>(f, kc, ak[m][x]);
      }
    }
  }
  T* dqp = reinterpret_cast<T*>(g.dq) + ((b * a.L + t0) * a.Hk + hk) * K;
  T* dkp = reinterpret_cast<T*>(g.dk) + ((b * a.L + t0) * a.Hk + hk) * K;
#pragma unroll
  for (int m = 0; m < NK; ++m) {
    const int tile = w + 4 * m, key = 32 * (tile >> 1) + 4 * (tile & 1) + ar;
    if (tile >= 2 * NS || key >= K) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 8 * j + e;
      if (t < rows) {
        stf(dqp + t * a.Hk * K + key, aq[m][e >> 2][e & 3]);
        stf(dkp + t * a.Hk * K + key, ak[m][e >> 2][e & 3]);
      }
    }
  }
}

template <typename T, int KP>
int grads_launch(const GradArgs& g, bool vec, hipStream_t s) {
  const int64_t wgs = g.a.B * g.a.Hk * g.nch;
  const auto go = [&](auto* f, int bytes) {
    if (bytes > 64 * 1024) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != hipSuccess) return (int)e;
    }
    f<<<(unsigned)wgs, 256, bytes, s>>>(g);
    return launch_status();
  };
  static_assert(sizeof(typename Grad<T, KP, true>::Lds) <= 160 * 1024, "LDS of a CU");
  return vec ? go(delta_grads_kernel<T, KP, true>, (int)sizeof(typename Grad<T, KP, true>::Lds))
             : go(delta_grads_kernel<T, KP, false>, (int)sizeof(typename Grad<T, KP, false>::Lds));
}

template <typename T>
int grads(const GradArgs& g, bool vec, hipStream_t s) {
  if (g.a.K <= 32) return grads_launch<T, 32>(g, vec, s);
  if (g.a.K <= 64) return grads_launch<T, 64>(g, vec, s);
  return grads_launch<T, 128>(g, vec, s);
}

}  // namespace

int delta_grads_launch(int dtype, const DeltaArgs& a, const DeltaGrads& d, bool vec,
                       const DeltaPlan& p, hipStream_t s) {
  const GradArgs g = {a, d.dout, d.d_b, d.d_l, d.d_h, reinterpret_cast<const ChunkWs*>(p.chunks),
                      p.states, p.grads, d.dq, d.dk, d.dv, d.dg, d.dbeta, p.nch};
  switch (dtype) {
    case TSSM_F32: return grads<float>(g, vec, s);
    case TSSM_BF16: return grads<bf16_t>(g, vec, s);
    default: return grads<f16_t>(g, vec, s);
  }
}

}  // namespace tssm
