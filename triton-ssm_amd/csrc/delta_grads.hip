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
//   dg_t = sum over s >= t of e^(G_s) sum_v (scale dO (Q S) - beta dR (K S))
//          + sum over s >= t > i of F[s][i] + sum over i < t of b_i + e^(G_last) <S, G'>,
//     F = dP P + dA A,  b_i = e^(G_last - G_i) sum_v U (K G').
// (Nothing but terms that hold e^(g_t): sums of F's rows less those of its columns, rounded
// to fp32, leave 1e-6 of the chunk's largest dg where a strong decay among slow ones makes
// it 1e-13.)
// A workgroup of four waves takes one chunk of one key head and goes through
// its value heads (whose gradients of q and k add up in registers, in order),
// and through V in slices of 64 columns: first column by column as the walks
// do (U, dR), then the sums over v, whose results are the tiles of 32 x K and
// 32 x 32 a wave keeps.  Products that reach dg and dbeta take three planes, X1
// to X3, M and E as many as dq and dk need (two for bf16).
//
// B=4 L=4096 H=16 K=V=64 bf16: 160 us for 450 MB in (268 of them S and G') and 107
// out, which would take 108 at a copy's rate; the rest is a chunk's phases, each
// waiting for the one before at the workgroup's barriers, of which two workgroups
// a CU (LDS) overlap.
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
  // planes where dq and dk alone are reached (0.26% of their bf16 are the one next
  // to the nearest; with three 0.02%, and 10 us more of the 160 above)
  static constexpr int NO = NP == 1 ? 2 : 3;
  static constexpr int NS = KP / 32, NK = NS < 2 ? 1 : NS / 2;  // tiles of 16 keys a wave keeps
  static constexpr int kLd = KP + 8, kVld = 64 + 8;
  // two workgroups a CU where LDS holds both
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
    // a wave's sums for each step: F, dA D kk, dR Y, e^G (scale dO (Q S) - beta dR (K S)),
    // e^(G_last - G) U (K G')
    float row[4][5][kC];
    float col[8][kC];     // and of F's columns, over four rows each
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

// ONE: one value head to a key head, and V in one slice.
template <typename T, int KP, bool VEC, bool ONE>
__global__ __launch_bounds__(256, (Grad<T, KP, VEC>::kWaves)) void delta_grads_kernel(GradArgs g) {
  typedef Grad<T, KP, VEC> W;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, NK = W::NK;
  constexpr int kNk = (kC * KP / 8 + 255) / 256;  // pieces of K a thread brings
  extern __shared__ __attribute__((aligned(16))) char raw[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(raw);
  const DeltaArgs& a = g.a;
  const int tid = threadIdx.x, lane = tid & 63, j = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), tx = w >> 1, ty = w & 1;
  const uint32_t heads = (uint32_t)a.Hk;  // of the keys
  const int K = (int)a.K, per = ONE ? 1 : (int)((uint32_t)a.Hv / heads);
  const int64_t Vp = (a.V + 15) / 16 * 16;
  // the chunks of one head follow each other
  const uint32_t block = block_of(), bk = block / (uint32_t)g.nch;
  const int64_t n = block - bk * (uint32_t)g.nch, b = bk / heads, hk = bk % heads;
  if (b >= a.B) return;
  const int64_t t0 = n * kC;
  const int rows = a.L - t0 < kC ? (int)(a.L - t0) : kC;

  // K and Q on their way; they go to LDS with the first head's operands
  Piece<T, VEC> pk[kNk], pq[kNk];
  {
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h + t0 * a.k_l;
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h + t0 * a.q_l;
#pragma unroll
    for (int i = 0; i < kNk; ++i) {
      const int id = tid + 256 * i, r = id / (KP / 8), col = id % (KP / 8) * 8;
      const int lim = r < rows ? K - col : 0;
      pk[i].load(kp + (r < rows ? r : 0) * a.k_l + (col < K ? col : 0), lim);
      pq[i].load(qp + (r < rows ? r : 0) * a.q_l + (col < K ? col : 0), lim);
    }
  }
  f32x4 aq[NK][2], ak[NK][2];  // dQ and dK, rows 8 j + 4 x + r, keys 16 (w + 4 m) + c
#pragma unroll
  for (int m = 0; m < NK; ++m)
#pragma unroll
    for (int x = 0; x < 2; ++x) aq[m][x] = ak[m][x] = zero4();

  for (int hh = 0; hh < per; ++hh) {
    const int64_t h = hk * per + hh, bh = b * a.Hv + h, unit = bh * g.nch + n;
    // the thread's place anew for each head: addresses that follow from it
    // would otherwise be kept in registers across the loop, more than there are
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, j = lane >> 4, c = lane & 15, ar = 8 * (c >> 2) + (c & 3);
    const int ti = ar + 4 * ty;  // the column i of this wave's 32 x 32 tile
    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + t0 * a.v_l;
    const T* dp = reinterpret_cast<const T*>(g.dout) + b * g.d_b + h * g.d_h + t0 * g.d_l;
    T* dvp = reinterpret_cast<T*>(g.dv) + ((b * a.L + t0) * a.Hv + h) * a.V;
    // S and G' through descriptors that end with them: columns past Vp read zero
    const auto Sp = rsrc_of(g.states + unit * Vp * KP, (int)(Vp * KP * 4));
    const auto Gp = rsrc_of(g.grads + unit * Vp * KP, (int)(Vp * KP * 4));
    // a slice of V and dO, and this wave's columns of S and G', on their way
    Piece<T, VEC> pv, pd;
    f32x4 S[2 * NS], G[2 * NS];
    const int sr = tid / 8, scol = tid % 8 * 8;  // this thread's piece of a slice
    auto slice = [&](int64_t v0) {
      const int64_t left = a.V - v0 - scol;
      const int lim = sr < rows ? (left < 0 ? 0 : (left < 8 ? (int)left : 8)) : 0;
      pv.load(vp + (sr < rows ? sr : 0) * a.v_l + (left > 0 ? v0 + scol : 0), lim);
      pd.load(dp + (sr < rows ? sr : 0) * g.d_l + (left > 0 ? v0 + scol : 0), lim);
      const uint32_t at = ((uint32_t)(v0 + 16 * w + c) * KP + 8 * j) * 4;
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        const int k = (32 * (i >> 1) + 4 * (i & 1)) * 4;
        S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(Sp, at + k, 0, 0));
        G[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(Gp, at + k, 0, 0));
      }
    };
    auto put_slice = [&](int64_t v0) {
      const int64_t left = a.V - v0 - scol;
      const int lim = sr < rows ? (left < 0 ? 0 : (left < 8 ? (int)left : 8)) : 0;
      u32x4 p[NP];
      pv.planes(lim, p);
#pragma unroll
      for (int m = 0; m < NP; ++m)
        *reinterpret_cast<u32x4*>(&lds.V[m][sr * W::kVld + scol]) = p[m];
      pd.planes(lim, p);
#pragma unroll
      for (int m = 0; m < NP; ++m)
        *reinterpret_cast<u32x4*>(&lds.D[m][sr * W::kVld + scol]) = p[m];
    };
    {
      const auto wp = rsrc_of(g.ws + unit, (int)sizeof(ChunkWs));
      u32x4 t[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        t[i] = __builtin_amdgcn_raw_buffer_load_b128(wp, t_at(2 * i + tid / 128, tid % 128), 0, 0);
      const float f = (&g.ws[unit].fac[0][0])[tid];
      slice(0);
      __syncthreads();
      if (hh == 0) {
#pragma unroll
        for (int i = 0; i < kNk; ++i) {
          const int id = tid + 256 * i, r = id / (KP / 8), col = id % (KP / 8) * 8;
          if (kC * KP / 8 % 256 && r >= kC) continue;
          const int lim = r < rows ? K - col : 0;
          u32x4 p[NP];
          pk[i].planes(lim, p);
#pragma unroll
          for (int m = 0; m < NP; ++m)
            *reinterpret_cast<u32x4*>(&lds.K[m][r * W::kLd + col]) = p[m];
          pq[i].planes(lim, p);
#pragma unroll
          for (int m = 0; m < NP; ++m)
            *reinterpret_cast<u32x4*>(&lds.Q[m][r * W::kLd + col]) = p[m];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int id = tid + 256 * i;
        if (id < 384)
          *reinterpret_cast<u32x4*>(&lds.Tm[id / 128][id % 128 / 4 * kTld + id % 4 * 8]) = t[i];
      }
      (&lds.fac[0][0])[tid] = f;
      put_slice(0);
      __syncthreads();
    }
    auto fac8 = [&](int which, float* x) {  // of rows 8 j + e
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(&lds.fac[which][8 * j]);
      *reinterpret_cast<float4*>(x + 4) =
          *reinterpret_cast<const float4*>(&lds.fac[which][8 * j + 4]);
    };
    // this wave's tile of D, P and D kk: rows t = 8 j + 4 tx + r, column ti
    f32x4 dd, pp = zero4(), dkk = zero4();
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
      const float4 h4 = *reinterpret_cast<const float4*>(&lds.fac[kGhi][8 * j + 4 * tx]);
      const float4 l4 = *reinterpret_cast<const float4*>(&lds.fac[kGlo][8 * j + 4 * tx]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 8 * j + 4 * tx + r;
        const float d = exp2_fast(((&h4.x)[r] - hi) + ((&l4.x)[r] - lo));
        dd[r] = ti <= t ? d : 0.0f;
        pp[r] = ti <= t ? d * pp[r] : 0.0f;
        dkk[r] = ti < t ? d * dkk[r] : 0.0f;
      }
      put4<3>(lds.PT, ti * kTld + 8 * j + 4 * tx, pp);
    }
    __syncthreads();
    f32x4 X1[NK][2], X2[NK][2], X3[NK][2], dP = zero4(), dA = zero4();
    float ss = 0.0f;
#pragma unroll
    for (int m = 0; m < NK; ++m)
#pragma unroll
      for (int x = 0; x < 2; ++x) X1[m][x] = X2[m][x] = X3[m][x] = zero4();
    for (int64_t v0 = 0; v0 < (ONE ? 1 : a.V); v0 += 64) {
      if (v0) {
        put_slice(v0);
        __syncthreads();
      }
      const int64_t vc = v0 + 16 * w + c;
      const bool act = v0 + 16 * w < Vp;
      f32x4 ks[2] = {zero4(), zero4()}, kg[2] = {zero4(), zero4()}, qs[2] = {zero4(), zero4()};
      if (act) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          u32x4 sp[3], gp[3];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) ss = __builtin_fmaf(S[2 * s + x][r], G[2 * s + x][r], ss);
          split_tiles<3>(S[2 * s], S[2 * s + 1], sp);
          split_tiles<3>(G[2 * s], G[2 * s + 1], gp);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            u32x4 f[NP], q[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              f[p] = lds16(&lds.K[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
              q[p] = lds16(&lds.Q[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
            }
            ks[x] = mfma_planes<NP, 3, 3>(f, sp, ks[x]);
            kg[x] = mfma_planes<NP, 3, 3>(f, gp, kg[x]);
            qs[x] = mfma_planes<NP, 3, 3>(q, sp, qs[x]);
          }
        }
      }
      // the sums over v want S and G' the other way round: on their way now
      float s8[2][NK][8], g8[2][NK][8];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int m = 0; m < NK; ++m) {
          const int tile = w + 4 * m < 2 * NS ? w + 4 * m : 0;
          const uint32_t at = ((uint32_t)(v0 + 32 * q + 8 * j) * KP + 16 * tile + c) * 4;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s8[q][m][e] = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(Sp, at + e * KP * 4, 0, 0));
            g8[q][m][e] = __uint_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(Gp, at + e * KP * 4, 0, 0));
          }
        }
      if (act) {
        float v[8], d[8], x8[8];
        // per row 8 j + e, over this slice's columns: dR Y,
        // e^G (scale dO (Q S) - beta dR (K S)), e^(G_last - G) U (K G')
        float db[8], s1[8], s2[8];
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
            const uint32_t y = e & 1 ? dop[p][e >> 1] & 0xffff0000u : dop[p][e >> 1] << 16;
            v[e] = p == 0 ? __uint_as_float(x) : v[e] + __uint_as_float(x);
            d[e] = p == 0 ? __uint_as_float(y) : d[e] + __uint_as_float(y);
          }
        }
        f32x4 R[2], U[2] = {zero4(), zero4()}, Z[2] = {zero4(), zero4()};
        fac8(kEg, x8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = __builtin_fmaf(-x8[e], ks[e >> 2][e & 3], v[e]);  // Y
          s1[e] = x8[e] * a.scale * d[e] * qs[e >> 2][e & 3];
          ks[e >> 2][e & 3] *= x8[e];  // e^G K S
        }
        fac8(kBeta, x8);
#pragma unroll
        for (int e = 0; e < 8; ++e) R[e >> 2][e & 3] = x8[e] * v[e];
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
        fac8(kEnd, x8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s2[e] = x8[e] * U[e >> 2][e & 3] * kg[e >> 2][e & 3];
          Z[e >> 2][e & 3] = __builtin_fmaf(x8[e], kg[e >> 2][e & 3], a.scale * Z[e >> 2][e & 3]);
        }
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
        fac8(kBeta, x8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float r = R[e >> 2][e & 3];
          db[e] = r * v[e];
          s1[e] = __builtin_fmaf(-x8[e] * r, ks[e >> 2][e & 3], s1[e]);
          // one plane: dV through LDS where this wave's V was; otherwise as it is
          if constexpr (NP == 1) lds.V[0][(8 * j + e) * W::kVld + 16 * w + c] = f32_to_bf16_bits(x8[e] * r);
          else if (8 * j + e < rows && vc < a.V) stf(dvp + (8 * j + e) * a.Hv * a.V + vc, x8[e] * r);
        }
        const auto add = [&](float* row, const float* x, int e0) {
          float4 q = v0 ? *reinterpret_cast<const float4*>(row + e0) : make_float4(0, 0, 0, 0);
          q.x += x[e0]; q.y += x[e0 + 1]; q.z += x[e0 + 2]; q.w += x[e0 + 3];
          *reinterpret_cast<float4*>(row + e0) = q;
        };
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          db[e] = group_sum<16>(db[e]);
          s1[e] = group_sum<16>(s1[e]);
          s2[e] = group_sum<16>(s2[e]);
        }
        if (c == 0) {
#pragma unroll
          for (int q = 0; q < 8; q += 4) {
            add(&lds.row[w][2][8 * j], db, q);
            add(&lds.row[w][3][8 * j], s1, q);
            add(&lds.row[w][4][8 * j], s2, q);
          }
        }
      } else {
        if (v0 == 0) {
          for (int i = lane; i < 3 * kC; i += 64) lds.row[w][2 + i / kC][i % kC] = 0.0f;
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          *reinterpret_cast<u32x4*>(&lds.c.U[p][(16 * w + c) * kTld + 8 * j]) = u32x4{0, 0, 0, 0};
          *reinterpret_cast<u32x4*>(&lds.c.R[p][(16 * w + c) * kTld + 8 * j]) = u32x4{0, 0, 0, 0};
        }
      }
      __syncthreads();
      if constexpr (NP == 1) {
        const int64_t left = a.V - v0 - scol;
        T* p = dvp + sr * a.Hv * a.V + v0 + scol;
        const T* q = reinterpret_cast<const T*>(&lds.V[0][sr * W::kVld + scol]);
        if (sr < rows) {
          if (VEC) {
            if (left > 0) *reinterpret_cast<u32x4*>(p) = *reinterpret_cast<const u32x4*>(q);
          } else {
            for (int e = 0; e < 8 && e < left; ++e) p[e] = q[e];
          }
        }
      }
      const bool more = !ONE && v0 + 64 < a.V;
      if (more) slice(v0 + 64);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (v0 + 32 * q >= Vp) continue;
        __builtin_amdgcn_sched_barrier(0);  // one half's operands in registers at a time
        const auto rows_d = [&](int x, u32x4* f) {
#pragma unroll
          for (int p = 0; p < NP; ++p)
            f[p] = lds16(&lds.D[p][(ar + 4 * x) * W::kVld + 32 * q + 8 * j]);
        };
        const auto rows_of = [&](const uint16_t (&m)[3][64 * kTld], int x, u32x4* f, int np) {
#pragma unroll
          for (int p = 0; p < 3; ++p)
            if (p < np) f[p] = lds_col(&m[p][32 * q * kTld], kTld, 4 * x, lane);
        };
        {
          u32x4 da[NP], ra[3], ub[3];
          rows_d(tx, da);
          rows_of(lds.c.U, ty, ub, 3);
          rows_of(lds.c.R, tx, ra, 3);
          dP = mfma_planes<NP, 3, 3>(da, ub, dP);
          dA = mfma_planes<3, 3, 3>(ra, ub, dA);
        }
        u32x4 sp[NK][NO], gp[NK][NO];
#pragma unroll
        for (int m = 0; m < NK; ++m) {
          split8<NO>(s8[q][m], sp[m]);
          split8<NO>(g8[q][m], gp[m]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 fd[NP], fu[3], fr[3];
          rows_d(x, fd);
          rows_of(lds.c.U, x, fu, NO);
          rows_of(lds.c.R, x, fr, NO);
#pragma unroll
          for (int m = 0; m < NK; ++m) {
            if (w + 4 * m >= 2 * NS) continue;
            X1[m][x] = mfma_planes<NP, NO, NO>(fd, sp[m], X1[m][x]);
            X2[m][x] = mfma_planes<NO, NO, NO>(fu, gp[m], X2[m][x]);
            X3[m][x] = mfma_planes<NO, NO, NO>(fr, sp[m], X3[m][x]);
          }
        }
      }
      __syncthreads();
    }

    // the 32 x 32 tiles: M, E and the sums of F
    {
      f32x4 M, E;
      float frow[4], kb[4];
      const float4 b4 = *reinterpret_cast<const float4*>(&lds.fac[kBeta][8 * j + 4 * tx]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float bt = (&b4.x)[r], p = a.scale * dP[r], q = -dA[r];
        M[r] = p * dd[r];
        E[r] = ti < 8 * j + 4 * tx + r ? q * dd[r] * bt : 0.0f;
        frow[r] = __builtin_fmaf(p, pp[r], q * bt * dkk[r]);
        kb[r] = group_sum<16>(q * dkk[r]);
      }
      // F's columns before each row, from it on: in four rows here, the later ones below
#pragma unroll
      for (int r = 2; r >= 0; --r) frow[r] += frow[r + 1];
      lds.col[2 * j + tx][ti] = frow[0];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        frow[r] = group_sum<16>(ti < 8 * j + 4 * tx + r ? frow[r] : 0.0f);
      if (c == 0) {
        *reinterpret_cast<float4*>(&lds.row[w][0][8 * j + 4 * tx]) =
            make_float4(frow[0], frow[1], frow[2], frow[3]);
        *reinterpret_cast<float4*>(&lds.row[w][1][8 * j + 4 * tx]) =
            make_float4(kb[0], kb[1], kb[2], kb[3]);
      }
      put4<NO>(lds.m.M, ti * kTld + 8 * j + 4 * tx, M);
      put4<NO>(lds.m.E, ti * kTld + 8 * j + 4 * tx, E);
    }
    ss = group_sum<64>(ss);
    if (lane == 0) lds.dot[w] = ss;
    __syncthreads();
    if (w == (int)(n & 3)) {  // (the waves' turn about)
      const int t = lane & 31, x = t >> 2 & 1;  // the tiles of row t: waves 2 x, 2 x + 1
      const auto sum4 = [&](int i) {
        return (lds.row[0][i][t] + lds.row[1][i][t]) + (lds.row[2][i][t] + lds.row[3][i][t]);
      };
      const float kb = lds.row[2 * x][1][t] + lds.row[2 * x + 1][1][t];
      float f = lds.row[2 * x][0][t] + lds.row[2 * x + 1][0][t], later = 0.0f;
#pragma unroll
      for (int i = 6; i >= 0; --i) {  // what crosses the rows of group i in the groups past it
        const float y = lds.col[i + 1][t ? t - 1 : 0];
        later += t ? y : 0.0f;
        const float before = scan_incl<32>(later);
        f += t >> 2 == i ? before : 0.0f;
      }
      const float prev = __shfl_up(sum4(4), 1, 32);
      f += scan_incl<32>(t ? prev : 0.0f);
      double G_ = (double)sum4(3);
#pragma unroll
      for (int s = 1; s < 32; s *= 2) {
        const double y = __shfl_down(G_, s, 32);
        if (t + s < 32) G_ += y;
      }
      G_ += (double)f + (double)lds.fac[kEg][31] *
                            (double)((lds.dot[0] + lds.dot[1]) + (lds.dot[2] + lds.dot[3]));
      if (lane < rows) {
        const int64_t at = (b * a.L + t0 + t) * a.Hv + h;
        g.dg[at] = (float)G_;
        g.dbeta[at] = sum4(2) + kb;
      }
    }
    float be[8], eg[8], en[8];
    fac8(kBeta, be);
    fac8(kEg, eg);
    fac8(kEnd, en);
#pragma unroll
    for (int m = 0; m < NK; ++m) {
      const int tile = w + 4 * m;
      if (tile >= 2 * NS) continue;
      u32x4 kc[NP], qc[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kc[p] = lds_col16(lds.K[p], W::kLd, 16 * tile, lane);
        qc[p] = lds_col16(lds.Q[p], W::kLd, 16 * tile, lane);
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
  // one plane: through LDS, where Q and K were, for whole accesses
  if constexpr (NP == 1) __syncthreads();
#pragma unroll
  for (int m = 0; m < NK; ++m) {
    const int tile = w + 4 * m, key = 16 * tile + c;
    if (tile >= 2 * NS) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int t = 8 * j + e;
      if constexpr (NP == 1) {
        lds.Q[0][t * W::kLd + key] = f32_to_bf16_bits(aq[m][e >> 2][e & 3]);
        lds.K[0][t * W::kLd + key] = f32_to_bf16_bits(ak[m][e >> 2][e & 3]);
      } else if (t < rows && key < K) {
        stf(dqp + t * a.Hk * K + key, aq[m][e >> 2][e & 3]);
        stf(dkp + t * a.Hk * K + key, ak[m][e >> 2][e & 3]);
      }
    }
  }
  if constexpr (NP == 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kNk; ++i) {
      const int id = tid + 256 * i, r = id / (KP / 8), col = id % (KP / 8) * 8;
      if (r >= rows || col >= K) continue;
      const T* q = reinterpret_cast<const T*>(&lds.Q[0][r * W::kLd + col]);
      const T* k = reinterpret_cast<const T*>(&lds.K[0][r * W::kLd + col]);
      const int64_t at = r * a.Hk * K + col;
      if (VEC) {
        *reinterpret_cast<u32x4*>(dqp + at) = *reinterpret_cast<const u32x4*>(q);
        *reinterpret_cast<u32x4*>(dkp + at) = *reinterpret_cast<const u32x4*>(k);
      } else {
        for (int e = 0; e < 8 && col + e < K; ++e) {
          dqp[at + e] = q[e];
          dkp[at + e] = k[e];
        }
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
    f<<<grid_of(wgs), 256, bytes, s>>>(g);
    return launch_status();
  };
  static_assert(sizeof(typename Grad<T, KP, true>::Lds) <= 160 * 1024, "LDS of a CU");
  const int bytes = (int)sizeof(typename Grad<T, KP, true>::Lds);
  // without the loops over heads and slices 256 registers hold everything (88
  // bytes a lane spilled with them: 232 us against 171 at B=4 L=4096 H=16 K=V=64,
  // both of a first call); Hv > Hk or V > 64 cannot do without them
  if constexpr (Grad<T, KP, true>::kWaves == 2) {
    if (g.a.Hv == g.a.Hk && g.a.V <= 64)
      return vec ? go(delta_grads_kernel<T, KP, true, true>, bytes)
                 : go(delta_grads_kernel<T, KP, false, true>, bytes);
  }
  return vec ? go(delta_grads_kernel<T, KP, true, false>, bytes)
             : go(delta_grads_kernel<T, KP, false, false>, bytes);
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
