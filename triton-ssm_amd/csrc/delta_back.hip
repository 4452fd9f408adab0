// Gated delta rule, chunked, the way back: the gradient of the state, chunk
// after chunk from the last.
//
// With G' the gradient of the state after a chunk, P[t][i] = e^(G_t - G_i)
// q_t.k_i (i <= t), and S, T, U, R as in the walk:
//   dU = scale P^T dO + e^(G_last - G) K G',   dR = T^T dU,
//   G = e^(G_last) G' + scale Q^T (e^G dO) - K^T (beta e^G dR).
// As on the way there a wave owns 16 columns of V and their gradient stays in
// its registers; the terms in dO alone (Z = scale P^T dO and Y = scale Q^T e^G
// dO) are formed by two helper waves a chunk ahead, and two loaders bring K, Q,
// dO and T.  The gradient after every chunk goes to the workspace, where the
// gradients of the inputs are formed from it in parallel (delta_grads.hip).
// The walk that leaves the states needs nothing of this one: both go in one
// launch, each workgroup of one or the other.
// Two barriers a chunk: before the first the loaders put the next chunk into
// LDS while the chain waves multiply K G', after it the helpers work on that
// chunk.
// Bound like the walk by the chain waves' instructions.  B=4 L=4096 H=16 K=V=64
// bf16, 256 workgroups of both kinds: 178 us in one launch, which also writes 268
// MB of states and gradients (190 in a first call, where one after the other took
// 124 and 185).
#include "delta_walk.h"

namespace tssm {
namespace {

struct BackArgs {
  DeltaArgs a;         // v: dO; h0: dh_last or null; h_last: dh0 or null
  const ChunkWs* ws;
  int nch, per, nseg;
  uint32_t nvb;
  const float* entry;  // [bh][nseg][Vp][KP], the gradient after the segment (of one: a.h0)
  float* grads;        // [bh][nch][Vp][KP] after every chunk; from zero: [bh][nseg][Vp][KP] before it
};

template <typename T, int KP, bool VEC, int NCW>
struct Back {
  static constexpr int NP = Piece<T, VEC>::NP, NS = KP / 32, NT = NP == 1 ? 128 : 256;
  static constexpr int kThreads = 64 * (NCW + 2) + NT;
  static constexpr int kLd = KP + 8;
  static constexpr int kNk = (kC * KP / 8 + NT - 1) / NT;
  static constexpr int kVp = 2 * NCW;
  static constexpr int kVld = NP == 1 ? 16 * NCW + 8 : 16 * NCW + 4;
  static constexpr bool kEarly = NP * KP <= 128;
  static constexpr int kWaves = VEC && NP * KP < 384 ? 2 : 1;
  typedef std::conditional_t<NP == 1, uint16_t, float> vlds_t;
  struct Operands {
    uint16_t K[NP][kC * kLd], Q[NP][kC * kLd], M[3][kC * kTld];  // M: T
    vlds_t D[kC * kVld];                                         // dO
    float fac[kFac][kC];
  };
  struct Ahead {  // by the helpers, as the chain waves hold them
    f32x4 Z[2][64], Y[2 * NS][64];
  };
  struct Lds {
    Operands op[2];
    Ahead ahead[2][NCW];
  };
};

template <typename W, int NCW, bool ZERO>
__device__ inline void back_chain(const BackArgs& g, typename W::Lds& lds, int64_t bh, int seg,
                                  int64_t vc, int wv, int n0, int n1) {
  constexpr int NP = W::NP, NS = W::NS, KP = 32 * NS;
  const DeltaArgs& a = g.a;
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int K = (int)a.K;
  const int64_t Vp = (a.V + 15) / 16 * 16;
  const int ar = 8 * (c >> 2) + (c & 3);
  f32x4 S[2 * NS];  // the gradient after the chunk at hand
  if (ZERO || vc >= Vp) {
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) S[i] = zero4();
  } else if (g.nseg == 1) {
    get_state<NS>(a.h0 ? a.h0 + bh * K * a.V : nullptr, S, vc, a.V, K, j);
  } else {
    get_cols<NS>(g.entry + (bh * g.nseg + seg) * Vp * KP, S, vc, j);
  }
  __builtin_amdgcn_s_setprio(3);
  lds_barrier();
  lds_barrier();
  for (int n = n1 - 1; n >= n0; --n) {
    const typename W::Operands& B = lds.op[n & 1];
    const typename W::Ahead& ahead = lds.ahead[n & 1][wv];
    u32x4 fk[NS][2][NP], ft[2][3], fc[NP][2 * NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          fk[s][x][p] = lds16(&B.K[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
    float eg[8], be[8], en[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      *reinterpret_cast<float4*>(eg + 4 * q) =
          *reinterpret_cast<const float4*>(&B.fac[kEg][8 * j + 4 * q]);
      *reinterpret_cast<float4*>(be + 4 * q) =
          *reinterpret_cast<const float4*>(&B.fac[kBeta][8 * j + 4 * q]);
      *reinterpret_cast<float4*>(en + 4 * q) =
          *reinterpret_cast<const float4*>(&B.fac[kEnd][8 * j + 4 * q]);
    }
    const float last = B.fac[kEg][kC - 1];
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int x = 0; x < 2; ++x) ft[x][p] = lds_col(B.M[p], kTld, 4 * x, lane);
    if constexpr (W::kEarly) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i)
          fc[p][i] = lds_col(B.K[p], W::kLd, 32 * (i >> 1) + 4 * (i & 1), lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!ZERO) {
      if (vc < Vp) put_cols<NS>(g.grads + (bh * g.nch + n) * Vp * KP, S, vc, j);
    }
    f32x4 kg[2] = {zero4(), zero4()};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      u32x4 sp[3];
      split_tiles<3>(S[2 * s], S[2 * s + 1], sp);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int q = 0; q + p < 3; ++q)
#pragma unroll
          for (int x = 0; x < 2; ++x) kg[x] = mfma32(fk[s][x][p], sp[q], kg[x]);
    }
    lds_barrier();
    f32x4 U[2], R[2] = {zero4(), zero4()}, N[2 * NS];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const f32x4 z = ahead.Z[x][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) U[x][r] = __builtin_fmaf(en[4 * x + r], kg[x][r], z[r]);
    }
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) N[i] = ahead.Y[i][lane];
    u32x4 rp[3];
    split_tiles<3>(U[0], U[1], rp);
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int q = 0; q + p < 3; ++q)
#pragma unroll
        for (int x = 0; x < 2; ++x) R[x] = mfma32(ft[x][p], rp[q], R[x]);
#pragma unroll
    for (int e = 0; e < 8; ++e) R[e >> 2][e & 3] *= -be[e] * eg[e];
    u32x4 ep[3];
    split_tiles<3>(R[0], R[1], ep);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[i][r] = __builtin_fmaf(last, S[i][r], N[i][r]);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if constexpr (!W::kEarly) {
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i)
          fc[p][i] = lds_col(B.K[p], W::kLd, 32 * (i >> 1) + 4 * (i & 1), lane);
      }
#pragma unroll
      for (int q = 0; q + p < 3; ++q)
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) S[i] = mfma32(fc[p][i], ep[q], S[i]);
    }
    lds_barrier();
  }
  if constexpr (ZERO) {
    if (vc < Vp) put_cols<NS>(g.grads + (bh * g.nseg + seg) * Vp * KP, S, vc, j);
  } else if (n0 == 0) {
    put_state<NS>(a.h_last ? a.h_last + bh * K * a.V : nullptr, S, vc, a.V, K, j);
  }
}

// Z's rows 8 j + 4 y + r and every other tile of Y, for the chunk that is in LDS.
template <typename T, int KP, bool VEC, int NCW>
__device__ inline void back_help(const BackArgs& g, typename Back<T, KP, VEC, NCW>::Lds& lds,
                                 int y, int n0, int n1) {
  typedef Back<T, KP, VEC, NCW> W;
  constexpr int NP = W::NP, NS = W::NS;
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int ar = 8 * (c >> 2) + (c & 3);
  const float scale = g.a.scale;
  auto work = [&](int n) {
    const typename W::Operands& B = lds.op[n & 1];
    // (Q K^T)[t][i]: its rows are the sum's index of P^T dO, so its tiles are
    // P^T's A operand as they stand
    f32x4 qk[2] = {zero4(), zero4()};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      u32x4 fk[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fk[p] = lds16(&B.K[p][(ar + 4 * y) * W::kLd + 32 * s + 8 * j]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4 f[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p)
          f[p] = lds16(&B.Q[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
        qk[x] = mfma_planes<NP, NP, 3>(f, fk, qk[x]);
      }
    }
    const int i = ar + 4 * y;
    const float hi = B.fac[kGhi][i], lo = B.fac[kGlo][i];
    float eg[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float4 h4 = *reinterpret_cast<const float4*>(&B.fac[kGhi][8 * j + 4 * x]);
      const float4 l4 = *reinterpret_cast<const float4*>(&B.fac[kGlo][8 * j + 4 * x]);
      *reinterpret_cast<float4*>(eg + 4 * x) =
          *reinterpret_cast<const float4*>(&B.fac[kEg][8 * j + 4 * x]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float d = exp2_fast(((&h4.x)[r] - hi) + ((&l4.x)[r] - lo)) * qk[x][r];
        qk[x][r] = i <= 8 * j + 4 * x + r ? d : 0.0f;
      }
    }
    u32x4 fp[3];
    split_tiles<3>(qk[0], qk[1], fp);
#pragma unroll
    for (int w = 0; w < NCW; ++w) {
      typename W::Ahead& out = lds.ahead[n & 1][w];
      float d[8];
      u32x4 dp[NP], yp[3];
      if constexpr (NP == 1) {
        const uint16_t* p = B.D + (8 * j + (c >> 2)) * W::kVld + 16 * w + 4 * (c & 3);
        const u32x2v u0 = lds_tr(p), u1 = lds_tr(p + 4 * W::kVld);
        dp[0] = u32x4{u0[0], u0[1], u1[0], u1[1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[2 * e] = __uint_as_float(dp[0][e] << 16);
          d[2 * e + 1] = __uint_as_float(dp[0][e] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = B.D[(8 * j + e) * W::kVld + 16 * w + c];
        split8<NP>(d, dp);
      }
      f32x4 z = mfma_planes<3, NP, 3>(fp, dp, zero4());
#pragma unroll
      for (int r = 0; r < 4; ++r) z[r] *= scale;
      out.Z[y][lane] = z;
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] *= scale * eg[e];
      split8<3>(d, yp);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        u32x4 f[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) f[p] = lds_col(B.Q[p], W::kLd, 32 * s + 4 * y, lane);
        out.Y[2 * s + y][lane] = mfma_planes<NP, 3, 3>(f, yp, zero4());
      }
    }
  };
  lds_barrier();
  work(n1 - 1);
  lds_barrier();
  for (int n = n1 - 1; n >= n0; --n) {
    lds_barrier();
    if (n > n0) work(n - 1);
    lds_barrier();
  }
}

template <typename T, int KP, bool VEC, int NCW>
__device__ inline void back_bring(const BackArgs& g, typename Back<T, KP, VEC, NCW>::Lds& lds,
                                  int64_t bh, int64_t v0, int n0, int n1) {
  typedef Back<T, KP, VEC, NCW> W;
  constexpr int NP = W::NP, NT = W::NT, kE = (int)sizeof(T);
  const DeltaArgs& a = g.a;
  const ChunkWs* ws = g.ws + bh * (int64_t)g.nch;
  const int id = threadIdx.x - (W::kThreads - NT);
  const auto [b, h, hk] = head_of(a, (uint32_t)bh);
  const int nv = a.V - v0 < 16 * NCW ? (int)(a.V - v0) : 16 * NCW, K = (int)a.K;
  ChunkRows rk, rq, rv;
  rk.init(reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, a.k_l, K, a.L);
  rq.init(reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h, a.q_l, K, a.L);
  rv.init(reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + v0, a.v_l, nv, a.L);
  uint32_t ok[W::kNk], oq[W::kNk];
#pragma unroll
  for (int i = 0; i < W::kNk; ++i) {
    const int r = (id + NT * i) / (KP / 8), col = (id + NT * i) % (KP / 8) * 8;
    ok[i] = r < kC && col < K ? r * rk.row + col * kE : kPast;
    oq[i] = r < kC && col < K ? r * rq.row + col * kE : kPast;
  }
  const uint32_t vid = id - (NT - 128);
  const int vr = (int)(vid / W::kVp), vcol = (int)(vid % W::kVp) * 8;
  const uint32_t ov = vr < kC && vcol < nv ? vr * rv.row + vcol * kE : kPast;
  struct Regs {
    Piece<T, VEC> k[W::kNk], q[W::kNk], v;
    u32x4 t[3];
    u32x2v f;
  };
  auto load = [&](Regs& r, int n) {
    const auto dk = rk.at(n), dq = rq.at(n), dv = rv.at(n);
    const auto dw = rsrc_of(chunk_at(ws, n, g.nch), (int)sizeof(ChunkWs));
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      r.k[i].load(dk, ok[i]);
      r.q[i].load(dq, oq[i]);
    }
    r.v.load(dv, ov);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      r.t[i] = __builtin_amdgcn_raw_buffer_load_b128(dw, id < 128 ? t_at(i, id) : kPast, 0, 0);
    r.f = __builtin_amdgcn_raw_buffer_load_b64(dw, 3 * kPlane + 8 * (id & 127), 0, 0);
  };
  auto store = [&](const Regs& r, int n) {
    typename W::Operands& B = lds.op[n & 1];
    u32x4 p[NP];
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int row = (id + NT * i) / (KP / 8), col = (id + NT * i) % (KP / 8) * 8;
      if (kC * KP / 8 < NT && row >= kC) continue;
      const int lim = VEC ? 8 : K - col;
      r.k[i].planes(lim, p);
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&B.K[x][row * W::kLd + col]) = p[x];
      r.q[i].planes(lim, p);
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&B.Q[x][row * W::kLd + col]) = p[x];
    }
    if (kC * W::kVp == NT || vr < kC) {
      const int lim = VEC ? 8 : nv - vcol;
      if constexpr (NP == 1) {
        r.v.planes(lim, p);
        *reinterpret_cast<u32x4*>(&B.D[vr * W::kVld + vcol]) = p[0];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          B.D[vr * W::kVld + vcol + e] = e < lim ? ldf(&r.v.e[e]) : 0.0f;
      }
    }
    if (NT == 128 || id < 128) {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        *reinterpret_cast<u32x4*>(&B.M[i][id / 4 * kTld + id % 4 * 8]) = r.t[i];
    }
    if (NT == 128 || id >= 128)
      *reinterpret_cast<u32x2v*>(&B.fac[0][0] + 2 * (id & 127)) = r.f;
  };
  Regs g0, g1;
  load(g0, n1 - 1);
  load(g1, n1 - 2);
  store(g0, n1 - 1);
  lds_barrier();
  lds_barrier();
  auto turn = [&](int n, Regs& y, Regs& x) {  // x holds chunk n - 1
    load(y, n - 2);
    if (n > n0) store(x, n - 1);
    lds_barrier();
    lds_barrier();
  };
  for (int n = n1 - 1; n >= n0; n -= 2) {
    turn(n, g0, g1);
    if (n - 1 >= n0) turn(n - 1, g1, g0);
  }
}

template <typename T, int KP, bool VEC, int NCW, bool ZERO>
__device__ inline void back_body(const BackArgs& g, char* raw, uint32_t block) {
  typedef Back<T, KP, VEC, NCW> W;
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(raw);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t heads = (uint32_t)(g.a.B * g.a.Hv);
  const uint32_t run = block / (8 * g.nvb) * 8 + (block & 7);
  const int seg = (int)(run / heads) + (ZERO ? 1 : 0);
  if (seg >= g.nseg) return;
  const int64_t bh = run % heads;
  const int n0 = seg * g.per, n1 = n0 + g.per < g.nch ? n0 + g.per : g.nch;
  const int64_t v0 = (int64_t)(block / 8 % g.nvb) * 16 * NCW;
  if (wv < NCW)
    back_chain<W, NCW, ZERO>(g, lds, bh, seg, v0 + 16 * wv + (threadIdx.x & 15), wv, n0, n1);
  else if (wv < NCW + 2)
    back_help<T, KP, VEC, NCW>(g, lds, wv - NCW, n0, n1);
  else
    back_bring<T, KP, VEC, NCW>(g, lds, bh, v0, n0, n1);
}

// The first nback workgroups walk back, the others there.  (Waves that one of
// the two has no use for end at once: barriers count the others.)
template <typename T, int KP, bool VEC, int NCW, bool ZERO>
struct Both {
  static constexpr int MODE = ZERO ? kTransfer : kStates;
  typedef Back<T, KP, VEC, NCW> B;
  typedef Walk<T, KP, VEC, 2, MODE> F;
  static constexpr int kThreads = B::kThreads > F::kThreads ? B::kThreads : F::kThreads;
  static constexpr int kBytes = sizeof(typename B::Lds) > sizeof(typename F::Lds)
                                    ? (int)sizeof(typename B::Lds) : (int)sizeof(typename F::Lds);
};
template <typename T, int KP, bool VEC, int NCW, bool ZERO>
__global__ __launch_bounds__((Both<T, KP, VEC, NCW, ZERO>::kThreads),
                             (Back<T, KP, VEC, NCW>::kWaves)) void
    delta_both_kernel(BackArgs g, WalkArgs f, uint32_t nback) {
  typedef Both<T, KP, VEC, NCW, ZERO> W;
  extern __shared__ __attribute__((aligned(16))) char raw[];
  const uint32_t block = block_of();
  if (block < nback) {
    if (threadIdx.x < W::B::kThreads) back_body<T, KP, VEC, NCW, ZERO>(g, raw, block);
  } else {
    if (threadIdx.x < W::F::kThreads)
      walk_body<T, KP, VEC, 2, W::MODE>(f, raw, block - nback);
  }
}

template <typename T, int KP, bool VEC, int NCW, bool ZERO>
int both_launch(BackArgs& g, WalkArgs& f, hipStream_t s) {
  typedef Both<T, KP, VEC, NCW, ZERO> W;
  g.nvb = (uint32_t)cdiv64(g.a.V, 16 * NCW);
  const int64_t nb = cdiv64(g.a.B * g.a.Hv * (ZERO ? g.nseg - 1 : g.nseg), 8) * 8 * g.nvb;
  const int64_t nf = walk_wgs<KP, 2, W::MODE>(f);
  if (nb > 0x3fffffff || nf < 0) return TSSM_ERR_UNSUPPORTED;
  static_assert(W::kBytes <= 160 * 1024, "LDS of a CU");
  auto* k = delta_both_kernel<T, KP, VEC, NCW, ZERO>;
  if (W::kBytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, W::kBytes);
    if (e != hipSuccess) return (int)e;
  }
  k<<<grid_of(nb + nf), W::kThreads, W::kBytes, s>>>(g, f, (uint32_t)nb);
  return launch_status();
}

template <typename T, bool ZERO>
int both_any(BackArgs& g, WalkArgs& f, bool vec, hipStream_t s) {
  constexpr int NW = std::is_same<T, bf16_t>::value ? 2 : 1;
  if (g.a.K <= 32)
    return vec ? both_launch<T, 32, true, 2, ZERO>(g, f, s)
               : both_launch<T, 32, false, 2, ZERO>(g, f, s);
  if (g.a.K <= 64)
    return vec ? both_launch<T, 64, true, 2, ZERO>(g, f, s)
               : both_launch<T, 64, false, 2, ZERO>(g, f, s);
  return vec ? both_launch<T, 128, true, NW, ZERO>(g, f, s)
             : both_launch<T, 128, false, NW, ZERO>(g, f, s);
}

template <bool ZERO>
int both(int dtype, BackArgs& g, WalkArgs& f, bool vec, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return both_any<float, ZERO>(g, f, vec, s);
    case TSSM_BF16: return both_any<bf16_t, ZERO>(g, f, vec, s);
    default: return both_any<f16_t, ZERO>(g, f, vec, s);
  }
}

}  // namespace

int delta_both_launch(int dtype, const DeltaArgs& a, const DeltaArgs& way, bool vec,
                      const DeltaPlan& p, hipStream_t s) {
  WalkArgs f = {};
  f.a = a;
  f.ws = reinterpret_cast<const ChunkWs*>(p.chunks);
  f.nch = p.nch;
  f.per = p.per;
  f.nseg = f.walked = p.nseg;
  BackArgs g = {};
  g.a = way;
  g.ws = f.ws;
  g.nch = p.nch;
  g.per = p.per;
  g.nseg = p.nseg;
  if (p.nseg > 1) {  // all segments' transfer: the last one's is for the way back
    f.states = p.transfer;
    g.grads = p.back;
    int rc = both<true>(dtype, g, f, vec, s);
    if (!rc) rc = delta_fold(a, p, s);
    if (!rc) rc = delta_fold_back(way, p, s);
    if (rc) return rc;
  }
  f.entry = p.entry;
  f.states = p.states;
  g.entry = p.gentry;
  g.grads = p.grads;
  return both<false>(dtype, g, f, vec, s);
}

}  // namespace tssm
