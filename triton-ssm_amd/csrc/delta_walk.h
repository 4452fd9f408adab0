// Gated delta rule, chunked: the walk over the chunks.
//
// Per chunk of 32 steps, with S the state before it, T and G from the
// preparing pass and P[t][i] = e^(G_t - G_i) q_t.k_i (i <= t):
//   R = beta (V - e^G K S),  U = T R,  O = scale (e^G Q S + P U),
//   S' = e^(G_last) S + K^T (e^(G_last - G) U).
// Columns of V never meet, so a wave owns 16 of them for the whole sequence,
// their state in its registers, and each product's result is the next one's B
// operand in place (delta_dev.h).
//
// The chain S -> R -> U -> S' sets the time, one chunk after the other, so it
// has waves of its own.  A workgroup is NCW of them, two output waves and two
// loaders, on the four SIMDs of a CU.  The loaders bring K, Q, V and T into LDS
// two chunks ahead.  The output waves form the outputs of the chunk before from
// the planes of S and U that the chain waves leave in LDS, one wave rows
// 8 j + r, one rows 8 j + 4 + r.  One barrier a chunk.
//
// Two more forms of the walk have chain waves and loaders only: one leaves the
// state before every chunk in the workspace (for the gradients), one walks
// the segments of a long sequence from zero, and V + K columns: the K more
// start as unit vectors and take no input, which gives the segment's transfer
// matrix (delta_states.hip joins them).
//
// A chunk whose U is not finite is done again step by step from S: zero
// weights would otherwise carry a later step's NaN to earlier outputs.
//
// What bounds it is the chain waves' own instructions, one after the other from one
// wave: about 300 a chunk of K = 64 bf16, 2100 cycles with the rest of the
// workgroup idle and 2170 with it at work (an 8-byte instruction leaves a wave
// every 6.5 cycles); 2980 of 3180 at K = 128, 2710 of 3150 in fp32 at K = 40.  112
// of the 300 split S, R and U into planes, 36 are matrix instructions.  B=8 L=4096
// H=16 K=V=64 bf16: 122 us once the clock has settled (148 in a first call), 128
// chunks in a row; B=2 L=2000 Hv=16 K=V=128: 96 us.  With its operands straight
// from memory, two chunks ahead, it took 145 against 128 us, with three chunks in
// LDS and reads a chunk ahead 127 against 122.
#pragma once

#include "delta_dev.h"

namespace tssm {
namespace {

enum { kOutputs, kStates, kTransfer };

// Sequences are walked in nseg segments of `per` chunks; a segment's entry
// state is entry[bh][seg] (a.h0 where there is one).
struct WalkArgs {
  DeltaArgs a;
  const ChunkWs* ws;
  int nch, per, nseg;
  int walked;          // the first segments that are walked
  uint32_t nvb;        // workgroups of a head and segment
  const float* entry;  // [bh][nseg][Vp][KP]
  float* states;       // kStates: [bh][nch][Vp][KP]; kTransfer: [bh][nseg][Vp + KP][KP]
};

template <typename T, int KP, bool VEC, int NCW, int MODE>
struct Walk {
  static constexpr int NP = Piece<T, VEC>::NP;  // planes of the inputs
  // of S, P and U in the products that reach the outputs alone: with bf16's two
  // (2^-17 of a value that is rounded to 2^-9) 0.34% of the outputs are the bf16
  // next to the nearest, with three 0.016%, at the same error against 64 bits
  // (1.7e-3, normwise) and 155 against 165 us for B=8 L=4096 H=16 K=V=64
  static constexpr int NO = NP == 1 ? 2 : 3;
  static constexpr int NS = KP / 32;
  // threads of the loaders: those of fp32 and fp16 split what they bring (B=3 L=1111
  // 12 heads of 40 x 72: 57.4 us with 128, 55.7 with 256)
  static constexpr int NT = NP == 1 ? 128 : 256;
  static constexpr int kThreads = 64 * (NCW + (MODE == kOutputs ? 2 : 0)) + NT;
  static constexpr int kLd = KP + 8;            // bf16 elements of a row of K or Q in LDS
  static constexpr int kNk = (kC * KP / 8 + NT - 1) / NT;  // 8-element pieces of K a thread brings
  static constexpr int kVp = 2 * NCW;           // pieces of a row of V
  static constexpr int kVld = NP == 1 ? 16 * NCW + 8 : 16 * NCW + 4;  // elements of V's row
  // 256 registers where they suffice: with more to give out the compiler puts
  // products into accumulation registers and copies them back
  static constexpr bool kEarly = NP * KP <= 128;  // registers for K^T's operands too
  static constexpr int kWaves = VEC && NP * KP < 384 ? 2 : 1;
  typedef std::conditional_t<NP == 1, uint16_t, float> vlds_t;
  struct Operands {  // of one chunk
    uint16_t K[NP][kC * kLd], Q[MODE == kOutputs ? NP : 1][MODE == kOutputs ? kC * kLd : 8];
    uint16_t M[3][kC * kTld];  // T
    vlds_t V[kC * kVld];
    float fac[kFac][kC];
  };
  struct Left {      // by a chain wave for its outputs: B operands, or the outputs themselves
    union {
      u32x4 S[NS][NO][64];
      float y[kC][16];
    };
    f32x4 U[2][64];
    int slow;
  };
  struct Lds {
    Operands op[2];
    Left left[MODE == kOutputs ? 2 : 1][MODE == kOutputs ? NCW : 1];
  };
};

// A wave's 16 columns through the chunks of a segment.
template <typename W, int NCW, int MODE>
__device__ inline void chain(const WalkArgs& g, typename W::Lds& lds, int64_t bh, int seg,
                             int64_t vc, int wv, int n0, int n1) {
  constexpr int NP = W::NP, NS = W::NS, KP = 32 * NS;
  const DeltaArgs& a = g.a;
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int K = (int)a.K;
  const int64_t Vp = (a.V + 15) / 16 * 16;
  const int ar = 8 * (c >> 2) + (c & 3);  // row of tile x that this lane holds of an A operand, less 4 x
  // S[k][c], k = 32 s + 8 j + 4 x + r, in tile 2 s + x register r
  f32x4 S[2 * NS];
  if constexpr (MODE == kTransfer) {
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S[i][r] = vc - Vp == 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r ? 1.0f : 0.0f;
  } else if (g.nseg == 1) {
    get_state<NS>(a.h0 ? a.h0 + bh * K * a.V : nullptr, S, vc, a.V, K, j);
  } else if (vc < Vp) {
    get_cols<NS>(g.entry + (bh * g.nseg + seg) * Vp * KP, S, vc, j);
  } else {
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) S[i] = zero4();
  }
  __builtin_amdgcn_s_setprio(3);  // before the loader on the same SIMD
  lds_barrier();
  for (int n = n0; n < n1; ++n) {
    const typename W::Operands& B = lds.op[n & 1];
    typename W::Left& left = lds.left[MODE == kOutputs ? n & 1 : 0][MODE == kOutputs ? wv : 0];
    // every operand but V's decays is asked for here: read where they are
    // used, each product would wait for LDS
    u32x4 fk[NS][2][NP], ft[2][3], fc[NP][2 * NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          fk[s][x][p] = lds16(&B.K[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
    float v[8], eg[8], be[8], en[8];
    if constexpr (NP == 1) {
      const uint16_t* p = B.V + (8 * j + (c >> 2)) * W::kVld + 16 * wv + 4 * (c & 3);
      const u32x2v lo = lds_tr(p), hi = lds_tr(p + 4 * W::kVld);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = e < 2 ? lo[e & 1] : hi[e & 1];
        v[2 * e] = __uint_as_float(w << 16);
        v[2 * e + 1] = __uint_as_float(w & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = B.V[(8 * j + e) * W::kVld + 16 * wv + c];
    }
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
      for (int x = 0; x < 2; ++x) ft[x][p] = lds16(&B.M[p][(ar + 4 * x) * kTld + 8 * j]);
    if constexpr (W::kEarly) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i)
          fc[p][i] = lds_col(B.K[p], W::kLd, 32 * (i >> 1) + 4 * (i & 1), lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MODE == kStates) {
      if (vc < Vp) put_cols<NS>(g.states + (bh * g.nch + n) * Vp * KP, S, vc, j);
    }
    f32x4 ks[2] = {zero4(), zero4()};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      u32x4 sp[3];
      split_tiles<3>(S[2 * s], S[2 * s + 1], sp);
      if constexpr (MODE == kOutputs) {
#pragma unroll
        for (int p = 0; p < W::NO; ++p) left.S[s][p][lane] = sp[p];
      }
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int q = 0; q + p < 3; ++q)
#pragma unroll
          for (int x = 0; x < 2; ++x) ks[x] = mfma32(fk[s][x][p], sp[q], ks[x]);
    }
    f32x4 R[2], U[2] = {zero4(), zero4()};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      R[e >> 2][e & 3] = be[e] * __builtin_fmaf(-eg[e], ks[e >> 2][e & 3], v[e]);
    u32x4 rp[3];
    split_tiles<3>(R[0], R[1], rp);
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int q = 0; q + p < 3; ++q)
#pragma unroll
        for (int x = 0; x < 2; ++x) U[x] = mfma32(ft[x][p], rp[q], U[x]);
    float big = 0.0f;
    f32x4 E[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      big += __builtin_fabsf(U[e >> 2][e & 3]);
      E[e >> 2][e & 3] = en[e] * U[e >> 2][e & 3];
    }
    if constexpr (MODE == kOutputs) {
      left.U[0][lane] = U[0];
      left.U[1][lane] = U[1];
    }
    u32x4 ep[3];
    split_tiles<3>(E[0], E[1], ep);
    f32x4 N[2 * NS];
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) N[i][r] = S[i][r] * last;
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
        for (int i = 0; i < 2 * NS; ++i) N[i] = mfma32(fc[p][i], ep[q], N[i]);
    }
    const bool slow = __ballot(!(big < __builtin_inff())) != 0;
    if (MODE == kOutputs && lane == 0) left.slow = slow;
    if (__builtin_expect(slow, 0)) {
      const int rows = a.L - (int64_t)n * kC < kC ? (int)(a.L - (int64_t)n * kC) : kC;
#pragma unroll 1
      for (int t = 0; t < rows; ++t) {
        const float al = exp_acc(B.fac[kG][t]), bt = B.fac[kBeta][t];
        auto row = [&](const auto& m, int i, int r) {
          const int at = t * W::kLd + 32 * (i >> 1) + 8 * j + 4 * (i & 1) + r;
          float x = 0.0f;
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) x += bf16_bits_to_f32(m[p][at]);
          return x;
        };
        float vt = 0.0f, s = 0.0f, y = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) vt = (t & 7) == e ? v[e] : vt;
        vt = __shfl(vt, (t >> 3) * 16 + c);
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
            if constexpr (MODE == kOutputs) y = __builtin_fmaf(row(B.Q, i, r), S[i][r], y);
          }
        if constexpr (MODE == kOutputs) {
          y += __shfl_xor(y, 16);
          y += __shfl_xor(y, 32);
          if (j == 0) left.y[t][c] = y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) S[i] = N[i];
    }
    lds_barrier();
  }
  if constexpr (MODE == kTransfer) {
    if (vc < Vp + KP) put_cols<NS>(g.states + (bh * g.nseg + seg) * (Vp + KP) * KP, S, vc, j);
  } else if (n1 == g.nch) {
    put_state<NS>(a.h_last ? a.h_last + bh * K * a.V : nullptr, S, vc, a.V, K, j);
  }
}

// The operands' way to LDS.
template <typename T, int KP, bool VEC, int NCW, int MODE>
__device__ inline void bring(const WalkArgs& wa, typename Walk<T, KP, VEC, NCW, MODE>::Lds& lds,
                             int64_t bh, int64_t v0, int n0, int n1) {
  typedef Walk<T, KP, VEC, NCW, MODE> W;
  const DeltaArgs& a = wa.a;
  const ChunkWs* ws = wa.ws + bh * (int64_t)wa.nch;
  constexpr int NP = W::NP, NT = W::NT, kE = (int)sizeof(T);
  const int id = threadIdx.x - (W::kThreads - NT);
  const auto [b, h, hk] = head_of(a, (uint32_t)bh);
  // columns past V (a transfer's unit vectors) have no input
  const int nv = a.V - v0 < 16 * NCW ? (a.V - v0 < 0 ? 0 : (int)(a.V - v0)) : 16 * NCW;
  const int K = (int)a.K;
  ChunkRows rk, rq, rv;
  rk.init(reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, a.k_l, K, a.L);
  rq.init(reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h, a.q_l, K, a.L);
  rv.init(reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + (nv ? v0 : 0),
          a.v_l, nv ? nv : 1, a.L);
  uint32_t ok[W::kNk], oq[W::kNk];
#pragma unroll
  for (int i = 0; i < W::kNk; ++i) {
    const int r = (id + NT * i) / (KP / 8), col = (id + NT * i) % (KP / 8) * 8;
    ok[i] = r < kC && col < K ? r * rk.row + col * kE : kPast;
    oq[i] = r < kC && col < K ? r * rq.row + col * kE : kPast;
  }
  // this thread's piece of V: with 256 the first half brings T, the second V
  const uint32_t vid = id - (NT - 128);
  const int vr = (int)(vid / W::kVp), vcol = (int)(vid % W::kVp) * 8;
  const uint32_t ov = vr < kC && vcol < nv ? vr * rv.row + vcol * kE : kPast;

  // as they lie in memory: a conversion on the way would wait for the load
  struct Regs {
    Piece<T, VEC> k[W::kNk], q[W::kNk], v;
    u32x4 t[3];
    u32x2v f;
  };
  auto load = [&](Regs& g, int n) {
    const auto dk = rk.at(n), dq = rq.at(n), dv = rv.at(n);
    const auto dw = rsrc_of(chunk_at(ws, n, wa.nch), (int)sizeof(ChunkWs));
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      g.k[i].load(dk, ok[i]);
      if constexpr (MODE == kOutputs) g.q[i].load(dq, oq[i]);
    }
    g.v.load(dv, ov);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      g.t[i] = __builtin_amdgcn_raw_buffer_load_b128(dw, id < 128 ? t_at(i, id) : kPast, 0, 0);
    g.f = __builtin_amdgcn_raw_buffer_load_b64(dw, 3 * kPlane + 8 * (id & 127), 0, 0);
  };
  // Only whole pieces are read with VEC, and what lies past a row or the
  // sequence reads zero; without it a piece may run into what follows its row.
  auto store = [&](const Regs& g, int n) {
    typename W::Operands& B = lds.op[n & 1];
    u32x4 p[NP];
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int r = (id + NT * i) / (KP / 8), col = (id + NT * i) % (KP / 8) * 8;
      if (kC * KP / 8 < NT && r >= kC) continue;
      const int lim = VEC ? 8 : K - col;
      g.k[i].planes(lim, p);
#pragma unroll
      for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&B.K[x][r * W::kLd + col]) = p[x];
      if constexpr (MODE == kOutputs) {
        g.q[i].planes(lim, p);
#pragma unroll
        for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x4*>(&B.Q[x][r * W::kLd + col]) = p[x];
      }
    }
    if (kC * W::kVp == NT || vr < kC) {
      const int lim = VEC ? 8 : nv - vcol;
      if constexpr (NP == 1) {
        g.v.planes(lim, p);
        *reinterpret_cast<u32x4*>(&B.V[vr * W::kVld + vcol]) = p[0];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          B.V[vr * W::kVld + vcol + e] = e < lim ? ldf(&g.v.e[e]) : 0.0f;
      }
    }
    if (NT == 128 || id < 128) {
#pragma unroll
      for (int i = 0; i < 3; ++i)  // 128 pieces are one plane
        *reinterpret_cast<u32x4*>(&B.M[i][id / 4 * kTld + id % 4 * 8]) = g.t[i];
    }
    if (NT == 128 || id >= 128)
      *reinterpret_cast<u32x2v*>(&B.fac[0][0] + 2 * (id & 127)) = g.f;
  };
  static_assert(kC * kC == 8 * 128 && kFac * kC == 2 * 128, "pieces of a chunk");

  Regs g0, g1;
  load(g0, n0);
  load(g1, n0 + 1);
  store(g0, n0);
  lds_barrier();
  // the chain waves are in chunk n; nx holds chunk n + 1, g takes n + 2
  auto turn = [&](int n, Regs& g, Regs& nx) {
    load(g, n + 2);
    store(nx, n + 1);
    lds_barrier();
  };
  for (int n = n0; n < n1; n += 2) {
    turn(n, g0, g1);
    if (n + 1 < n1) turn(n + 1, g1, g0);
  }
}

// The outputs of rows 8 j + 4 y + r, one chunk behind the chain waves.
template <typename T, int KP, bool VEC, int NCW>
__device__ inline void outputs(const DeltaArgs& a, typename Walk<T, KP, VEC, NCW, kOutputs>::Lds& lds,
                               int64_t bh, int64_t v0, int y, int n0, int n1) {
  typedef Walk<T, KP, VEC, NCW, kOutputs> W;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, kE = (int)sizeof(T);
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int ar = 8 * (c >> 2) + (c & 3);
  const auto [b, h, hk] = head_of(a, (uint32_t)bh);
  const int nv = a.V - v0 < 16 * NCW ? (int)(a.V - v0) : 16 * NCW;
  ChunkRows ro;
  ro.init(reinterpret_cast<T*>(a.o) + b * a.o_b + h * a.o_h + v0, a.o_l, nv, a.L);
  uint32_t oo[NCW][4];
#pragma unroll
  for (int g = 0; g < NCW; ++g)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      oo[g][r] = 16 * g + c < nv ? (8 * j + 4 * y + r) * ro.row + (16 * g + c) * kE : kPast;

  // what the outputs of a chunk need besides S and U: read while the chunk is
  // in LDS, used when the chain waves are past it
  u32x4 fq[NS][NP], fp[NO];
  float eg[4];
  auto weights = [&](int n) {
    const typename W::Operands& B = lds.op[n & 1];
    // (K Q^T)[i][t]: its rows are the sum's index of P U, so P^T's tiles are
    // P's A operand as they stand
    f32x4 kq[2] = {zero4(), zero4()};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
        fq[s][p] = lds16(&B.Q[p][(ar + 4 * y) * W::kLd + 32 * s + 8 * j]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4 f[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p)
          f[p] = lds16(&B.K[p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
        kq[x] = mfma_planes<NP, NP, 3>(f, fq[s], kq[x]);
      }
    }
    const int t = ar + 4 * y;
    const float hi = B.fac[kGhi][t], lo = B.fac[kGlo][t];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float4 h4 = *reinterpret_cast<const float4*>(&B.fac[kGhi][8 * j + 4 * x]);
      const float4 l4 = *reinterpret_cast<const float4*>(&B.fac[kGlo][8 * j + 4 * x]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float d = exp2_fast((hi - (&h4.x)[r]) + (lo - (&l4.x)[r])) * kq[x][r];
        kq[x][r] = 8 * j + 4 * x + r <= t ? d : 0.0f;
      }
    }
    split_tiles<NO>(kq[0], kq[1], fp);
    *reinterpret_cast<float4*>(eg) =
        *reinterpret_cast<const float4*>(&B.fac[kEg][8 * j + 4 * y]);
  };
  auto put = [&](int n) {
    const auto dst = ro.at(n);
    f32x4 o[NCW];
    int slow = 0;
#pragma unroll
    for (int g = 0; g < NCW; ++g) {
      const typename W::Left& left = lds.left[n & 1][g];
      slow |= left.slow << g;
      o[g] = zero4();
      u32x4 u[NO];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        u32x4 sp[NO];
#pragma unroll
        for (int p = 0; p < NO; ++p) sp[p] = left.S[s][p][lane];
        o[g] = mfma_planes<NP, NO, NO>(fq[s], sp, o[g]);
      }
      split_tiles<NO>(left.U[0][lane], left.U[1][lane], u);
#pragma unroll
      for (int r = 0; r < 4; ++r) o[g][r] *= eg[r];
      o[g] = mfma_planes<NO, NO, NO>(fp, u, o[g]);
    }
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(slow), 0)) {
#pragma unroll
      for (int g = 0; g < NCW; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[g][r] = slow >> g & 1 ? lds.left[n & 1][g].y[8 * j + 4 * y + r][c] : o[g][r];
    }
#pragma unroll
    for (int g = 0; g < NCW; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) buf_put<T>(dst, oo[g][r], a.scale * o[g][r]);
  };

  lds_barrier();
  for (int n = n0; n < n1; ++n) {
    if (n > n0) put(n - 1);
    weights(n);
    lds_barrier();
  }
  put(n1 - 1);
}

template <typename T, int KP, bool VEC, int NCW, int MODE>
__device__ inline void walk_body(const WalkArgs& g, char* raw, uint32_t block) {
  typedef Walk<T, KP, VEC, NCW, MODE> W;
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(raw);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // workgroups of one head and segment on one XCD: they share its keys and queries
  const uint32_t heads = (uint32_t)(g.a.B * g.a.Hv);
  const uint32_t run = block / (8 * g.nvb) * 8 + (block & 7);
  const int seg = (int)(run / heads);
  if (seg >= g.walked) return;
  const int64_t bh = run - seg * heads;
  const int n0 = seg * g.per, n1 = n0 + g.per < g.nch ? n0 + g.per : g.nch;
  const int64_t v0 = (int64_t)(block / 8 % g.nvb) * 16 * NCW;
  if (wv < NCW)
    chain<W, NCW, MODE>(g, lds, bh, seg, v0 + 16 * wv + (threadIdx.x & 15), wv, n0, n1);
  else if (MODE != kOutputs || wv >= NCW + 2)
    bring<T, KP, VEC, NCW, MODE>(g, lds, bh, v0, n0, n1);
  else if constexpr (MODE == kOutputs)
    outputs<T, KP, VEC, NCW>(g.a, lds, bh, v0, wv - NCW, n0, n1);
}

template <typename T, int KP, bool VEC, int NCW, int MODE>
__global__ __launch_bounds__((Walk<T, KP, VEC, NCW, MODE>::kThreads),
                             (Walk<T, KP, VEC, NCW, MODE>::kWaves)) void
    delta_walk_kernel(WalkArgs g) {
  extern __shared__ __attribute__((aligned(16))) char raw[];
  walk_body<T, KP, VEC, NCW, MODE>(g, raw, block_of());
}

// Workgroups of a walk (nvb is set), or -1.
template <int KP, int NCW, int MODE>
int64_t walk_wgs(WalkArgs& g) {
  const int64_t cols = MODE == kTransfer ? (g.a.V + 15) / 16 * 16 + KP : g.a.V;
  g.nvb = (uint32_t)cdiv64(cols, 16 * NCW);
  const int64_t wgs = cdiv64(g.a.B * g.a.Hv * g.walked, 8) * 8 * g.nvb;
  return wgs > 0x3fffffff ? -1 : wgs;
}

template <typename T, int KP, bool VEC, int NCW, int MODE>
int walk_launch(WalkArgs& g, hipStream_t s) {
  typedef Walk<T, KP, VEC, NCW, MODE> W;
  const int64_t wgs = walk_wgs<KP, NCW, MODE>(g);
  if (wgs < 0) return TSSM_ERR_UNSUPPORTED;
  constexpr int bytes = (int)sizeof(typename W::Lds);
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  auto* f = delta_walk_kernel<T, KP, VEC, NCW, MODE>;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return (int)e;
  }
  f<<<grid_of(wgs), W::kThreads, bytes, s>>>(g);
  return launch_status();
}

// Two chain waves a workgroup where LDS holds what they leave.
template <typename T, int MODE>
int walk_any(WalkArgs& g, bool vec, hipStream_t s) {
  constexpr int NW = MODE != kOutputs || std::is_same<T, bf16_t>::value ? 2 : 1;
  if (g.a.K <= 32)
    return vec ? walk_launch<T, 32, true, 2, MODE>(g, s) : walk_launch<T, 32, false, 2, MODE>(g, s);
  if (g.a.K <= 64)
    return vec ? walk_launch<T, 64, true, 2, MODE>(g, s) : walk_launch<T, 64, false, 2, MODE>(g, s);
  return vec ? walk_launch<T, 128, true, NW, MODE>(g, s) : walk_launch<T, 128, false, NW, MODE>(g, s);
}

template <int MODE>
int walk_mode(int dtype, WalkArgs& g, bool vec, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return walk_any<float, MODE>(g, vec, s);
    case TSSM_BF16: return walk_any<bf16_t, MODE>(g, vec, s);
    default: return walk_any<f16_t, MODE>(g, vec, s);
  }
}

}  // namespace
}  // namespace tssm
