// Linear attention, chunked: the walk over the chunks.
//
// Per chunk of C steps, with S the state before it, G the sums of g and D[t][i] =
// e^(G_t - G_i) for i <= t, 0 above:
//   O = scale (e^G Q S + (Q K^T D) V),   S' = e^(G_end) S + K^T (e^(G_end - G) V).
// Only S' waits for S, by one product and a sum; all the rest of a chunk is its own.
//
// A workgroup walks 32 columns of V of one head's segment, with C / 16 waves for the
// outputs and as many for the states.  An output wave has 16 steps of the chunk.  A
// state wave brings its share of K and V to LDS and forms K^T V of 32 steps and 16
// columns, all of K, of which it keeps the tiles of the state that are its own and
// hands the others to their owners through LDS.  Everything is formed transposed
// (planes.h): P^T = K Q^T is the next product's operand in place, queries come to
// their wave straight from memory, and a lane ends up with 8 neighbouring columns of
// one step's output.  One barrier a chunk:
//   before it: P and its part of the output | K^T V, the next chunk to LDS,
//   after it: the state's part of the output from planes that the owners left in
//     LDS a chunk ago | the next state and its planes.
// K and V are in LDS twice, a third chunk's loads are in flight.
//
// D of the 32 steps before the wave's own is a product of two factors with the decay
// from that block's end between them: one exponential for a lane and block and a
// table of the chunk's, instead of one for every weight.
//
// Two more forms leave out the outputs: the state at the end of a segment that starts
// from zero, and the states before all chunks (for the gradients).  Walked backwards,
// with queries for keys and dO for V, they give the gradients of the states.
//
// A wave whose own block's output is not finite forms it again without the steps
// after each row: weights of zero would carry a later step's NaN to earlier outputs.
#pragma once

#include "linattn_dev.h"

namespace tssm {
namespace {

enum { kOutputs, kEnds, kStates };

// Sequences are walked in nseg segments of `steps` steps (a multiple of 128); a
// segment's entry state is entry[bh][seg] (a.h0 where there is one segment).
struct LinWalkArgs {
  LinArgs a;           // backwards: q for k, dO for v, dh_last for h0, dh0 for h_last
  int64_t steps;
  int nseg;
  int first, walked;   // the segments that are walked
  int nch, per;        // chunks, chunks of a segment        (the launch sets these)
  uint32_t nvb, units; // blocks of 32 columns; heads times segments walked
  const float* entry;  // [bh][nseg][state]
  float* states;       // kStates: [bh][nch][state]; kEnds: [bh][nseg][state]
  double* sums;        // kEnds: [bh][nseg], of g / log 2
};

template <typename T, int KP, int C, int MODE>
struct LinWalk {
  static constexpr int NP = kPlanes<T>, NO = kOutPlanes<T>;
  static constexpr int NS = KP / 32, KT = KP / 16, NW = C / 16, NT = 64 * NW, NIQ = C / 32;
  static constexpr int OWN = KT / NIQ;       // tiles of the state that a wave keeps
  typedef Swizzled<KP> KR;                   // rows of K and of the state's planes
  typedef Swizzled<32> VR;                   // of V
  // outputs and states have waves of their own
  static constexpr int kThreads = MODE == kOutputs ? 2 * NT : NT;
  static constexpr int kNk = C * KP / 8 / NT;    // 8-element pieces of K a thread brings
  static_assert(KT % NIQ == 0, "every wave owns tiles");
  struct Operands {  // of one chunk
    uint16_t K[NP][C * KP], V[NP][C * 32];
    Decays<C> d;
  };
  struct Lds {
    Operands op[2];
    f32x4 part[2][NW][KT - OWN ? KT - OWN : 1][64];
    // planes of S^T, a row for each column of V
    uint16_t S[MODE == kOutputs ? 2 : 1][NO][MODE == kOutputs ? 32 * KP : 8];
  };
};

// What a workgroup walks.
template <int C>
struct LinUnit {
  int64_t bh, b, h, hk, v0;
  int seg, n0, n1, nv;
  // workgroups of one head's segment, which share Q and K, are on one XCD
  __device__ inline bool init(const LinWalkArgs& g, uint32_t id) {
    const uint32_t vb = (id >> 3) % g.nvb, u = (id >> 3) / g.nvb * 8 + (id & 7);
    if (u >= g.units) return false;
    bh = u / (uint32_t)g.walked;
    seg = g.first + (int)(u - (uint32_t)bh * (uint32_t)g.walked);
    n0 = seg * g.per;
    n1 = n0 + g.per < g.nch ? n0 + g.per : g.nch;
    const LinHead x = lin_head(g.a, (uint32_t)bh);
    b = x.b;
    h = x.h;
    hk = x.hk;
    v0 = (int64_t)vb * 32;
    nv = g.a.V - v0 < 32 ? (int)(g.a.V - v0) : 32;
    return true;
  }
};

// The waves of the states, and of K and V's way to LDS.
template <typename T, int KP, bool VEC, int C, int MODE, bool REV>
__device__ inline void lin_states(const LinWalkArgs& g, const LinUnit<C>& u,
                                  typename LinWalk<T, KP, C, MODE>::Lds& lds, int id) {
  typedef LinWalk<T, KP, C, MODE> W;
  typedef typename W::KR KR;
  typedef typename W::VR VR;
  constexpr int NP = W::NP, NO = W::NO, KT = W::KT, NT = W::NT, NIQ = W::NIQ, OWN = W::OWN,
                kE = (int)sizeof(T);
  const LinArgs& a = g.a;
  const int lane = id & 63, j = lane >> 4, c = lane & 15, cnt = u.n1 - u.n0, K = (int)a.K;
  const int w = __builtin_amdgcn_readfirstlane(id >> 6);
  const int iq = w >> 1, vt = w & 1;         // 32 steps, 16 columns for K^T V
  const int64_t elems = lin_state_elems(KP, a.V), col = u.v0 + 16 * vt + c;
  const int64_t tile0 = ((u.v0 / 16 + vt) * KT + iq * OWN) * 256 + lane * 4;

  RowsOf<C> rk, rv;
  rk.init(reinterpret_cast<const T*>(a.k) + u.b * a.k_b + u.hk * a.k_h, a.k_l, K, a.L);
  rv.init(reinterpret_cast<const T*>(a.v) + u.b * a.v_b + u.h * a.v_h + u.v0, a.v_l, u.nv, a.L);
  const float* gp = a.g + u.b * a.g_b + u.h * a.g_h;
  const auto chunk = [&](int m) {   // the chunk of step m of the walk
    const int x = m < cnt ? m : cnt - 1;
    return REV ? u.n1 - 1 - x : u.n0 + x;
  };
  Piece<T, VEC, NP> ink[W::kNk], inv;
  Gaps<C> gaps;
  const auto fetch = [&](int m) {
    const int n = chunk(m);
    const auto dk = rk.at(n), dv = rv.at(n);
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = id + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      ink[i].load(dk, x < K ? r * rk.row + x * kE : kPast);
    }
    const int r = id >> 2, x = (id & 3) * 8;
    inv.load(dv, x < u.nv ? r * rv.row + x * kE : kPast);
    if (w == 0) {
      const int64_t t0 = (int64_t)n * C, rest = a.L - t0;
      gaps.load(gp + t0 * a.g_l, a.g_l, lane, rest < C ? (int)rest : C);
    }
  };
  const auto leave = [&](typename W::Operands& o) {  // what fetch() brought, to LDS
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = id + NT * i, r = at / (KP / 8), x = at % (KP / 8);
      u32x4 p[NP];
      planes_apart(ink[i], K - 8 * x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&o.K[y][KR::at(r, x)]) = p[y];
    }
    const int r = id >> 2, x = id & 3;
    u32x4 p[NP];
    planes_apart(inv, u.nv - 8 * x, p);
#pragma unroll
    for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&o.V[y][VR::at(r, x)]) = p[y];
    if (w == 0) gaps.decays(o.d, lane);
  };
  f32x4 S[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    if constexpr (MODE == kEnds) S[i] = zero4();
    else if (g.nseg == 1)
      S[i] = get_tile(a.h0 ? a.h0 + u.bh * K * a.V : nullptr, iq * OWN + i, col, a.V, K, j);
    else
      S[i] = *reinterpret_cast<const f32x4*>(g.entry + (u.bh * g.nseg + u.seg) * elems + tile0 +
                                             256 * i);
  }
  const auto show = [&](int par) {  // the state's planes, for the outputs
    if constexpr (MODE == kOutputs) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int kt = iq * OWN + i;
        float x0 = S[i][0], x1 = S[i][1], x2 = S[i][2], x3 = S[i][3];
#pragma unroll
        for (int p = 0; p < NO; ++p) {
          const uint32_t lo = pk_bf16(x0, x1), hi = pk_bf16(x2, x3);
          *reinterpret_cast<uint2*>(&lds.S[par][p][KR::at(16 * vt + c, 4 * (kt >> 1) + j) +
                                                   4 * (kt & 1)]) = make_uint2(lo, hi);
          if (p + 1 < NO) {
            take_plane(lo, x0, x1);
            take_plane(hi, x2, x3);
          }
        }
      }
    }
  };
  double total = 0.0;
  fetch(0);
  leave(lds.op[0]);
  show(0);
  fetch(1);
  lds_barrier();
  for (int m = 0; m < cnt; ++m) {
    const int par = m & 1;
    const typename W::Operands& B = lds.op[par];
    const float hend = B.d.hi[C - 1], lend = B.d.lo[C - 1];
    const float last = exp2_fast(hend + lend);
    if constexpr (MODE == kEnds) total += (double)hend + (double)lend;
    // this wave's 32 steps of K^T V
    float v8[8], e8[8];
    lds_values<NP, 32>(&B.V[0][0], C * 32, 32 * iq, 16 * vt, lane, v8);
    if constexpr (REV) {
      float h8[8], l8[8];
      lds8(&B.d.hi[32 * iq + 8 * j], h8);
      lds8(&B.d.lo[32 * iq + 8 * j], l8);
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = a.scale * exp2_fast(h8[e] + l8[e]);
    } else {
      lds8(&B.d.u[32 * iq + 8 * j], e8);
      const float from = diff2(hend, lend, B.d.hi[32 * iq + 31], B.d.lo[32 * iq + 31]);
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] *= from;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v8[e] *= e8[e];
    u32x4 vp[3];
    split8<3>(v8, vp);
    f32x4 mine[OWN];
#pragma unroll
    for (int o = 0; o < NIQ; ++o) {  // the tiles of this wave, then of the others
      const int other = (iq + o) % NIQ;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int kt = other * OWN + i;
        u32x4 fk[NP];
#pragma unroll
        for (int y = 0; y < NP; ++y)
          fk[y] = KR::col(B.K[y], 32 * iq, 32 * (kt >> 1) + 4 * (kt & 1), lane);
        const f32x4 x = mfma_planes<NP, 3, 3>(fk, vp, zero4());
        if (o == 0) mine[i] = x;
        else lds.part[par][w][other < iq ? kt : kt - OWN][lane] = x;
      }
    }
    leave(lds.op[par ^ 1]);
    fetch(m + 2);
    lds_barrier();
    if constexpr (MODE == kStates) {
      float* p = g.states + (u.bh * g.nch + chunk(m)) * elems + tile0;
#pragma unroll
      for (int i = 0; i < OWN; ++i) *reinterpret_cast<f32x4*>(p + 256 * i) = S[i];
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      f32x4 x = mine[i];
#pragma unroll
      for (int o = 1; o < NIQ; ++o) {
        const int other = (iq + o) % NIQ, kt = iq * OWN + i;
        x += lds.part[par][2 * other + vt][iq < other ? kt : kt - OWN][lane];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) S[i][r] = __builtin_fmaf(S[i][r], last, x[r]);
    }
    show(par ^ 1);
  }
  if constexpr (MODE == kEnds) {
    float* p = g.states + (u.bh * g.nseg + u.seg) * elems + tile0;
#pragma unroll
    for (int i = 0; i < OWN; ++i) *reinterpret_cast<f32x4*>(p + 256 * i) = S[i];
    if (u.v0 == 0 && id == 0) g.sums[u.bh * g.nseg + u.seg] = total;
  } else if (REV ? u.n0 == 0 : u.n1 == g.nch) {
    float* p = a.h_last ? a.h_last + u.bh * K * a.V : nullptr;
#pragma unroll
    for (int i = 0; i < OWN; ++i) put_tile(p, S[i], iq * OWN + i, col, a.V, K, j);
  }
}

// The waves of the outputs.
template <typename T, int KP, bool VEC, int C>
__device__ inline void lin_outputs(const LinWalkArgs& g, const LinUnit<C>& u,
                                   typename LinWalk<T, KP, C, kOutputs>::Lds& lds, int id) {
  typedef LinWalk<T, KP, C, kOutputs> W;
  typedef typename W::KR KR;
  typedef typename W::VR VR;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, kE = (int)sizeof(T);
  const LinArgs& a = g.a;
  const int lane = id & 63, j = lane >> 4, c = lane & 15, cnt = u.n1 - u.n0, K = (int)a.K;
  const int w = __builtin_amdgcn_readfirstlane(id >> 6);
  // 16 steps: waves w and w + 4, on one SIMD, have equal work together
  const int tw = C == 128 && w >= 4 ? 11 - w : w, db = tw >> 1, t = 16 * tw + c;
  const int ar = 8 * (c >> 2) + (c & 3);     // row of tile x of an A operand, less 4 x
  RowsOf<C> rq, ro;
  rq.init(reinterpret_cast<const T*>(a.q) + u.b * a.q_b + u.hk * a.q_h, a.q_l, K, a.L);
  ro.init(reinterpret_cast<const T*>(a.o) + u.b * a.o_b + u.h * a.o_h + u.v0, a.o_l, u.nv, a.L);
  Piece<T, VEC, NP> in[NS];
  const auto fetch = [&](int m) {
    const auto d = rq.at(u.n0 + (m < cnt ? m : cnt - 1));
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int y = 32 * s + 8 * j;
      in[s].load(d, y < K ? t * rq.row + y * kE : kPast);
    }
  };
  fetch(0);
  lds_barrier();
  for (int m = 0; m < cnt; ++m) {
    const int par = m & 1;
    const typename W::Operands& B = lds.op[par];
    u32x4 qb[NS][NP];
#pragma unroll
    for (int s = 0; s < NS; ++s) in[s].planes(K - 32 * s - 8 * j, qb[s]);
    fetch(m + 1);
    f32x4 acc[2] = {zero4(), zero4()}, own[2] = {zero4(), zero4()};
    const float ht = B.d.hi[t], lt = B.d.lo[t], eg = exp2_fast(ht + lt);
    float p8[8];  // of the last block, the wave's own
    // NB blocks of 32 steps, in one piece so that they overlap; the last is masked
    const auto blocks = [&](auto count) {
      constexpr int NB = decltype(count)::value;
      f32x4 p[NB][2];
      float from[NB];
#pragma unroll
      for (int ib = 0; ib < NB; ++ib) {
        from[ib] = diff2(ht, lt, B.d.hi[32 * ib + 31], B.d.lo[32 * ib + 31]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          p[ib][x] = zero4();
#pragma unroll
          for (int s = 0; s < NS; ++s) {  // rows i = 32 ib + 8 j + 4 x + r of K Q^T
            u32x4 fk[NP];
#pragma unroll
            for (int y = 0; y < NP; ++y)
              fk[y] = lds16(&B.K[y][KR::at(ar, 4 * s + j) + (32 * ib + 4 * x) * KP]);
            p[ib][x] = mfma_planes<NP, NP, NO>(fk, qb[s], p[ib][x]);
          }
        }
      }
#pragma unroll
      for (int ib = 0; ib < NB; ++ib) {
        if (ib + 1 < NB) {
          float u8[8];
          lds8(&B.d.u[32 * ib + 8 * j], u8);
#pragma unroll
          for (int e = 0; e < 8; ++e) p8[e] = p[ib][e >> 2][e & 3] * (u8[e] * from[ib]);
        } else {
          float h8[8], l8[8];
          lds8(&B.d.hi[32 * ib + 8 * j], h8);
          lds8(&B.d.lo[32 * ib + 8 * j], l8);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p8[e] = 32 * ib + 8 * j + e <= t
                        ? p[ib][e >> 2][e & 3] * diff2(ht, lt, h8[e], l8[e]) : 0.0f;
        }
        u32x4 pb[NO];
        split8<NO>(p8, pb);
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // V^T P^T
          u32x4 fv[NP];
#pragma unroll
          for (int y = 0; y < NP; ++y) fv[y] = VR::col(B.V[y], 32 * ib, 4 * x, lane);
          f32x4& o = ib + 1 < NB ? acc[x] : own[x];
          o = mfma_planes<NP, NO, NO>(fv, pb, o);
        }
      }
    };
    if (C == 32 || db == 0) blocks(std::integral_constant<int, 1>());
    else if (C == 64 || db == 1) blocks(std::integral_constant<int, 2>());
    else if (db == 2) blocks(std::integral_constant<int, 3>());
    else blocks(std::integral_constant<int, 4>());
    float big = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) big += __builtin_fabsf(own[e >> 2][e & 3]);
    if (__builtin_expect(__ballot(!(big < __builtin_inff())) != 0, 0)) {
      own[0] = own[1] = zero4();
#pragma unroll 1
      for (int i = 0; i < 32; ++i) {
        float p = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) p = (i & 7) == e ? p8[e] : p;
        p = __shfl(p, (i >> 3) * 16 + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = 0.0f;
#pragma unroll
          for (int y = NP - 1; y >= 0; --y)
            v += bf16_bits_to_f32(B.V[y][VR::at(32 * db + i, j) + e]);
          if (32 * db + i <= t) own[e >> 2][e & 3] += p * v;
        }
      }
    }
    lds_barrier();
    f32x4 y[2] = {zero4(), zero4()};
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4 fs[NO];
#pragma unroll
        for (int p = 0; p < NO; ++p)
          fs[p] = lds16(&lds.S[par][p][KR::at(ar, 4 * s + j) + 4 * x * KP]);
        y[x] = mfma_planes<NO, NP, NO>(fs, qb[s], y[x]);
      }
    const auto dst = ro.at(u.n0 + m);
    const uint32_t off = (uint32_t)(t * ro.row + 8 * j * kE);
    float o8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      o8[e] = a.scale * __builtin_fmaf(y[e >> 2][e & 3], eg,
                                       acc[e >> 2][e & 3] + own[e >> 2][e & 3]);
    if constexpr (VEC) {
      const uint32_t to = 8 * j < u.nv ? off : kPast;
      union {
        T e[8];
        u32x4 v[kE / 2];
      } x;
#pragma unroll
      for (int e = 0; e < 8; ++e) stf(&x.e[e], o8[e]);
#pragma unroll
      for (int i = 0; i < kE / 2; ++i)
        __builtin_amdgcn_raw_buffer_store_b128(x.v[i], dst, to + 16 * i, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        buf_put<T>(dst, 8 * j + e < u.nv ? off + e * kE : kPast, o8[e]);
    }
  }
}

// Steps of a chunk: as many as LDS holds (two chunks of K's planes).  The gradients'
// kernel asks for chunks of its own.
template <typename T, int KP>
constexpr int kWalkSteps = kPlanes<T> == 1 && KP == 64 ? 128
                           : (kPlanes<T> == 3 && KP == 128 ? 32 : 64);
template <typename T, int KP>
constexpr int kStateSteps = kPlanes<T> == 3 && KP == 128 ? 32 : 64;

template <typename T, int KP, bool VEC>
__global__ __launch_bounds__((8 * kWalkSteps<T, KP>)) void lin_walk_kernel(LinWalkArgs g) {
  constexpr int C = kWalkSteps<T, KP>;
  typedef LinWalk<T, KP, C, kOutputs> W;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  LinUnit<C> u;
  if (!u.init(g, block_of())) return;
  const int id = (int)threadIdx.x;
  if (id < W::NT) lin_outputs<T, KP, VEC, C>(g, u, lds, id);
  else lin_states<T, KP, VEC, C, kOutputs, false>(g, u, lds, id - W::NT);
}

// The states' walk and its way back, side by side: the first nf workgroups go forward.
template <typename T, int KP, bool VEC, int MODE>
__global__ __launch_bounds__((4 * kStateSteps<T, KP>)) void lin_states_kernel(LinWalkArgs f,
                                                                              LinWalkArgs back,
                                                                              uint32_t nf) {
  constexpr int C = kStateSteps<T, KP>;
  typedef LinWalk<T, KP, C, MODE> W;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  const uint32_t id = block_of();
  LinUnit<C> u;
  if (id < nf) {
    if (u.init(f, id)) lin_states<T, KP, VEC, C, MODE, false>(f, u, lds, (int)threadIdx.x);
  } else {
    if (u.init(back, id - nf)) lin_states<T, KP, VEC, C, MODE, true>(back, u, lds, (int)threadIdx.x);
  }
}

// Sizes that a launch sets; returns its workgroups, or -1.
inline int64_t lin_walk_sizes(LinWalkArgs& g, int C) {
  g.nvb = (uint32_t)cdiv64(g.a.V, 32);
  g.nch = (int)cdiv64(g.a.L, C);
  g.per = (int)cdiv64(g.steps, C);
  const int64_t units = g.a.B * g.a.Hv * g.walked, wgs = cdiv64(units, 8) * 8 * g.nvb;
  if (wgs > 0x3fffffff) return -1;
  g.units = (uint32_t)units;
  return wgs;
}

template <typename K>
int lin_lds(K kernel, int bytes) {
  return bytes <= 65536 ? TSSM_OK
                        : (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize,
                                                   bytes);
}

template <typename T, int KP, bool VEC>
int lin_walk_run(LinWalkArgs g, hipStream_t s) {
  typedef LinWalk<T, KP, kWalkSteps<T, KP>, kOutputs> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t wgs = lin_walk_sizes(g, kWalkSteps<T, KP>);
  if (wgs < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_walk_kernel<T, KP, VEC>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(wgs), W::kThreads, sizeof(typename W::Lds), s>>>(g);
  return launch_status();
}

// back.walked = 0: forward alone.
template <typename T, int KP, bool VEC, int MODE>
int lin_states_run(LinWalkArgs f, LinWalkArgs back, hipStream_t s) {
  typedef LinWalk<T, KP, kStateSteps<T, KP>, MODE> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t nf = lin_walk_sizes(f, kStateSteps<T, KP>);
  const int64_t nb = lin_walk_sizes(back, kStateSteps<T, KP>);
  if (nf < 0 || nb < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_states_kernel<T, KP, VEC, MODE>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(nf + nb), W::kThreads, sizeof(typename W::Lds), s>>>(f, back, (uint32_t)nf);
  return launch_status();
}

}  // namespace
}  // namespace tssm
