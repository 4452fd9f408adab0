// Linear attention, chunked: the walk over the chunks.
//
// Per chunk of C steps, with S the state before it, G the sums of g and D[t][i] =
// e^(G_t - G_i) for i <= t, 0 above:
//   O = scale (e^G Q S + (Q K^T D) V),   S' = e^(G_end) S + K^T (e^(G_end - G) V).
// Only S' waits for S, by one product and a sum; all the rest of a chunk is its own.
//
// A workgroup walks 32 columns of V of one head's segment.  Its waves have roles, one
// barrier a chunk:
//   two teams of C / 32 output waves: 32 steps of a chunk each, as two tiles of 16.  A
//     team has every other chunk, and two chunks' time for it.  (Where LDS does not hold
//     three chunks, one team with a wave for each tile: 128 x 128 fp32, B=2 L=2048 H=16,
//     114 us a call; 237 with one wave for both tiles of 32 steps.)
//   2 state waves: 16 columns each.  K^T V of the whole chunk on top of the decayed
//     state, whose planes go to LDS for the next chunk's outputs,
//   2 loaders (4 beside two output waves): the chunk after this one to LDS, from loads
//     that are two chunks ahead; where there are no outputs also a wave for the decays
//     (which beside four output waves would be a third wave on a SIMD and take a third of
//     the others' registers: B=3 L=1111 12 heads 40 x 72 fp32 46 -> 88 us).
// Everything is formed transposed (planes.h): P^T = K Q^T is the next product's operand
// in place, queries come to their wave straight from memory, and a lane ends up with 8
// neighbouring columns of one step's output.
//
// What bounds it: one wave's chain and LDS.  B=8 L=4096 H=16 64 x 64 bf16 takes 85 us
// for 270 MB (3.2 TB/s; 256 workgroups, one on a CU), a chunk of 128 steps 3800 cycles,
// of which the state waves work 3200, the outputs 2400 to 3100 and the loader with the
// decays 3000.  fp32 (3 planes) is bound by LDS: 3700 of a chunk's 5000 cycles (64
// steps, K = 64).  LDS takes 16 cycles for a 16-byte read, so an operand that is read
// should serve as many products as it can: the two tiles of an output wave share K, V
// and the state's planes (with a wave for each tile 90 us), and a state wave that has
// all steps of its columns needs no exchange.  In a chunk of 128 the tiles are dealt so
// that an output wave beside a state wave on its SIMD has 2 blocks of K and one beside a
// loader 4, for what is left of the SIMD's time.
//
// D of the 32 steps before a tile's own is a product of two factors with the decay from
// that block's end between them: one exponential for a lane and block and a table of
// the chunk's, instead of one for every weight.
//
// Two more forms leave out the outputs: the state at the end of a segment that starts
// from zero, and the states before all chunks (for the gradients).  Walked backwards,
// with queries for keys and dO for V, they give the gradients of the states.
//
// A tile whose own block's output is not finite forms it again without the steps after
// each row: weights of zero would carry a later step's NaN to earlier outputs.
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

// Teams of output waves, and steps of a chunk, by what LDS holds (a chunk more of K's and
// the state's planes than there are teams).  128 x 128 fp16 would fit two teams of 32
// steps: 51 against 47 us (B=2 L=2000 16 heads); 128 x 128 bf16 a chunk of 128 for one: 89
// against 51 a call (B=2 L=2048 H=16).
constexpr int lin_teams(int NP, int KP) { return NP * KP <= 192 ? 2 : 1; }
template <typename T, int KP>
constexpr int kWalkSteps = kPlanes<T> * KP <= 64 ? 128 : (kPlanes<T> * KP <= 256 ? 64 : 32);

template <typename T, int KP, int C, int MODE>
struct LinWalk {
  static constexpr int NP = kPlanes<T>, NO = kOutPlanes<T>;
  static constexpr int NS = KP / 32, KT = KP / 16, NB = C / 32;
  static constexpr int TEAMS = MODE == kOutputs ? lin_teams(NP, KP) : 1, RING = TEAMS + 1;
  // output waves: of two tiles of 16 steps, or one where there is one team
  static constexpr int NW = MODE == kOutputs ? (TEAMS == 1 ? C / 16 : TEAMS * C / 32) : 0;
  static constexpr int NT = NW == 2 && TEAMS == 1 ? 256 : 128;  // threads of the loaders
  static constexpr bool CLOCK = NW == 0;                    // a wave for the decays
  static constexpr int kThreads = 64 * (NW + 2 + CLOCK) + NT;
  static constexpr int kNk = (C * KP / 8 + NT - 1) / NT, kNv = (C * 4 + NT - 1) / NT;
  static constexpr int AHEAD = 2;            // chunks on their way from memory
  typedef Swizzled<KP> KR;                   // rows of K and of the state's planes
  typedef Swizzled<32> VR;                   // of V
  struct Operands {  // of one chunk
    uint16_t K[NP][C * KP], V[NP][C * 32];
    Decays<C> d;
  };
  struct Lds {
    Operands op[RING];
    // planes of S^T, a row for each column of V
    uint16_t S[MODE == kOutputs ? RING : 1][NO][MODE == kOutputs ? 32 * KP : 8];
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

// The chunk of step m of a walk.
template <int C, bool REV>
__device__ inline int lin_chunk(const LinUnit<C>& u, int m) {
  const int cnt = u.n1 - u.n0, x = m < cnt ? m : cnt - 1;
  return REV ? u.n1 - 1 - x : u.n0 + x;
}

// K's, V's and the decays' way to LDS.
template <typename T, int KP, LinRows ROWS, int C, int MODE, bool REV>
__device__ inline void lin_bring(const LinWalkArgs& g, const LinUnit<C>& u,
                                 typename LinWalk<T, KP, C, MODE>::Lds& lds, int id) {
  typedef LinWalk<T, KP, C, MODE> W;
  constexpr int NP = W::NP, NT = W::NT, kE = (int)sizeof(T), U = KP / 8;
  const LinArgs& a = g.a;
  const int lane = id & 63, cnt = u.n1 - u.n0, K = (int)a.K;
  const int wave = __builtin_amdgcn_readfirstlane(id >> 6);
  const bool clock = wave == (W::CLOCK ? NT / 64 : 0), rows = wave < NT / 64;
  RowsOf<C> rk, rv;
  rk.init(reinterpret_cast<const T*>(a.k) + u.b * a.k_b + u.hk * a.k_h, a.k_l, K, a.L);
  rv.init(reinterpret_cast<const T*>(a.v) + u.b * a.v_b + u.h * a.v_h + u.v0, a.v_l, u.nv, a.L);
  const float* gp = a.g + u.b * a.g_b + u.h * a.g_h;
  struct Regs {
    Piece<T, ROWS != kNoRows, NP> k[W::kNk];
    Piece<T, ROWS == kAllRows, NP> v[W::kNv];
    Gaps<C> g;
  } in[W::AHEAD];
  const auto fetch = [&](Regs& in, int m) {
    const int n = lin_chunk<C, REV>(u, m);
    if (rows) {
      const auto dk = rk.at(n), dv = rv.at(n);
#pragma unroll
      for (int i = 0; i < W::kNk; ++i) {
        const int at = id + NT * i, r = at / U, x = at % U * 8;
        in.k[i].load(dk, r < C && x < K ? r * rk.row + x * kE : kPast);
      }
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) {
        const int at = id + NT * i, r = at >> 2, x = (at & 3) * 8;
        in.v[i].load(dv, r < C && x < u.nv ? r * rv.row + x * kE : kPast);
      }
    }
    if (clock) {
      const int64_t t0 = (int64_t)n * C, rest = a.L - t0;
      in.g.load(gp + t0 * a.g_l, a.g_l, lane, rest < C ? (int)rest : C);
    }
  };
  const auto leave = [&](const Regs& in, typename W::Operands& o) {
    if (rows) {
#pragma unroll
      for (int i = 0; i < W::kNk; ++i) {
        const int at = id + NT * i, r = at / U, x = at % U;
        u32x4 p[NP];
        planes_apart(in.k[i], K - 8 * x, p);
        if (C * U % NT == 0 || r < C) {
#pragma unroll
          for (int y = 0; y < NP; ++y)
            *reinterpret_cast<u32x4*>(&o.K[y][W::KR::at(r, x)]) = p[y];
        }
      }
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) {
        const int at = id + NT * i, r = at >> 2, x = at & 3;
        u32x4 p[NP];
        planes_apart(in.v[i], u.nv - 8 * x, p);
        if (C * 4 % NT == 0 || r < C) {
#pragma unroll
          for (int y = 0; y < NP; ++y)
            *reinterpret_cast<u32x4*>(&o.V[y][W::VR::at(r, x)]) = p[y];
        }
      }
    }
    if (clock) in.g.template decays<REV>(o.d, lane, a.scale);
  };
#pragma unroll
  for (int i = 0; i < W::AHEAD; ++i) fetch(in[i], i);
  leave(in[0], lds.op[0]);
  fetch(in[0], W::AHEAD);
  lds_barrier();
  int slot = 1;
  const auto turn = [&](int m, Regs& x) {  // x holds chunk m + 1
    leave(x, lds.op[slot]);
    slot = slot + 1 < W::RING ? slot + 1 : 0;
    fetch(x, m + 1 + W::AHEAD);
    lds_barrier();
  };
  for (int m = 0; m < cnt; m += W::AHEAD) {
#pragma unroll
    for (int i = 0; i < W::AHEAD; ++i)
      if (m + i < cnt) turn(m + i, in[(i + 1) % W::AHEAD]);
  }
  if constexpr (W::TEAMS == 2) lds_barrier();
}

// The states' waves: vt, 16 columns.
template <typename T, int KP, int C, int MODE, bool REV>
__device__ inline void lin_states(const LinWalkArgs& g, const LinUnit<C>& u,
                                  typename LinWalk<T, KP, C, MODE>::Lds& lds, int lane, int vt) {
  typedef LinWalk<T, KP, C, MODE> W;
  typedef typename W::KR KR;
  constexpr int NP = W::NP, NO = W::NO, KT = W::KT, NB = W::NB;
  const LinArgs& a = g.a;
  const int j = lane >> 4, c = lane & 15, cnt = u.n1 - u.n0, K = (int)a.K;
  const int64_t elems = lin_state_elems(KP, a.V), col = u.v0 + 16 * vt + c;
  const int64_t tile0 = (u.v0 / 16 + vt) * KT * 256 + lane * 4;
  f32x4 S[KT];
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    if constexpr (MODE == kEnds) S[i] = zero4();
    else if (g.nseg == 1)
      S[i] = get_tile(a.h0 ? a.h0 + u.bh * K * a.V : nullptr, i, col, a.V, K, j);
    else
      S[i] = *reinterpret_cast<const f32x4*>(g.entry + (u.bh * g.nseg + u.seg) * elems + tile0 +
                                             256 * i);
  }
  const auto show = [&](int slot) {  // the state's planes, for the outputs
    if constexpr (MODE == kOutputs) {
#pragma unroll
      for (int s = 0; s < KT / 2; ++s) {
        u32x4 p[NO];
        split_tiles<NO>(S[2 * s], S[2 * s + 1], p);
#pragma unroll
        for (int y = 0; y < NO; ++y)
          *reinterpret_cast<u32x4*>(&lds.S[slot][y][KR::at(16 * vt + c, 4 * s + j)]) = p[y];
      }
    }
  };
  double total = 0.0;
  int slot = 0;
  show(0);
  __builtin_amdgcn_s_setprio(3);  // the outputs have two chunks' time, this chain one
  lds_barrier();
  for (int m = 0; m < cnt; ++m) {
    const typename W::Operands& B = lds.op[slot];
    const float hend = B.d.hi[C - 1], lend = B.d.lo[C - 1];
    const float last = exp2_fast(hend + lend);
    if constexpr (MODE == kEnds) total += (double)hend + (double)lend;
    if constexpr (MODE == kStates) {
      float* p = g.states + (u.bh * g.nch + lin_chunk<C, REV>(u, m)) * elems + tile0;
#pragma unroll
      for (int i = 0; i < KT; ++i) *reinterpret_cast<f32x4*>(p + 256 * i) = S[i];
    }
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[i][r] *= last;
    // operands asked for a block ahead: waited for, they would be a third of the time
    float w1[2];
    u32x4 fk[2][KT][NP], fv[2][NP];
    const auto ask = [&](int ib) {
#pragma unroll
      for (int y = 0; y < NP; ++y)
        fv[ib & 1][y] = Swizzled<32>::col16(B.V[y], 32 * ib, 16 * vt, lane);
      w1[ib & 1] = one_of8(&B.d.w[32 * ib], lane);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int y = 0; y < NP; ++y)
          fk[ib & 1][kt][y] = KR::col(B.K[y], 32 * ib, 32 * (kt >> 1) + 4 * (kt & 1), lane);
    };
    ask(0);
#pragma unroll
    for (int ib = 0; ib < NB; ++ib) {
      if (ib + 1 < NB) ask(ib + 1);
      __builtin_amdgcn_sched_barrier(0);
      float v8[8], w8[8];
      operand_values<NP>(fv[ib & 1], v8);
      eight(w1[ib & 1], w8);
#pragma unroll
      for (int e = 0; e < 8; ++e) v8[e] *= w8[e];
      u32x4 vp[3];
      split8<3>(v8, vp);
      // (tiles within planes: a tile's products wait for each other)
#pragma unroll
      for (int x = 0; x < NP; ++x)
#pragma unroll
        for (int y = 0; y + x < 3; ++y)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) S[kt] = mfma32(fk[ib & 1][kt][x], vp[y], S[kt]);
    }
    slot = slot + 1 < W::RING ? slot + 1 : 0;
    show(slot);
    lds_barrier();
  }
  if constexpr (W::TEAMS == 2) lds_barrier();
  if constexpr (MODE == kEnds) {
    float* p = g.states + (u.bh * g.nseg + u.seg) * elems + tile0;
#pragma unroll
    for (int i = 0; i < KT; ++i) *reinterpret_cast<f32x4*>(p + 256 * i) = S[i];
    if (u.v0 == 0 && vt == 0 && lane == 0) g.sums[u.bh * g.nseg + u.seg] = total;
  } else if (REV ? u.n0 == 0 : u.n1 == g.nch) {
    float* p = a.h_last ? a.h_last + u.bh * K * a.V : nullptr;
#pragma unroll
    for (int i = 0; i < KT; ++i) put_tile(p, S[i], i, col, a.V, K, j);
  }
}

// The outputs' waves: tiles of 16 steps, at 16 tile[i], whose own blocks of 32 steps are OWN.
template <typename T, int KP, LinRows ROWS, int C, int... OWN>
__device__ inline void lin_outputs(const LinWalkArgs& g, const LinUnit<C>& u,
                                   typename LinWalk<T, KP, C, kOutputs>::Lds& lds, int lane,
                                   const int (&tile)[sizeof...(OWN)], int team) {
  typedef LinWalk<T, KP, C, kOutputs> W;
  typedef typename W::KR KR;
  typedef typename W::VR VR;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, TEAMS = W::TEAMS, kE = (int)sizeof(T);
  constexpr int NI = sizeof...(OWN), kOwn[NI] = {OWN...}, LB = kOwn[NI - 1];  // the last is latest
  const LinArgs& a = g.a;
  const int j = lane >> 4, c = lane & 15, cnt = u.n1 - u.n0, K = (int)a.K;
  int t[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) t[i] = 16 * tile[i] + c;
  const int ar = 8 * (c >> 2) + (c & 3);     // row of tile x of an A operand, less 4 x
  RowsOf<C> rq, ro;
  rq.init(reinterpret_cast<const T*>(a.q) + u.b * a.q_b + u.hk * a.q_h, a.q_l, K, a.L);
  ro.init(reinterpret_cast<const T*>(a.o) + u.b * a.o_b + u.h * a.o_h + u.v0, a.o_l, u.nv, a.L);
  Piece<T, ROWS != kNoRows, NP> in[NI][NS];
  const auto fetch = [&](int m) {
    const auto d = rq.at(lin_chunk<C, false>(u, m));
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int y = 32 * s + 8 * j;
        in[i][s].load(d, y < K ? t[i] * rq.row + y * kE : kPast);
      }
  };
  u32x4 qb[NI][NS][NP];
  const auto queries = [&](int m) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s) planes_apart(in[i][s], K - 32 * s - 8 * j, qb[i][s]);
    fetch(m + TEAMS);
  };
  fetch(team);
  lds_barrier();
  if (team) lds_barrier();
  int slot = team;
  for (int m = team; m < cnt; m += TEAMS) {
    const typename W::Operands& B = lds.op[slot];
    const auto& Sp = lds.S[slot];
    slot = slot + TEAMS < W::RING ? slot + TEAMS : slot + TEAMS - W::RING;
    u32x4 fk[2][NS][NP], fv[2][NP];
    float u1, h1, l1, ht[NI], lt[NI];
    const auto keys = [&](int ib) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < NP; ++y)
            fk[x][s][y] = lds16(&B.K[y][KR::at(ar, 4 * s + j) + (32 * ib + 4 * x) * KP]);
    };
    const auto decays = [&](int ib) {
      if (ib < LB) u1 = one_of8(&B.d.u[32 * ib], lane);
      if (((ib == OWN) || ...)) {
        h1 = one_of8(&B.d.hi[32 * ib], lane);
        l1 = one_of8(&B.d.lo[32 * ib], lane);
      }
    };
    const auto values = [&](int ib) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < NP; ++y) fv[x][y] = VR::col(B.V[y], 32 * ib, 4 * x, lane);
    };
    // Operands are asked for a product ahead: read where they are used, each would
    // wait for LDS.
    keys(0);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      ht[i] = B.d.hi[t[i]];
      lt[i] = B.d.lo[t[i]];
    }
    decays(0);
    values(0);
    queries(m);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 acc[NI][2], own[2];
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[i][0] = acc[i][1] = zero4();
#pragma unroll
    for (int ib = 0; ib <= LB; ++ib) {
      f32x4 p[NI][2];  // rows i = 32 ib + 8 j + 4 x + r of K Q^T
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (ib > kOwn[i]) continue;
        p[i][0] = p[i][1] = zero4();
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            p[i][x] = mfma_planes<NP, NP, NO>(fk[x][s], qb[i][s], p[i][x]);
      }
      if (ib < LB) keys(ib + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if (ib > kOwn[i]) continue;
        float w8[8];
        if (ib < kOwn[i]) {
          const float from = diff2(ht[i], lt[i], B.d.hi[32 * ib + 31], B.d.lo[32 * ib + 31]);
          float u8[8];
          eight(u1, u8);
#pragma unroll
          for (int e = 0; e < 8; ++e) w8[e] = p[i][e >> 2][e & 3] * (u8[e] * from);
        } else {
          float h8[8], l8[8];
          eight(h1, h8);
          eight(l1, l8);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float y = p[i][e >> 2][e & 3] * diff2(ht[i], lt[i], h8[e], l8[e]);
            asm("" : "+v"(y));  // formed for all, then chosen: no branch
            w8[e] = 32 * ib + 8 * j + e <= t[i] ? y : 0.0f;
          }
        }
        u32x4 pb[NO];
        split8<NO>(w8, pb);
        if (ib < kOwn[i]) {
#pragma unroll
          for (int x = 0; x < 2; ++x)  // V^T P^T
            acc[i][x] = mfma_planes<NP, NO, NO>(fv[x], pb, acc[i][x]);
          continue;
        }
        float big = 0.0f;
#pragma unroll
        for (int x = 0; x < 2; ++x) own[x] = mfma_planes<NP, NO, NO>(fv[x], pb, zero4());
#pragma unroll
        for (int e = 0; e < 8; ++e) big += __builtin_fabsf(own[e >> 2][e & 3]);
        if (__builtin_expect(__ballot(!(big < __builtin_inff())) != 0, 0)) {
          own[0] = own[1] = zero4();
#pragma unroll 1
          for (int n = 0; n < 32; ++n) {
            float w = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) w = (n & 7) == e ? w8[e] : w;
            w = __shfl(w, (n >> 3) * 16 + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float v = 0.0f;
#pragma unroll
              for (int y = NP - 1; y >= 0; --y)
                v += bf16_bits_to_f32(B.V[y][VR::at(32 * ib + n, j) + e]);
              if (32 * ib + n <= t[i]) own[e >> 2][e & 3] += w * v;
            }
          }
        }
        acc[i][0] += own[0];
        acc[i][1] += own[1];
      }
      if (ib < LB) {
        decays(ib + 1);
        values(ib + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      // half of the work: the rest while the other team has its first half
      if (TEAMS == 2 && ib == LB / 2) lds_barrier();
    }
    // the state's part
    u32x4 fs[NS][2][NO];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int p = 0; p < NO; ++p)
          fs[s][x][p] = lds16(&Sp[p][KR::at(ar, 4 * s + j) + 4 * x * KP]);
    const auto dst = ro.at(u.n0 + m);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      f32x4 y[2] = {zero4(), zero4()};
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) y[x] = mfma_planes<NO, NP, NO>(fs[s][x], qb[i][s], y[x]);
      const float eg = exp2_fast(ht[i] + lt[i]);
      const uint32_t off = (uint32_t)(t[i] * ro.row + 8 * j * kE);
      float o8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o8[e] = a.scale * __builtin_fmaf(y[e >> 2][e & 3], eg, acc[i][e >> 2][e & 3]);
      if constexpr (ROWS == kAllRows) {
        const uint32_t to = 8 * j < u.nv ? off : kPast;
        union {
          T e[8];
          u32x4 v[kE / 2];
        } x;
#pragma unroll
        for (int e = 0; e < 8; ++e) stf(&x.e[e], o8[e]);
#pragma unroll
        for (int n = 0; n < kE / 2; ++n)
          __builtin_amdgcn_raw_buffer_store_b128(x.v[n], dst, to + 16 * n, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          buf_put<T>(dst, 8 * j + e < u.nv ? off + e * kE : kPast, o8[e]);
      }
    }
    lds_barrier();
  }
  // the barriers that are left of cnt + 1: this team's chunks have had two each
  if (TEAMS == 2 && ((cnt - team) & 1) == 0) lds_barrier();
}

template <typename T, int KP, LinRows ROWS>
__global__ __launch_bounds__((LinWalk<T, KP, kWalkSteps<T, KP>, kOutputs>::kThreads)) void
    lin_walk_kernel(LinWalkArgs g) {
  constexpr int C = kWalkSteps<T, KP>;
  typedef LinWalk<T, KP, C, kOutputs> W;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  LinUnit<C> u;
  if (!u.init(g, block_of())) return;
  const int id = (int)threadIdx.x, lane = id & 63;
  const int w = __builtin_amdgcn_readfirstlane(id >> 6);
  if (w >= W::NW + 2) {
    lin_bring<T, KP, ROWS, C, kOutputs, false>(g, u, lds, id - 64 * (W::NW + 2));
  } else if (w >= W::NW) {
    lin_states<T, KP, C, kOutputs, false>(g, u, lds, lane, w - W::NW);
  } else {
    constexpr int kTeam = C / 32;  // waves of a team
    const int team = w / kTeam, n = w % kTeam;
    if constexpr (W::TEAMS == 1) {
      if (w < 2) lin_outputs<T, KP, ROWS, C, 0>(g, u, lds, lane, {w}, 0);
      else if constexpr (C == 64) lin_outputs<T, KP, ROWS, C, 1>(g, u, lds, lane, {w}, 0);
    } else if constexpr (C == 128) {
      if (n < 2) lin_outputs<T, KP, ROWS, C, 0, 1>(g, u, lds, lane, {n, 3 - n}, team);
      else lin_outputs<T, KP, ROWS, C, 2, 3>(g, u, lds, lane, {n + 2, 9 - n}, team);
    } else {
      lin_outputs<T, KP, ROWS, C, 0, C / 32 - 1>(g, u, lds, lane, {n, C / 16 - 1 - n}, team);
    }
  }
}

// The states' walk and its way back, side by side: the first nf workgroups go forward.
template <typename T, int KP, LinRows ROWS, int MODE>
__global__ __launch_bounds__((LinWalk<T, KP, kLinChunk, MODE>::kThreads)) void
    lin_states_kernel(LinWalkArgs f, LinWalkArgs back, uint32_t nf) {
  constexpr int C = kLinChunk;
  typedef LinWalk<T, KP, C, MODE> W;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  const uint32_t block = block_of();
  const int id = (int)threadIdx.x, lane = id & 63;
  const int w = __builtin_amdgcn_readfirstlane(id >> 6);
  LinUnit<C> u;
  if (block < nf) {
    if (!u.init(f, block)) return;
    if (w < 2) lin_states<T, KP, C, MODE, false>(f, u, lds, lane, w);
    else lin_bring<T, KP, ROWS, C, MODE, false>(f, u, lds, id - 128);
  } else {
    if (!u.init(back, block - nf)) return;
    if (w < 2) lin_states<T, KP, C, MODE, true>(back, u, lds, lane, w);
    else lin_bring<T, KP, ROWS, C, MODE, true>(back, u, lds, id - 128);
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

template <typename T, int KP, LinRows ROWS>
int lin_walk_run(LinWalkArgs g, hipStream_t s) {
  typedef LinWalk<T, KP, kWalkSteps<T, KP>, kOutputs> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t wgs = lin_walk_sizes(g, kWalkSteps<T, KP>);
  if (wgs < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_walk_kernel<T, KP, ROWS>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(wgs), W::kThreads, sizeof(typename W::Lds), s>>>(g);
  return launch_status();
}

// back.walked = 0: forward alone.
template <typename T, int KP, LinRows ROWS, int MODE>
int lin_states_run(LinWalkArgs f, LinWalkArgs back, hipStream_t s) {
  typedef LinWalk<T, KP, kLinChunk, MODE> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t nf = lin_walk_sizes(f, kLinChunk);
  const int64_t nb = lin_walk_sizes(back, kLinChunk);
  if (nf < 0 || nb < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_states_kernel<T, KP, ROWS, MODE>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(nf + nb), W::kThreads, sizeof(typename W::Lds), s>>>(f, back, (uint32_t)nf);
  return launch_status();
}

}  // namespace
}  // namespace tssm
