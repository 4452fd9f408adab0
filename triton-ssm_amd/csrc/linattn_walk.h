// Linear attention, chunked: the walk over the chunks.
//
// Per chunk of C steps, with S the state before it, G the sums of g and D[t][i] =
// e^(G_t - G_i) for i <= t, 0 above:
//   O = scale (e^G Q S + (Q K^T D) V),   S' = e^(G_end) S + K^T (e^(G_end - G) V).
// Only S' waits for S, by one product and a sum; all the rest of a chunk is its own.
//
// A workgroup of C / 16 waves walks 32 columns of V of one head's segment.  A wave
// has 16 steps of the chunk for the outputs and a share of K^T V: 32 steps for 16
// columns, all of K, of which it keeps the tiles of the state that are its own and
// hands the others to their owners through LDS.  Everything is formed transposed
// (planes.h): a wave's P^T = K Q^T is the next product's operand in place, queries
// come to it straight from memory, and a lane ends up with 8 neighbouring columns of
// one step's output.  Per chunk
//   before the barrier: P and its part of the output, K^T V, the next chunk to LDS,
//   after it: the state's part of the output from planes that the owners left in
//     LDS a chunk ago, and the next state.
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
  static constexpr int kLd = KP + 8, kVld = 40;  // bf16 elements of a row in LDS
  static constexpr int kNk = C * KP / 8 / NT;    // 8-element pieces of K a thread brings
  static_assert(KT % NIQ == 0, "every wave owns tiles");
  struct Operands {  // of one chunk
    uint16_t K[NP][C * kLd], V[NP][C * kVld];
    Decays<C> d;
  };
  struct Lds {
    Operands op[2];
    f32x4 part[2][NW][KT - OWN ? KT - OWN : 1][64];
    // planes of S^T, a row for each column of V
    uint16_t S[MODE == kOutputs ? 2 : 1][NO][MODE == kOutputs ? 32 * kLd : 8];
  };
};

template <typename T, int KP, bool VEC, int C, int MODE, bool REV>
__device__ inline void lin_walk_body(const LinWalkArgs& g, char* smem, uint32_t id) {
  typedef LinWalk<T, KP, C, MODE> W;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, KT = W::KT, NT = W::NT, NIQ = W::NIQ,
                OWN = W::OWN, kE = (int)sizeof(T);
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  const LinArgs& a = g.a;
  // workgroups of one head's segment, which share Q and K, on one XCD
  const uint32_t vb = (id >> 3) % g.nvb, u = (id >> 3) / g.nvb * 8 + (id & 7);
  if (u >= g.units) return;
  const int64_t bh = u / (uint32_t)g.walked;
  const int seg = g.first + (int)(u - (uint32_t)bh * (uint32_t)g.walked);
  const int n0 = seg * g.per, n1 = n0 + g.per < g.nch ? n0 + g.per : g.nch, cnt = n1 - n0;
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // 16 steps for the outputs: waves w and w + 4, on one SIMD, have equal work together
  const int tw = C == 128 && w >= 4 ? 11 - w : w;
  const int iq = w >> 1, vt = w & 1;         // 32 steps, 16 columns for K^T V
  const int ar = 8 * (c >> 2) + (c & 3);     // row of tile x of an A operand, less 4 x
  const auto [b, h, hk] = lin_head(a, (uint32_t)bh);
  const int64_t v0 = (int64_t)vb * 32;
  const int nv = a.V - v0 < 32 ? (int)(a.V - v0) : 32, K = (int)a.K;
  const int64_t elems = lin_state_elems(KP, a.V), col = v0 + 16 * vt + c;
  const int64_t tile0 = ((int64_t)(2 * vb + vt) * KT + iq * OWN) * 256 + lane * 4;

  RowsOf<C> rk, rq, rv, ro;
  rk.init(reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, a.k_l, K, a.L);
  rv.init(reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + v0, a.v_l, nv, a.L);
  if constexpr (MODE == kOutputs) {
    rq.init(reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h, a.q_l, K, a.L);
    ro.init(reinterpret_cast<const T*>(a.o) + b * a.o_b + h * a.o_h + v0, a.o_l, nv, a.L);
  }
  const float* gp = a.g + b * a.g_b + h * a.g_h;

  struct Regs {
    Piece<T, VEC, NP> k[W::kNk], v, q[MODE == kOutputs ? NS : 1];
    Gaps<C> g;
  } in;
  const auto chunk = [&](int m) {   // the chunk of step m of the walk
    const int x = m < cnt ? m : cnt - 1;
    return REV ? n1 - 1 - x : n0 + x;
  };
  const auto fetch = [&](int m) {
    const int n = chunk(m);
    const auto dk = rk.at(n), dv = rv.at(n);
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      in.k[i].load(dk, x < K ? r * rk.row + x * kE : kPast);
    }
    const int r = (int)threadIdx.x >> 2, x = ((int)threadIdx.x & 3) * 8;
    in.v.load(dv, x < nv ? r * rv.row + x * kE : kPast);
    if constexpr (MODE == kOutputs) {
      const auto dq = rq.at(n);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int y = 32 * s + 8 * j;
        in.q[s].load(dq, y < K ? (16 * tw + c) * rq.row + y * kE : kPast);
      }
    }
    if (w == 0) {
      const int64_t t0 = (int64_t)n * C, rest = a.L - t0;
      in.g.load(gp + t0 * a.g_l, a.g_l, lane, rest < C ? (int)rest : C);
    }
  };
  const auto leave = [&](typename W::Operands& o) {  // what fetch() brought, to LDS
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      u32x4 p[NP];
      planes_apart(in.k[i], K - x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&o.K[y][r * W::kLd + x]) = p[y];
    }
    const int r = (int)threadIdx.x >> 2, x = ((int)threadIdx.x & 3) * 8;
    u32x4 p[NP];
    planes_apart(in.v, nv - x, p);
#pragma unroll
    for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&o.V[y][r * W::kVld + x]) = p[y];
    if (w == 0) in.g.decays(o.d, lane);
  };
  u32x4 qb[NS][NP], qn[NS][NP];
  const auto queries = [&](u32x4 (&q)[NS][NP]) {
    if constexpr (MODE == kOutputs) {
#pragma unroll
      for (int s = 0; s < NS; ++s) in.q[s].planes(K - 32 * s - 8 * j, q[s]);
    }
  };

  f32x4 S[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    if constexpr (MODE == kEnds) S[i] = zero4();
    else if (g.nseg == 1)
      S[i] = get_tile(a.h0 ? a.h0 + bh * K * a.V : nullptr, iq * OWN + i, col, a.V, K, j);
    else
      S[i] = *reinterpret_cast<const f32x4*>(g.entry + (bh * g.nseg + seg) * elems + tile0 + 256 * i);
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
          *reinterpret_cast<uint2*>(&lds.S[par][p][(16 * vt + c) * W::kLd + 32 * (kt >> 1) +
                                                   8 * j + 4 * (kt & 1)]) = make_uint2(lo, hi);
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
  queries(qb);
  show(0);
  fetch(1);
  lds_barrier();
  for (int m = 0; m < cnt; ++m) {
    const int n = chunk(m), par = m & 1;
    const typename W::Operands& B = lds.op[par];
    const float hend = B.d.hi[C - 1], lend = B.d.lo[C - 1];
    const float last = exp2_fast(hend + lend);
    float eg = 0.0f;
    f32x4 acc[2] = {zero4(), zero4()}, own[2] = {zero4(), zero4()};
    if constexpr (MODE == kEnds) total += (double)hend + (double)lend;
    if constexpr (MODE == kOutputs) {
      const int db = tw >> 1, t = 16 * tw + c;
      const float ht = B.d.hi[t], lt = B.d.lo[t];
      eg = exp2_fast(ht + lt);
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
                fk[y] = lds16(&B.K[y][(32 * ib + ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
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
            for (int y = 0; y < NP; ++y)
              fv[y] = lds_col(&B.V[y][32 * ib * W::kVld], W::kVld, 4 * x, lane);
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
              v += bf16_bits_to_f32(B.V[y][(32 * db + i) * W::kVld + 8 * j + e]);
            if (32 * db + i <= t) own[e >> 2][e & 3] += p * v;
          }
        }
      }
    }
    // this wave's 32 steps of K^T V
    float v8[8], e8[8];
    lds_values<NP>(&B.V[0][0], C * W::kVld, W::kVld, 32 * iq, 16 * vt, lane, v8);
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
    for (int kt = 0; kt < KT; ++kt) {
      u32x4 fk[NP];
#pragma unroll
      for (int y = 0; y < NP; ++y)
        fk[y] = lds_col(&B.K[y][32 * iq * W::kLd], W::kLd, 32 * (kt >> 1) + 4 * (kt & 1), lane);
      const f32x4 x = mfma_planes<NP, 3, 3>(fk, vp, zero4());
      if (kt / OWN == iq) {
#pragma unroll
        for (int i = 0; i < OWN; ++i)
          if (kt % OWN == i) mine[i] = x;
      } else {
        lds.part[par][w][kt / OWN < iq ? kt : kt - OWN][lane] = x;
      }
    }
    leave(lds.op[par ^ 1]);
    queries(qn);
    fetch(m + 2);
    lds_barrier();
    if constexpr (MODE == kStates) {
      float* p = g.states + (bh * g.nch + n) * elems + tile0;
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
    if constexpr (MODE == kOutputs) {
      show(par ^ 1);
      f32x4 y[2] = {zero4(), zero4()};
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4 fs[NO];
#pragma unroll
          for (int p = 0; p < NO; ++p)
            fs[p] = lds16(&lds.S[par][p][(ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
          y[x] = mfma_planes<NO, NP, NO>(fs, qb[s], y[x]);
        }
      const auto dst = ro.at(n);
      const uint32_t off = (uint32_t)((16 * tw + c) * ro.row + 8 * j * kE);
      float o8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o8[e] = a.scale * __builtin_fmaf(y[e >> 2][e & 3], eg,
                                         acc[e >> 2][e & 3] + own[e >> 2][e & 3]);
      if constexpr (VEC) {
        const uint32_t to = 8 * j < nv ? off : kPast;
        if constexpr (kE == 4) {
          typedef uint32_t vec4 __attribute__((ext_vector_type(4)));
          __builtin_amdgcn_raw_buffer_store_b128(
              vec4{__float_as_uint(o8[0]), __float_as_uint(o8[1]), __float_as_uint(o8[2]),
                   __float_as_uint(o8[3])}, dst, to, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b128(
              vec4{__float_as_uint(o8[4]), __float_as_uint(o8[5]), __float_as_uint(o8[6]),
                   __float_as_uint(o8[7])}, dst, to + 16, 0, 0);
        } else {
          union {
            T e[8];
            u32x4 v;
          } x;
#pragma unroll
          for (int e = 0; e < 8; ++e) stf(&x.e[e], o8[e]);
          __builtin_amdgcn_raw_buffer_store_b128(x.v, dst, to, 0, 0);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          buf_put<T>(dst, 8 * j + e < nv ? off + e * kE : kPast, o8[e]);
      }
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int p = 0; p < NP; ++p) qb[s][p] = qn[s][p];
    }
  }
  if constexpr (MODE == kEnds) {
    float* p = g.states + (bh * g.nseg + seg) * elems + tile0;
#pragma unroll
    for (int i = 0; i < OWN; ++i) *reinterpret_cast<f32x4*>(p + 256 * i) = S[i];
    if (vb == 0 && threadIdx.x == 0) g.sums[bh * g.nseg + seg] = total;
  } else if (REV ? n0 == 0 : n1 == g.nch) {
    float* p = a.h_last ? a.h_last + bh * K * a.V : nullptr;
#pragma unroll
    for (int i = 0; i < OWN; ++i) put_tile(p, S[i], iq * OWN + i, col, a.V, K, j);
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
__global__ __launch_bounds__((4 * kWalkSteps<T, KP>)) void lin_walk_kernel(LinWalkArgs g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  lin_walk_body<T, KP, VEC, kWalkSteps<T, KP>, kOutputs, false>(g, smem, block_of());
}

// The states' walk and its way back, side by side: the first nf workgroups go forward.
template <typename T, int KP, bool VEC, int MODE>
__global__ __launch_bounds__((4 * kStateSteps<T, KP>)) void lin_states_kernel(LinWalkArgs f,
                                                                              LinWalkArgs back,
                                                                              uint32_t nf) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t id = block_of();
  if (id < nf)
    lin_walk_body<T, KP, VEC, kStateSteps<T, KP>, MODE, false>(f, smem, id);
  else
    lin_walk_body<T, KP, VEC, kStateSteps<T, KP>, MODE, true>(back, smem, id - nf);
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
int lin_walk(LinWalkArgs g, hipStream_t s) {
  typedef LinWalk<T, KP, kWalkSteps<T, KP>, kOutputs> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t wgs = lin_walk_sizes(g, kWalkSteps<T, KP>);
  if (wgs < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_walk_kernel<T, KP, VEC>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(wgs), W::NT, sizeof(typename W::Lds), s>>>(g);
  return launch_status();
}

// back.walked = 0: forward alone.
template <typename T, int KP, bool VEC, int MODE>
int lin_states(LinWalkArgs f, LinWalkArgs back, hipStream_t s) {
  typedef LinWalk<T, KP, kStateSteps<T, KP>, MODE> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  const int64_t nf = lin_walk_sizes(f, kStateSteps<T, KP>);
  const int64_t nb = lin_walk_sizes(back, kStateSteps<T, KP>);
  if (nf < 0 || nb < 0) return TSSM_ERR_UNSUPPORTED;
  const auto kernel = lin_states_kernel<T, KP, VEC, MODE>;
  const int rc = lin_lds(kernel, (int)sizeof(typename W::Lds));
  if (rc) return rc;
  kernel<<<grid_of(nf + nb), W::NT, sizeof(typename W::Lds), s>>>(f, back, (uint32_t)nf);
  return launch_status();
}

}  // namespace
}  // namespace tssm
