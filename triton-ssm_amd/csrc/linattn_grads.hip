// Linear attention, chunked: the gradients of the inputs, every chunk on its own.
//
// With S the state before a chunk of C steps, dS the gradient of the one after it, D
// as in linattn_walk.h, P = scale D (Q K^T) and R = scale D (dO V^T):
//   dQ = R K + scale e^G (dO S^T),   dK = R^T Q + e^(G_end - G) (V dS^T),
//   dV = P^T dO + e^(G_end - G) (K dS).
// g_t counts for whatever goes past step t: with W = P (dO V^T) element by element,
// x_t = q_t . (the state's part of dQ), y_i = k_i . (the gradient's part of dK),
//   dg_t = sum over s >= t > i of W[s][i] + sum over s >= t of x_s
//          + sum over i < t of y_i + e^(G_end) <S, dS>
// which sums over one chunk only, and nothing but terms that hold e^(g_t): the weights W
// that cross step t are added up as such, x from the end and y from the start.  (The sums
// of W's rows less those of its columns, over a chunk as over the whole sequence, are
// differences of large sums: rounded to fp32 they leave 1e-6 of the chunk's largest dg
// where a strong decay among slow ones makes it 1e-13.)
//
// A workgroup of C / 16 waves has one chunk of one key head and goes through its
// value heads and blocks of V, whose dQ and dK add up in registers, in order (where that
// leaves CUs idle, a workgroup for each value head and a sum of theirs).  A wave
// has 16 steps: as keys (columns of P and R) for dK and dV, as queries (columns of
// R^T) for dQ, so that every product's result is the next one's operand in place
// (planes.h); R is formed in both places.  The states' planes take one buffer after
// the other: S for dQ, then dS for dK and dV.
//
// What bounds it: memory.  B=4 L=4096 H=16 64 x 64 bf16 takes 87 us for 134 MB of inputs,
// 134 MB of states and 100 MB of gradients, 4.2 TB/s where a copy reaches 5.1: two
// workgroups are on a CU (one, with 266 registers, took 160 us), and what one waits for
// is hidden by the other's work alone.  The states are read once, past the caches
// (through them 6 us more).  Chunks of 128 steps would halve the states and leave LDS for
// one workgroup; chunks of 32 in fp32 took 380 us for 344 (the same sizes, all kernels),
// and 483 for 278 at B=2 L=2048 H=16 128 x 128: two waves on a CU.
#include "linattn_dev.h"

namespace tssm {
namespace {

struct LinGradArgs {
  LinArgs a;
  LinGrads d;
  const float *states, *grads;  // [bh][nch][state]
  float* part;                  // split > 1: [dQ, dK][split][B, L, Hk, K]
  int nch, nvb;                 // chunks; blocks of VB columns
  int split, heads;             // workgroups of a key head's value heads; heads of each
  uint32_t units;
};

template <typename T, int KP, int C>
struct Grad {
  static constexpr int NP = kPlanes<T>, NO = kOutPlanes<T>;
  // (two planes of 64 columns would leave LDS for one workgroup: 246 against 221 us a call
  // at B=4 L=4096 H=16 64 x 64 fp16)
  static constexpr int VB = KP == 128 || NP == 2 ? 32 : 64, NS = KP / 32, KT = KP / 16, VS = VB / 32,
                       VT = VB / 16, NW = C / 16, NT = 64 * NW;
  typedef Swizzled<KP> KR;  // rows of Q, K and the states' planes
  typedef Swizzled<VB> VR;  // of V and dO
  static constexpr int kNk = C * KP / 8 / NT, kNv = C * VB / 8 / NT, kNs = VT * KT * 64 / NT;
  struct Lds {
    uint16_t Q[NP][C * KP], K[NP][C * KP], V[NP][C * VB], O[NP][C * VB];
    uint16_t S[3][VB * KP];  // planes of S^T, then of dS^T
    Decays<C> d;
    // of W, a wave's 16 keys: sums of the rows past its tile, and what crosses the tile's
    // steps up to the next eighth; then dg without z, by the waves
    float r[NW][C], z[NW];
  };
};

// Sums of 16 lanes' values, from the lane on or before it.
__device__ inline float from16(float v) {
  v += dpp_mov<0x101>(v);  // row_shl:1, zero into the last
  v += dpp_mov<0x102>(v);
  v += dpp_mov<0x104>(v);
  v += dpp_mov<0x108>(v);
  return v;
}
__device__ inline float before16(float v) {
  v = dpp_mov<0x111>(v);  // row_shr:1, zero into the first
  v += dpp_mov<0x111>(v);
  v += dpp_mov<0x112>(v);
  v += dpp_mov<0x114>(v);
  v += dpp_mov<0x118>(v);
  return v;
}
__device__ inline float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

template <typename T, int KP, LinRows ROWS, int C>
// two workgroups on a CU but where their registers would spill
__global__ __launch_bounds__(4 * C, kPlanes<T> < 3 && KP <= 64 ? 2 : 1) void
    lin_grads_kernel(LinGradArgs g) {
  typedef Grad<T, KP, C> W;
  typedef typename W::KR KR;
  typedef typename W::VR VR;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, KT = W::KT, VS = W::VS, VT = W::VT,
                NT = W::NT, NW = W::NW, VB = W::VB, kE = (int)sizeof(T), NB = C / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  const LinArgs& a = g.a;
  const uint32_t id = block_of();
  if (id >= g.units) return;
  const uint32_t bnk = id / (uint32_t)g.split, bn = bnk / (uint32_t)a.Hk;
  const int64_t hk = bnk - bn * (uint32_t)a.Hk, b = bn / (uint32_t)g.nch;
  const int hs = (int)(id - bnk * (uint32_t)g.split), h0 = hs * g.heads, h1 = h0 + g.heads;
  const int n = (int)(bn - (uint32_t)b * (uint32_t)g.nch);
  const int per = (int)(a.Hv / a.Hk), K = (int)a.K;
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int own = 16 * w + c, db = w >> 1, ar = 8 * (c >> 2) + (c & 3);
  const int64_t elems = lin_state_elems(KP, a.V), t0 = (int64_t)n * C;
  const int rows = a.L - t0 < C ? (int)(a.L - t0) : C;
  const int tiles = (int)((a.V + 31) / 32) * 2;  // tiles of 16 columns that a state has

  RowsOf<C> rq, rk;
  rq.init(reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h, a.q_l, K, a.L);
  rk.init(reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, a.k_l, K, a.L);
  // A value head's block of V, dO and the states, on their way from memory: the first
  // with Q and K, the next ones behind the last use of the registers before them.
  Piece<T, ROWS == kAllRows, NP> pv[W::kNv], po[W::kNv];
  f32x4 st[W::kNs], gr[W::kNs];
  Gaps<C> gaps;
  const auto fetch = [&](int hi, int vb) {
    const int64_t h = hk * per + hi, bh = b * a.Hv + h, v0 = (int64_t)vb * VB;
    const int nv = a.V - v0 < VB ? (int)(a.V - v0) : VB;
    RowsOf<C> rv, ro;
    rv.init(reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + v0, a.v_l, nv, a.L);
    ro.init(reinterpret_cast<const T*>(g.d.dout) + b * g.d.d_b + h * g.d.d_h + v0, g.d.d_l, nv,
            a.L);
    const auto dv = rv.at(n), dd = ro.at(n);
#pragma unroll
    for (int i = 0; i < W::kNv; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (VB / 8), x = at % (VB / 8) * 8;
      pv[i].load(dv, x < nv ? r * rv.row + x * kE : kPast);
      po[i].load(dd, x < nv ? r * ro.row + x * kE : kPast);
    }
#pragma unroll
    for (int i = 0; i < W::kNs; ++i) {
      const int tile = w + NW * i, vt = vb * VT + tile / KT;
      const int64_t at = (bh * g.nch + n) * elems +
                         ((int64_t)(vt < tiles ? vt : 0) * KT + tile % KT) * 256 + lane * 4;
      st[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(g.states + at));
      gr[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(g.grads + at));
    }
    gaps.load(a.g + b * a.g_b + h * a.g_h + t0 * a.g_l, a.g_l, lane, rows);
  };
  {
    const auto dq = rq.at(n), dk = rk.at(n);
    Piece<T, ROWS != kNoRows, NP> pq[W::kNk], pk[W::kNk];
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      pq[i].load(dq, x < K ? r * rq.row + x * kE : kPast);
      pk[i].load(dk, x < K ? r * rk.row + x * kE : kPast);
    }
    fetch(h0, 0);
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8);
      u32x4 p[NP];
      planes_apart(pq[i], K - 8 * x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.Q[y][KR::at(r, x)]) = p[y];
      planes_apart(pk[i], K - 8 * x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.K[y][KR::at(r, x)]) = p[y];
    }
  }
  f32x4 dq[KT], dk[KT];
#pragma unroll
  for (int i = 0; i < KT; ++i) dq[i] = dk[i] = zero4();

  for (int hi = h0; hi < h1; ++hi) {
    const int64_t h = hk * per + hi;
    float sumx = 0.0f, sumy = 0.0f, sumz = 0.0f;
    float past8 = 0.0f, past16 = 0.0f;  // of W's column, past 8 and 16 rows of the tile
    for (int vb = 0; vb < g.nvb; ++vb) {
      const int64_t v0 = (int64_t)vb * VB;
      const int nv = a.V - v0 < VB ? (int)(a.V - v0) : VB;
      if (vb > 0 || hi > h0) fetch(hi, vb);
      lds_barrier();  // the one before is done with LDS
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) {
        const int at = (int)threadIdx.x + NT * i, r = at / (VB / 8), x = at % (VB / 8);
        u32x4 p[NP];
        planes_apart(pv[i], nv - 8 * x, p);
#pragma unroll
        for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.V[y][VR::at(r, x)]) = p[y];
        planes_apart(po[i], nv - 8 * x, p);
#pragma unroll
        for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.O[y][VR::at(r, x)]) = p[y];
      }
#pragma unroll
      for (int i = 0; i < W::kNs; ++i)  // (tiles past the state's read its first)
        if (vb * VT + (w + NW * i) / KT >= tiles) st[i] = gr[i] = zero4();
      const auto show = [&](const f32x4 (&m)[W::kNs]) {
#pragma unroll
        for (int i = 0; i < W::kNs; ++i) {
          const int tile = w + NW * i, vt = tile / KT, kt = tile % KT;
          float x0 = m[i][0], x1 = m[i][1], x2 = m[i][2], x3 = m[i][3];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const uint32_t lo = pk_bf16(x0, x1), hi2 = pk_bf16(x2, x3);
            *reinterpret_cast<uint2*>(
                &lds.S[p][KR::at(16 * vt + c, 4 * (kt >> 1) + j) + 4 * (kt & 1)]) =
                make_uint2(lo, hi2);
            if (p < 2) {
              take_plane(lo, x0, x1);
              take_plane(hi2, x2, x3);
            }
          }
        }
      };
      show(st);
      float z = 0.0f;
#pragma unroll
      for (int i = 0; i < W::kNs; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(st[i][r], gr[i][r], z);
      sumz += group_sum<64>(z);
      if (vb == 0) {
        if (w == 0) gaps.decays(lds.d, lane);
        for (int i = (int)threadIdx.x; i < NW * C; i += NT) (&lds.r[0][0])[i] = 0.0f;
      }
      lds_barrier();

      const float ht = lds.d.hi[own], lt = lds.d.lo[own];
      const float hend = lds.d.hi[C - 1], lend = lds.d.lo[C - 1];
      u32x4 ob[VS][NP];
#pragma unroll
      for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int y = 0; y < NP; ++y) ob[s][y] = VR::get(lds.O[y], own, 4 * s + j);
      // ---- 16 queries: dQ
      {
        for (int ib = 0; ib <= db; ++ib) {
          u32x4 fv[VS][2][NP], fk[KT][NP];
          float h8[8], l8[8], p8[8];
#pragma unroll
          for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int y = 0; y < NP; ++y)
                fv[s][x][y] = VR::get(lds.V[y], 32 * ib + ar + 4 * x, 4 * s + j);
          const float h1 = one_of8(&lds.d.hi[32 * ib], lane), l1 = one_of8(&lds.d.lo[32 * ib], lane);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int y = 0; y < NP; ++y)
              fk[kt][y] = KR::col(lds.K[y], 32 * ib, 32 * (kt >> 1) + 4 * (kt & 1), lane);
          if constexpr (NP == 1) __builtin_amdgcn_sched_barrier(0);
          f32x4 q[2] = {zero4(), zero4()};  // V dO^T, rows i
#pragma unroll
          for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x) q[x] = mfma_planes<NP, NP, NO>(fv[s][x], ob[s], q[x]);
          eight(h1, h8);
          eight(l1, l8);
#pragma unroll
          for (int e = 0; e < 8; ++e) p8[e] = a.scale * diff2(ht, lt, h8[e], l8[e]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            asm("" : "+v"(p8[e]));  // no branch around the exponential
            p8[e] = 32 * ib + 8 * j + e <= own ? q[e >> 2][e & 3] * p8[e] : 0.0f;
          }
          u32x4 pb[NO];
          split8<NO>(p8, pb);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) dq[kt] = mfma_planes<NP, NO, NO>(fk[kt], pb, dq[kt]);
        }
        const float from = a.scale * exp2_fast(ht + lt);
        float dot = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float q8[8];
#pragma unroll
          for (int y = NP - 1; y >= 0; --y) {
            const u32x4 v = KR::get(lds.Q[y], own, 4 * s + j);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
              q8[e] = y == NP - 1 ? x : q8[e] + x;
            }
          }
          u32x4 f[VS][2][3];
#pragma unroll
          for (int vs = 0; vs < VS; ++vs)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int p = 0; p < 3; ++p)
                f[vs][x][p] = KR::col(lds.S[p], 32 * vs, 32 * s + 4 * x, lane);
          if constexpr (NP == 1) __builtin_amdgcn_sched_barrier(0);
          f32x4 q[2] = {zero4(), zero4()};
#pragma unroll
          for (int vs = 0; vs < VS; ++vs)
#pragma unroll
            for (int x = 0; x < 2; ++x) q[x] = mfma_planes<3, NP, 3>(f[vs][x], ob[vs], q[x]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float y = q[x][r] * from;
              dq[2 * s + x][r] += y;
              dot = __builtin_fmaf(q8[4 * x + r], y, dot);
            }
        }
        dot += __shfl_xor(dot, 16);
        dot += __shfl_xor(dot, 32);
        sumx += dot;
      }
      // ---- 16 keys: dK and dV
      u32x4 kb[NS][NP], vbf[VS][NP];
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int y = 0; y < NP; ++y) kb[s][y] = KR::get(lds.K[y], own, 4 * s + j);
#pragma unroll
      for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int y = 0; y < NP; ++y) vbf[s][y] = VR::get(lds.V[y], own, 4 * s + j);
      f32x4 dvt[VT];
#pragma unroll
      for (int i = 0; i < VT; ++i) dvt[i] = zero4();
      for (int tb = db; tb < NB; ++tb) {
        u32x4 fq[NS][2][NP], fo[VS][2][NP];
        float h8[8], l8[8], p8[8], r8[8], w8[8];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < NP; ++y) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
              fq[s][x][y] = KR::get(lds.Q[y], 32 * tb + ar + 4 * x, 4 * s + j);
#pragma unroll
            for (int s = 0; s < VS; ++s)
              fo[s][x][y] = VR::get(lds.O[y], 32 * tb + ar + 4 * x, 4 * s + j);
          }
        const float h1 = one_of8(&lds.d.hi[32 * tb], lane), l1 = one_of8(&lds.d.lo[32 * tb], lane);
        if constexpr (NP == 1) __builtin_amdgcn_sched_barrier(0);
        f32x4 qk[2] = {zero4(), zero4()}, ov[2] = {zero4(), zero4()};  // rows t
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int x = 0; x < 2; ++x) qk[x] = mfma_planes<NP, NP, 3>(fq[s][x], kb[s], qk[x]);
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
          for (int x = 0; x < 2; ++x) ov[x] = mfma_planes<NP, NP, 3>(fo[s][x], vbf[s], ov[x]);
        float d8[8];
        eight(h1, h8);
        eight(l1, l8);
#pragma unroll
        for (int e = 0; e < 8; ++e) d8[e] = a.scale * diff2(h8[e], l8[e], ht, lt);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          asm("" : "+v"(d8[e]));  // no branch around the exponential
          const int t = 32 * tb + 8 * j + e;
          p8[e] = t >= own ? qk[e >> 2][e & 3] * d8[e] : 0.0f;
          r8[e] = t >= own ? ov[e >> 2][e & 3] * d8[e] : 0.0f;
          w8[e] = t > own ? p8[e] * ov[e >> 2][e & 3] : 0.0f;
        }
        u32x4 co[VT][NP], cq[KT][NP];
#pragma unroll
        for (int y = 0; y < NP; ++y) {
#pragma unroll
          for (int i = 0; i < VT; ++i)
            co[i][y] = VR::col(lds.O[y], 32 * tb, 32 * (i >> 1) + 4 * (i & 1), lane);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
            cq[kt][y] = KR::col(lds.Q[y], 32 * tb, 32 * (kt >> 1) + 4 * (kt & 1), lane);
        }
        u32x4 pb[NO], rb[NO];
        split8<NO>(p8, pb);
        split8<NO>(r8, rb);
#pragma unroll
        for (int i = 0; i < VT; ++i) dvt[i] = mfma_planes<NP, NO, NO>(co[i], pb, dvt[i]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) dk[kt] = mfma_planes<NP, NO, NO>(cq[kt], rb, dk[kt]);
        // W's rows, but in the wave's own tile its columns from their end up to each row, and
        // of those the ones before it.  (Here, behind the products, and with what they read
        // asked for after W is formed: 10 to 25 registers fewer, no spills, and the time that
        // rows less columns took.)
        const bool tile = tb == db && (j >> 1) == (w & 1);
        float down = 0.0f;
#pragma unroll
        for (int e = 7; e >= 0; --e) {
          down += w8[e];
          w8[e] = group_sum<16>(tile && 32 * tb + 8 * j + e > own ? down : w8[e]);
        }
        past16 += tile ? 0.0f : down;
        past8 += tile && !(j & 1) ? 0.0f : down;
        if (c == 0) {
          float* p = &lds.r[w][32 * tb + 8 * j];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] += w8[e];
        }
      }
      lds_barrier();  // S is read
      show(gr);
      lds_barrier();
      const float to = diff2(hend, lend, ht, lt);
      float dot = 0.0f;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        float k8[8];
#pragma unroll
        for (int y = NP - 1; y >= 0; --y)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x =
                __uint_as_float(e & 1 ? kb[s][y][e >> 1] & 0xffff0000u : kb[s][y][e >> 1] << 16);
            k8[e] = y == NP - 1 ? x : k8[e] + x;
          }
        u32x4 f[VS][2][3];
#pragma unroll
        for (int vs = 0; vs < VS; ++vs)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int p = 0; p < 3; ++p)
              f[vs][x][p] = KR::col(lds.S[p], 32 * vs, 32 * s + 4 * x, lane);
        if constexpr (NP == 1) __builtin_amdgcn_sched_barrier(0);
        f32x4 q[2] = {zero4(), zero4()};
#pragma unroll
        for (int vs = 0; vs < VS; ++vs)
#pragma unroll
          for (int x = 0; x < 2; ++x) q[x] = mfma_planes<3, NP, 3>(f[vs][x], vbf[vs], q[x]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float y = q[x][r] * to;
            dk[2 * s + x][r] += y;
            dot = __builtin_fmaf(k8[4 * x + r], y, dot);
          }
      }
      dot += __shfl_xor(dot, 16);
      dot += __shfl_xor(dot, 32);
      sumy += dot;
#pragma unroll
      for (int i = 0; i < VT; ++i) {
        f32x4 q = zero4();
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          u32x4 f[NO];
#pragma unroll
          for (int p = 0; p < NO; ++p)
            f[p] = KR::get(lds.S[p], 32 * (i >> 1) + ar + 4 * (i & 1), 4 * s + j);
          q = mfma_planes<NO, NP, NO>(f, kb[s], q);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) dvt[i][r] = __builtin_fmaf(q[r], to, dvt[i][r]);
      }
      // dV of the wave's 16 keys: 8 neighbouring columns a lane and pair of tiles
      if (own < rows) {
        T* p = reinterpret_cast<T*>(g.d.dv) + ((b * a.L + t0 + own) * a.Hv + h) * a.V + v0;
#pragma unroll
        for (int i = 0; i < VS; ++i) {
          const int x = 32 * i + 8 * j;
          const float o8[8] = {dvt[2 * i][0], dvt[2 * i][1], dvt[2 * i][2], dvt[2 * i][3],
                               dvt[2 * i + 1][0], dvt[2 * i + 1][1], dvt[2 * i + 1][2],
                               dvt[2 * i + 1][3]};
          if constexpr (ROWS == kAllRows) {
            if (x < nv) {
              st_lanes<T, 4>(p + x, o8);
              st_lanes<T, 4>(p + x + 4, o8 + 4);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (x + e < nv) stf(p + x + e, o8[e]);
          }
        }
      }
      // (that these are loaded again is more than the compiler sees)
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) pv[i] = po[i] = {};
#pragma unroll
      for (int i = 0; i < W::kNs; ++i) st[i] = gr[i] = zero4();
    }
    // dg of this value head: what the wave's 16 steps leave at each step, a lane each
    static_assert(C == 64, "a lane for each step");
    {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      const float r = lds.r[w][lane];
      past8 += __shfl_xor(past8, 16);
      past8 = before16(past8 + __shfl_xor(past8, 32));
      past16 += __shfl_xor(past16, 16);
      past16 = before16(past16 + __shfl_xor(past16, 32));
      float rest = from16(j > w ? r : 0.0f);  // rows past the tile, from the step on
      const float r1 = lane_of(rest, 16), r2 = lane_of(rest, 32), r3 = lane_of(rest, 48);
      rest += (j < 1 ? r1 : 0.0f) + (j < 2 ? r2 : 0.0f) + (j < 3 ? r3 : 0.0f);
      const float ahead = from16(sumx), behind = before16(sumy);
      const float allx = lane_of(ahead, 0), ally = lane_of(behind + sumy, 15);
      const float tile = r + (c < 8 ? past8 : past16) + (ahead + behind);
      lds.r[w][lane] = j == w ? tile : (j > w ? rest + ally : allx);
      if (lane == 0) lds.z[w] = sumz;
    }
    lds_barrier();
    if (w == 0) {
      double sum = 0.0, z = 0.0;
      for (int i = 0; i < NW; ++i) sum += (double)lds.r[i][lane];
      for (int i = 0; i < NW; ++i) z += (double)lds.z[i];
      z *= (double)exp2_fast(lds.d.hi[C - 1] + lds.d.lo[C - 1]);
      // nothing passes a step whose decay is 0 in fp32
      if (lane < rows)
        g.d.dg[(b * a.L + t0 + lane) * a.Hv + h] = gaps.g[0] < -104.0f ? 0.0f : (float)(sum + z);
    }
  }
  // dQ and dK of the wave's 16 steps
  if (own < rows) {
    const int64_t at = ((b * a.L + t0 + own) * a.Hk + hk) * a.K, n = a.B * a.L * a.Hk * a.K;
    const auto store = [&](auto* pq, auto* pk) {
      typedef std::remove_reference_t<decltype(*pq)> O;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int x = 32 * s + 8 * j;
        float q8[8], k8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          q8[e] = dq[2 * s + (e >> 2)][e & 3];
          k8[e] = dk[2 * s + (e >> 2)][e & 3];
        }
        if constexpr (ROWS != kNoRows) {
          if (x < K) {
            st_lanes<O, 4>(pq + x, q8);
            st_lanes<O, 4>(pq + x + 4, q8 + 4);
            st_lanes<O, 4>(pk + x, k8);
            st_lanes<O, 4>(pk + x + 4, k8 + 4);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (x + e < K) {
              stf(pq + x + e, q8[e]);
              stf(pk + x + e, k8[e]);
            }
        }
      }
    };
    if (g.part) store(g.part + hs * n + at, g.part + (g.split + hs) * n + at);
    else store(reinterpret_cast<T*>(g.d.dq) + at, reinterpret_cast<T*>(g.d.dk) + at);
  }
}

// dQ and dK of value heads that had workgroups of their own, added up in order (4 us for
// what 104 workgroups left: a launch).
template <typename T>
__global__ __launch_bounds__(256) void lin_parts_kernel(const float* part, T* dq, T* dk, int64_t n,
                                                        int split) {
  const int64_t i = (int64_t)block_of() * 256 + threadIdx.x;
  if (i >= 2 * n) return;
  const bool isk = i >= n;
  const int64_t at = isk ? i - n : i;
  const float* p = part + (isk ? split * n : 0) + at;
  float s = p[0];
  for (int h = 1; h < split; ++h) s += p[h * n];
  stf((isk ? dk : dq) + at, s);
}

template <typename T, int KP, LinRows ROWS>
int launch(LinGradArgs g, hipStream_t s) {
  constexpr int C = kLinChunk;
  typedef Grad<T, KP, C> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  g.nch = (int)cdiv64(g.a.L, C);
  g.nvb = (int)cdiv64(g.a.V, W::VB);
  g.heads = (int)(g.a.Hv / g.a.Hk) / g.split;
  const int64_t units = g.a.B * g.a.Hk * g.nch * g.split;
  if (units > 0x7fffffff) return TSSM_ERR_UNSUPPORTED;
  g.units = (uint32_t)units;
  const auto kernel = lin_grads_kernel<T, KP, ROWS, C>;
  if (sizeof(typename W::Lds) > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)sizeof(typename W::Lds));
    if (e != hipSuccess) return (int)e;
  }
  kernel<<<grid_of(units), W::NT, sizeof(typename W::Lds), s>>>(g);
  const int rc = launch_status();
  if (rc || !g.part) return rc;
  const int64_t n = g.a.B * g.a.L * g.a.Hk * g.a.K;
  lin_parts_kernel<T><<<grid_of(cdiv64(2 * n, 256)), 256, 0, s>>>(
      g.part, reinterpret_cast<T*>(g.d.dq), reinterpret_cast<T*>(g.d.dk), n, g.split);
  return launch_status();
}

template <typename T>
int by_keys(const LinGradArgs& g, LinRows rows, hipStream_t s) {
#define TSSM_GRADS(KP)                                   \
  (rows == kAllRows   ? launch<T, KP, kAllRows>(g, s)    \
   : rows == kKeyRows ? launch<T, KP, kKeyRows>(g, s)    \
                      : launch<T, KP, kNoRows>(g, s))
  if (g.a.K <= 32) return TSSM_GRADS(32);
  if (g.a.K <= 64) return TSSM_GRADS(64);
  return TSSM_GRADS(128);
#undef TSSM_GRADS
}

}  // namespace

int lin_grads_launch(int dtype, const LinArgs& a, const LinGrads& d, LinRows rows, const LinPlan& p,
                     hipStream_t s) {
  LinGradArgs g = {};
  g.a = a;
  g.d = d;
  g.states = p.states;
  g.grads = p.grads;
  g.part = p.part;
  g.split = (int)p.split;
  switch (dtype) {
    case TSSM_F32: return by_keys<float>(g, rows, s);
    case TSSM_BF16: return by_keys<bf16_t>(g, rows, s);
    default: return by_keys<f16_t>(g, rows, s);
  }
}

}  // namespace tssm
