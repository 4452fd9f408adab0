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
// which sums over one chunk only: over the whole sequence (q . dQ - k . dK, summed
// from the end) the differences of large sums would cost digits of small gradients.
//
// A workgroup of C / 16 waves has one chunk of one key head and goes through its
// value heads and blocks of V, whose dQ and dK add up in registers, in order.  A wave
// has 16 steps: as keys (columns of P and R) for dK and dV, as queries (columns of
// R^T) for dQ, so that every product's result is the next one's operand in place
// (planes.h); R is formed in both places.  The states' planes take one buffer after
// the other: S for dQ, then dS for dK and dV.
#include "linattn_dev.h"

namespace tssm {
namespace {

struct LinGradArgs {
  LinArgs a;
  LinGrads d;
  const float *states, *grads;  // [bh][nch][state]
  int nch, nvb;                 // chunks; blocks of VB columns
  uint32_t units;
};

template <typename T, int KP, int C>
struct Grad {
  static constexpr int NP = kPlanes<T>, NO = kOutPlanes<T>;
  static constexpr int VB = KP == 128 ? 32 : 64, NS = KP / 32, KT = KP / 16, VS = VB / 32,
                       VT = VB / 16, NW = C / 16, NT = 64 * NW;
  static constexpr int kLd = KP + 8, kVld = VB + 8;
  static constexpr int kNk = C * KP / 8 / NT, kNv = C * VB / 8 / NT, kNs = VT * KT * 64 / NT;
  struct Lds {
    uint16_t Q[NP][C * kLd], K[NP][C * kLd], V[NP][C * kVld], O[NP][C * kVld];
    uint16_t S[3][VB * kLd];  // planes of S^T, then of dS^T
    Decays<C> d;
    float r[NW][C], c[C], x[C], y[C], z[NW];
  };
};

template <typename T, int KP, bool VEC, int C>
__global__ __launch_bounds__(4 * C) void lin_grads_kernel(LinGradArgs g) {
  typedef Grad<T, KP, C> W;
  constexpr int NP = W::NP, NO = W::NO, NS = W::NS, KT = W::KT, VS = W::VS, VT = W::VT,
                NT = W::NT, NW = W::NW, VB = W::VB, kE = (int)sizeof(T), NB = C / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typename W::Lds& lds = *reinterpret_cast<typename W::Lds*>(smem);
  const LinArgs& a = g.a;
  const uint32_t id = block_of();
  if (id >= g.units) return;
  const int n = (int)(id % (uint32_t)g.nch);
  const uint32_t bk = id / (uint32_t)g.nch;
  const int64_t b = bk / (uint32_t)a.Hk, hk = bk - (uint32_t)b * (uint32_t)a.Hk;
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
  {
    const auto dq = rq.at(n), dk = rk.at(n);
    Piece<T, VEC, NP> pq[W::kNk], pk[W::kNk];
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      pq[i].load(dq, x < K ? r * rq.row + x * kE : kPast);
      pk[i].load(dk, x < K ? r * rk.row + x * kE : kPast);
    }
#pragma unroll
    for (int i = 0; i < W::kNk; ++i) {
      const int at = (int)threadIdx.x + NT * i, r = at / (KP / 8), x = at % (KP / 8) * 8;
      u32x4 p[NP];
      pq[i].planes(K - x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.Q[y][r * W::kLd + x]) = p[y];
      pk[i].planes(K - x, p);
#pragma unroll
      for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.K[y][r * W::kLd + x]) = p[y];
    }
  }
  f32x4 dq[KT], dk[KT];
#pragma unroll
  for (int i = 0; i < KT; ++i) dq[i] = dk[i] = zero4();

  for (int hi = 0; hi < per; ++hi) {
    const int64_t h = hk * per + hi, bh = b * a.Hv + h;
    float sumx = 0.0f, sumy = 0.0f, sumc = 0.0f, sumz = 0.0f;
    Gaps<C> gaps;
    for (int vb = 0; vb < g.nvb; ++vb) {
      const int64_t v0 = (int64_t)vb * VB;
      const int nv = a.V - v0 < VB ? (int)(a.V - v0) : VB;
      // this head's block of V, dO and the states
      RowsOf<C> rv, ro;
      rv.init(reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + v0, a.v_l, nv, a.L);
      ro.init(reinterpret_cast<const T*>(g.d.dout) + b * g.d.d_b + h * g.d.d_h + v0, g.d.d_l, nv,
              a.L);
      Piece<T, VEC, NP> pv[W::kNv], po[W::kNv];
      const auto dv = rv.at(n), dd = ro.at(n);
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) {
        const int at = (int)threadIdx.x + NT * i, r = at / (VB / 8), x = at % (VB / 8) * 8;
        pv[i].load(dv, x < nv ? r * rv.row + x * kE : kPast);
        po[i].load(dd, x < nv ? r * ro.row + x * kE : kPast);
      }
      f32x4 st[W::kNs], gr[W::kNs];
#pragma unroll
      for (int i = 0; i < W::kNs; ++i) {
        const int tile = w + NW * i, vt = vb * VT + tile / KT;
        const int64_t at = (bh * g.nch + n) * elems +
                           ((int64_t)(vt < tiles ? vt : 0) * KT + tile % KT) * 256 + lane * 4;
        st[i] = *reinterpret_cast<const f32x4*>(g.states + at);
        gr[i] = *reinterpret_cast<const f32x4*>(g.grads + at);
        if (vt >= tiles) st[i] = gr[i] = zero4();
      }
      if (vb == 0 && w == 0)
        gaps.load(a.g + b * a.g_b + h * a.g_h + t0 * a.g_l, a.g_l, lane, rows);
      lds_barrier();  // the one before is done with LDS
#pragma unroll
      for (int i = 0; i < W::kNv; ++i) {
        const int at = (int)threadIdx.x + NT * i, r = at / (VB / 8), x = at % (VB / 8) * 8;
        u32x4 p[NP];
        pv[i].planes(nv - x, p);
#pragma unroll
        for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.V[y][r * W::kVld + x]) = p[y];
        po[i].planes(nv - x, p);
#pragma unroll
        for (int y = 0; y < NP; ++y) *reinterpret_cast<u32x4*>(&lds.O[y][r * W::kVld + x]) = p[y];
      }
      const auto show = [&](const f32x4 (&m)[W::kNs]) {
#pragma unroll
        for (int i = 0; i < W::kNs; ++i) {
          const int tile = w + NW * i, vt = tile / KT, kt = tile % KT;
          float x0 = m[i][0], x1 = m[i][1], x2 = m[i][2], x3 = m[i][3];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const uint32_t lo = pk_bf16(x0, x1), hi2 = pk_bf16(x2, x3);
            *reinterpret_cast<uint2*>(
                &lds.S[p][(16 * vt + c) * W::kLd + 32 * (kt >> 1) + 8 * j + 4 * (kt & 1)]) =
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
        for (int y = 0; y < NP; ++y) ob[s][y] = lds16(&lds.O[y][own * W::kVld + 32 * s + 8 * j]);
      // ---- 16 queries: dQ
      {
        for (int ib = 0; ib <= db; ++ib) {
          f32x4 q[2] = {zero4(), zero4()};  // V dO^T, rows i
#pragma unroll
          for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              u32x4 f[NP];
#pragma unroll
              for (int y = 0; y < NP; ++y)
                f[y] = lds16(&lds.V[y][(32 * ib + ar + 4 * x) * W::kVld + 32 * s + 8 * j]);
              q[x] = mfma_planes<NP, NP, NO>(f, ob[s], q[x]);
            }
          float h8[8], l8[8], p8[8];
          lds8(&lds.d.hi[32 * ib + 8 * j], h8);
          lds8(&lds.d.lo[32 * ib + 8 * j], l8);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            p8[e] = 32 * ib + 8 * j + e <= own
                        ? q[e >> 2][e & 3] * (a.scale * diff2(ht, lt, h8[e], l8[e])) : 0.0f;
          u32x4 pb[NO];
          split8<NO>(p8, pb);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            u32x4 f[NP];
#pragma unroll
            for (int y = 0; y < NP; ++y)
              f[y] = lds_col(&lds.K[y][32 * ib * W::kLd], W::kLd, 32 * (kt >> 1) + 4 * (kt & 1),
                             lane);
            dq[kt] = mfma_planes<NP, NO, NO>(f, pb, dq[kt]);
          }
        }
        const float from = a.scale * exp2_fast(ht + lt);
        float dot = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float q8[8];
#pragma unroll
          for (int y = NP - 1; y >= 0; --y) {
            const u32x4 v = lds16(&lds.Q[y][own * W::kLd + 32 * s + 8 * j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float x = __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
              q8[e] = y == NP - 1 ? x : q8[e] + x;
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            f32x4 q = zero4();
#pragma unroll
            for (int vs = 0; vs < VS; ++vs) {
              u32x4 f[3];
#pragma unroll
              for (int p = 0; p < 3; ++p)
                f[p] = lds_col(&lds.S[p][32 * vs * W::kLd], W::kLd, 32 * s + 4 * x, lane);
              q = mfma_planes<3, NP, 3>(f, ob[vs], q);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float y = q[r] * from;
              dq[2 * s + x][r] += y;
              dot = __builtin_fmaf(q8[4 * x + r], y, dot);
            }
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
        for (int y = 0; y < NP; ++y) kb[s][y] = lds16(&lds.K[y][own * W::kLd + 32 * s + 8 * j]);
#pragma unroll
      for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int y = 0; y < NP; ++y) vbf[s][y] = lds16(&lds.V[y][own * W::kVld + 32 * s + 8 * j]);
      f32x4 dvt[VT];
#pragma unroll
      for (int i = 0; i < VT; ++i) dvt[i] = zero4();
      for (int tb = db; tb < NB; ++tb) {
        f32x4 qk[2] = {zero4(), zero4()}, ov[2] = {zero4(), zero4()};  // rows t
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            u32x4 f[NP];
#pragma unroll
            for (int y = 0; y < NP; ++y)
              f[y] = lds16(&lds.Q[y][(32 * tb + ar + 4 * x) * W::kLd + 32 * s + 8 * j]);
            qk[x] = mfma_planes<NP, NP, 3>(f, kb[s], qk[x]);
          }
#pragma unroll
          for (int s = 0; s < VS; ++s) {
            u32x4 f[NP];
#pragma unroll
            for (int y = 0; y < NP; ++y)
              f[y] = lds16(&lds.O[y][(32 * tb + ar + 4 * x) * W::kVld + 32 * s + 8 * j]);
            ov[x] = mfma_planes<NP, NP, 3>(f, vbf[s], ov[x]);
          }
        }
        float h8[8], l8[8], p8[8], r8[8], w8[8];
        lds8(&lds.d.hi[32 * tb + 8 * j], h8);
        lds8(&lds.d.lo[32 * tb + 8 * j], l8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = 32 * tb + 8 * j + e;
          const float d = a.scale * diff2(h8[e], l8[e], ht, lt);
          p8[e] = t >= own ? qk[e >> 2][e & 3] * d : 0.0f;
          r8[e] = t >= own ? ov[e >> 2][e & 3] * d : 0.0f;
          w8[e] = t > own ? p8[e] * ov[e >> 2][e & 3] : 0.0f;
          sumc += w8[e];
          w8[e] = group_sum<16>(w8[e]);
        }
        if (c == 0) {
          float* p = &lds.r[w][32 * tb + 8 * j];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] += w8[e];
        }
        u32x4 pb[NO], rb[NO];
        split8<NO>(p8, pb);
        split8<NO>(r8, rb);
#pragma unroll
        for (int i = 0; i < VT; ++i) {
          u32x4 f[NP];
#pragma unroll
          for (int y = 0; y < NP; ++y)
            f[y] = lds_col(&lds.O[y][32 * tb * W::kVld], W::kVld, 32 * (i >> 1) + 4 * (i & 1), lane);
          dvt[i] = mfma_planes<NP, NO, NO>(f, pb, dvt[i]);
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          u32x4 f[NP];
#pragma unroll
          for (int y = 0; y < NP; ++y)
            f[y] = lds_col(&lds.Q[y][32 * tb * W::kLd], W::kLd, 32 * (kt >> 1) + 4 * (kt & 1), lane);
          dk[kt] = mfma_planes<NP, NO, NO>(f, rb, dk[kt]);
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
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          f32x4 q = zero4();
#pragma unroll
          for (int vs = 0; vs < VS; ++vs) {
            u32x4 f[3];
#pragma unroll
            for (int p = 0; p < 3; ++p)
              f[p] = lds_col(&lds.S[p][32 * vs * W::kLd], W::kLd, 32 * s + 4 * x, lane);
            q = mfma_planes<3, NP, 3>(f, vbf[vs], q);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float y = q[r] * to;
            dk[2 * s + x][r] += y;
            dot = __builtin_fmaf(k8[4 * x + r], y, dot);
          }
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
            f[p] = lds16(&lds.S[p][(32 * (i >> 1) + ar + 4 * (i & 1)) * W::kLd + 32 * s + 8 * j]);
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
          if constexpr (VEC) {
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
    }
    // dg of this value head
    sumc += __shfl_xor(sumc, 16);
    sumc += __shfl_xor(sumc, 32);
    if (j == 0) {
      lds.c[own] = sumc;
      lds.x[own] = sumx;
      lds.y[own] = sumy;
    }
    if (lane == 0) lds.z[w] = sumz;
    lds_barrier();
    if (w == 0) {
      const int t = lane < C ? lane : 0;
      double past = 0.0, y = 0.0, z = 0.0;
      if (lane < C) {
        for (int i = 0; i < NW; ++i) past += (double)lds.r[i][t];
        past += (double)lds.x[t] - (double)lds.c[t];
        y = (double)lds.y[t];
      }
      for (int i = 0; i < NW; ++i) z += (double)lds.z[i];
      double before = y;
#pragma unroll
      for (int i = 1; i < 64; i *= 2) {
        const double p = __shfl_down(past, i), q = __shfl_up(before, i);
        if (lane + i < 64) past += p;
        if (lane >= i) before += q;
      }
      z *= (double)exp2_fast(lds.d.hi[C - 1] + lds.d.lo[C - 1]);
      // nothing passes a step whose decay is 0 in fp32
      if (lane < rows)
        g.d.dg[(b * a.L + t0 + lane) * a.Hv + h] =
            gaps.g[0] < -104.0f ? 0.0f : (float)(past + (before - y) + z);
    }
  }
  // dQ and dK of the wave's 16 steps
  if (own < rows) {
    const int64_t at = ((b * a.L + t0 + own) * a.Hk + hk) * a.K;
    T* pq = reinterpret_cast<T*>(g.d.dq) + at;
    T* pk = reinterpret_cast<T*>(g.d.dk) + at;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int x = 32 * s + 8 * j;
      float q8[8], k8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q8[e] = dq[2 * s + (e >> 2)][e & 3];
        k8[e] = dk[2 * s + (e >> 2)][e & 3];
      }
      if constexpr (VEC) {
        if (x < K) {
          st_lanes<T, 4>(pq + x, q8);
          st_lanes<T, 4>(pq + x + 4, q8 + 4);
          st_lanes<T, 4>(pk + x, k8);
          st_lanes<T, 4>(pk + x + 4, k8 + 4);
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
  }
}

template <typename T, int KP, bool VEC>
int launch(LinGradArgs g, hipStream_t s) {
  constexpr int C = kPlanes<T> == 3 && KP == 128 ? 32 : 64;
  typedef Grad<T, KP, C> W;
  static_assert(sizeof(typename W::Lds) <= 160 * 1024, "LDS of a CU");
  g.nch = (int)cdiv64(g.a.L, C);
  g.nvb = (int)cdiv64(g.a.V, W::VB);
  const int64_t units = g.a.B * g.a.Hk * g.nch;
  if (units > 0x7fffffff) return TSSM_ERR_UNSUPPORTED;
  g.units = (uint32_t)units;
  const auto kernel = lin_grads_kernel<T, KP, VEC, C>;
  if (sizeof(typename W::Lds) > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)sizeof(typename W::Lds));
    if (e != hipSuccess) return (int)e;
  }
  kernel<<<grid_of(units), W::NT, sizeof(typename W::Lds), s>>>(g);
  return launch_status();
}

template <typename T>
int by_keys(const LinGradArgs& g, bool vec, hipStream_t s) {
#define TSSM_GRADS(KP) (vec ? launch<T, KP, true>(g, s) : launch<T, KP, false>(g, s))
  if (g.a.K <= 32) return TSSM_GRADS(32);
  if (g.a.K <= 64) return TSSM_GRADS(64);
  return TSSM_GRADS(128);
#undef TSSM_GRADS
}

}  // namespace

int lin_grads_launch(int dtype, const LinArgs& a, const LinGrads& d, bool vec, const LinPlan& p,
                     hipStream_t s) {
  LinGradArgs g = {};
  g.a = a;
  g.d = d;
  g.states = p.states;
  g.grads = p.grads;
  switch (dtype) {
    case TSSM_F32: return by_keys<float>(g, vec, s);
    case TSSM_BF16: return by_keys<bf16_t>(g, vec, s);
    default: return by_keys<f16_t>(g, vec, s);
  }
}

}  // namespace tssm
