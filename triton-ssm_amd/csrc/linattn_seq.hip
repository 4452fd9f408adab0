// Linear attention with a decay for each head, step by step: decoding (one step,
// the state in place) and short sequences.
//
//   S = e^g S + k v^T,  o = scale S^T q
//
// A wave owns 4 CQ columns of one head's state for the whole call: lane
// (kg, cq) = (lane / CQ, lane % CQ) holds rows kg KR .. kg KR + KR - 1 of columns
// 4 cq .. 4 cq + 3 in registers.  Columns never meet, so waves are independent;
// the sum over k runs in each lane, then over the row groups by lane exchanges.
// The state is read and written once whatever L is, 16 CQ bytes of a row at a
// time: what bounds one step of many streams (S=4096 H=32 128 x 64: 1.68 ms for 8.6 GB,
// 5.1 TB/s, a copy's rate).  A sequence's steps take 0.4 us each, a step's loads and the
// exchange of its sum.
#include "linattn.h"
#include "rows.h"

namespace tssm {
namespace {

// How a lane reaches its four columns and its rows of q, k and v: element by element, the
// state's rows 16 bytes at a time, or everything in whole pieces.
enum { kElements, kStateRows, kWhole };

typedef float f32x4a __attribute__((ext_vector_type(4), aligned(4)));

template <typename T, int CQ, int KR, int FORM>
__global__ __launch_bounds__(256) void lin_seq_kernel(LinArgs a, uint32_t ncb, uint32_t units) {
  const int lane = threadIdx.x & 63, kg = lane / CQ, cq = lane % CQ;
  constexpr bool VEC = FORM == kWhole;
  const uint32_t unit = block_of() * 4 +
                        __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (unit >= units) return;
  const uint32_t nth = unit / ncb;
  const auto [b, h, hk] = lin_head(a, nth);
  const int64_t bh = nth;
  const int K = (int)a.K, k0 = kg * KR, c0 = (int)(unit - nth * ncb) * 4 * CQ + 4 * cq;
  const int64_t V = a.V;
  const int klim = K - k0 < 0 ? 0 : K - k0, clim = V - c0 > 4 ? 4 : (V - c0 < 0 ? 0 : (int)(V - c0));
  // lanes past K or V read row 0 or column 0 of their head, store nothing
  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + hk * a.q_h + (klim ? k0 : 0);
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h + (klim ? k0 : 0);
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_b + h * a.v_h + (clim ? c0 : 0);
  T* op = reinterpret_cast<T*>(a.o) + b * a.o_b + h * a.o_h + c0;
  const float* gp = a.g + b * a.g_b + h * a.g_h;
  const int64_t sbase = bh * K * V + c0;

  // Loads from rows and columns that exist, zeroes by selection: a branch
  // around each load would wait for it alone.
  float S[KR][4];
#pragma unroll
  for (int i = 0; i < KR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) S[i][j] = 0.0f;
  if (a.h0) {
    const float* hp = a.h0 + bh * K * V + (clim ? c0 : 0);
    const int back = clim ? 4 - clim : 0;
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const float* p = hp + (int64_t)(i < klim ? k0 + i : 0) * V;
      if constexpr (VEC) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
      } else if constexpr (FORM == kStateRows) {
        // fewer than four columns: the row's last four
        const f32x4a x = *reinterpret_cast<const f32x4a*>(p - back);
        S[i][0] = back & 2 ? (back & 1 ? x[3] : x[2]) : (back & 1 ? x[1] : x[0]);
        S[i][1] = back & 2 ? x[3] : (back & 1 ? x[2] : x[1]);
        S[i][2] = back & 1 ? x[3] : x[2];
        S[i][3] = x[3];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) S[i][j] = p[j < clim ? j : 0];
      }
    }
#pragma unroll
    for (int i = 0; i < KR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!(i < klim && j < clim)) S[i][j] = 0.0f;
  }

  Row<T, KR, VEC> nq, nk, q, k;
  Row<T, 4, VEC> nv, v;
  float ng = 0.0f;
  auto fetch = [&](int64_t t) {
    nq.load(qp + t * a.q_l, klim);
    nk.load(kp + t * a.k_l, klim);
    nv.load(vp + t * a.v_l, clim);
    ng = gp[t * a.g_l];
  };
  if (a.L > 0) fetch(0);
  for (int64_t t = 0; t < a.L; ++t) {
    q = nq; k = nk; v = nv;
    const float al = exp_acc(ng);
    if (t + 1 < a.L) fetch(t + 1);
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const float kf = k.get(i, klim), qf = q.get(i, klim);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[i][j] = __builtin_fmaf(kf, v.get(j, clim), S[i][j] * al);
        y[j] = __builtin_fmaf(qf, S[i][j], y[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = a.scale * sum_kg<CQ>(y[j]);
    if (kg == 0) {
      T* p = op + t * a.o_l;
      if (VEC && clim) {
        st_lanes<T, 4>(p, y);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < clim) stf(p + j, y[j]);
      }
    }
  }
  if (!a.h_last || !clim) return;
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    float* p = a.h_last + sbase + (int64_t)(k0 + i) * V;
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(p) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
    } else if (FORM == kStateRows && i < klim && clim == 4) {
      *reinterpret_cast<f32x4a*>(p) = f32x4a{S[i][0], S[i][1], S[i][2], S[i][3]};
    } else if (i < klim) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < clim) p[j] = S[i][j];
    }
  }
}

template <typename T, int CQ>
int launch(const LinArgs& a, hipStream_t s) {
  constexpr int kR = CQ / 4;  // rows of a lane for every 16 of K
  const int64_t ncb = cdiv64(a.V, 4 * CQ), units = a.B * a.Hv * ncb;
  if (units > 0x7fffffff || a.B > 0x7fffffff / a.Hv) return TSSM_ERR_UNSUPPORTED;
  const dim3 wgs = grid_of(cdiv64(units, 4));
  const int E = (int)sizeof(T);
  const int kr = (a.K <= 16 ? 1 : (a.K <= 32 ? 2 : (a.K <= 64 ? 4 : 8))) * kR;
  // every row of every operand starts on the widest access a lane makes
  const int64_t kb = kr * E < 16 ? kr * E : 16, vb = 4 * E;
  const bool vec =
      a.K == 64 / CQ * kr && a.V % 4 == 0 && aligned(a.q, kb) && aligned(a.k, kb) &&
      aligned(a.v, vb) && aligned(a.o, vb) && (!a.h0 || aligned(a.h0, 16)) &&
      (!a.h_last || aligned(a.h_last, 16)) &&
      (a.q_b | a.q_l | a.q_h | a.k_b | a.k_l | a.k_h) * E % kb == 0 &&
      (a.v_b | a.v_l | a.v_h | a.o_b | a.o_l | a.o_h) * E % vb == 0;
  // (the state's rows alone in pieces, S=327 H=16 100 x 128: 107 us, element by element 178;
  // S=280 128 x 117, whose last lanes move back to the row's last four: 121 and 187)
  const bool state = a.V >= 4 && (!a.h0 || aligned(a.h0, 4)) && (!a.h_last || aligned(a.h_last, 4));
#define TSSM_SEQ_AS(KR, FORM) \
  lin_seq_kernel<T, CQ, KR, FORM><<<wgs, 256, 0, s>>>(a, (uint32_t)ncb, (uint32_t)units)
#define TSSM_SEQ(KR)                            \
  if (vec) TSSM_SEQ_AS(KR, kWhole);             \
  else if (state) TSSM_SEQ_AS(KR, kStateRows);  \
  else TSSM_SEQ_AS(KR, kElements)
  if (a.K <= 16) { TSSM_SEQ(kR); }
  else if (a.K <= 32) { TSSM_SEQ(2 * kR); }
  else if (a.K <= 64) { TSSM_SEQ(4 * kR); }
  else { TSSM_SEQ(8 * kR); }
#undef TSSM_SEQ
#undef TSSM_SEQ_AS
  return launch_status();
}

// 16 columns a wave while that gives at most one wave to each SIMD.
template <typename T>
int columns(const LinArgs& a, hipStream_t s) {
  return a.B * a.Hv * cdiv64(a.V, 16) <= 1024 ? launch<T, 4>(a, s) : launch<T, 8>(a, s);
}

}  // namespace

int lin_seq_launch(int dtype, const LinArgs& a, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return columns<float>(a, s);
    case TSSM_BF16: return columns<bf16_t>(a, s);
    default: return columns<f16_t>(a, s);
  }
}

}  // namespace tssm
