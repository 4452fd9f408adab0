// Gated delta rule, step by step: decoding (one step, the state in place) and
// short sequences.
//
// A wave owns 4 CQ columns of one head's state for the whole call: lane
// (kg, cq) = (lane / CQ, lane % CQ) holds rows kg KR .. kg KR + KR - 1 of columns
// 4 cq .. 4 cq + 3 in registers.  Columns never meet (S^T k, the update and
// S^T q are all per column), so waves are independent; the sums over k run in
// each lane, then over the row groups by lane exchanges.  The state is read and
// written once whatever L is, 16 CQ bytes of a row at a time.
//
// One step of many streams is bound by that traffic (S=4096 H=32 K=128 V=64: 8.7
// GB at 5.2 TB/s, the rate of a copy); a few steps of one stream by the launch
// and a chain of two such sums a step, which CQ = 4 shortens where the waves of
// CQ = 8 leave SIMDs idle.
#include "delta.h"

namespace tssm {
namespace {

// Sum over the lanes that share lane % CQ.
template <int CQ>
__device__ inline float sum_kg(float v) {
  if constexpr (CQ == 4) v += dpp_mov<0x124>(v);  // row_ror:4
  v += dpp_mov<0x128>(v);                         // row_ror:8
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// N consecutive elements of T as floats; VEC: p is aligned to the widest access.
template <typename T, int N, bool VEC>
struct Row {
  static constexpr int kBytes = N * (int)sizeof(T);
  static constexpr int kW = VEC ? (kBytes < 16 ? kBytes : 16) : (int)sizeof(T);
  static constexpr int kN = kBytes / kW;
  typedef std::conditional_t<
      kW == 16, u32x4,
      std::conditional_t<kW == 8, uint2, std::conditional_t<kW == 4, uint32_t, uint16_t>>>
      word;
  union {
    word w[kN];
    T e[N];
  };
  // elements lim and up read element 0 (which exists) and count as zero
  __device__ inline void load(const T* p, int lim) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      w[i] = reinterpret_cast<const word*>(p)[VEC || i < lim ? i : 0];
  }
  __device__ inline float get(int i, int lim) const {
    return VEC || i < lim ? ldf(&e[i]) : 0.0f;
  }
};

template <typename T, int CQ, int KR, bool VEC>
__global__ __launch_bounds__(256) void delta_seq_kernel(DeltaArgs a, uint32_t ncb, uint32_t units) {
  const int lane = threadIdx.x & 63, kg = lane / CQ, cq = lane % CQ;
  const uint32_t unit = block_of() * 4 +
                        __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (unit >= units) return;
  const uint32_t nth = unit / ncb;
  const auto [b, h, hk] = head_of(a, nth);
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
  const float* ep = a.beta + b * a.be_b + h * a.be_h;
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
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const float* p = hp + (int64_t)(i < klim ? k0 + i : 0) * V;
      if constexpr (VEC) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
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
  float ng = 0.0f, ne = 0.0f;
  auto fetch = [&](int64_t t) {
    nq.load(qp + t * a.q_l, klim);
    nk.load(kp + t * a.k_l, klim);
    nv.load(vp + t * a.v_l, clim);
    ng = gp[t * a.g_l];
    ne = ep[t * a.be_l];
  };
  if (a.L > 0) fetch(0);
  for (int64_t t = 0; t < a.L; ++t) {
    q = nq; k = nk; v = nv;
    const float al = exp_acc(ng), be = ne;
    if (t + 1 < a.L) fetch(t + 1);
    float kf[KR], r[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      kf[i] = k.get(i, klim);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[i][j] *= al;
        r[j] = __builtin_fmaf(kf[i], S[i][j], r[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = be * (v.get(j, clim) - sum_kg<CQ>(r[j]));
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const float qf = q.get(i, klim);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[i][j] = __builtin_fmaf(kf[i], r[j], S[i][j]);
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
    } else if (i < klim) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < clim) p[j] = S[i][j];
    }
  }
}

template <typename T, int CQ>
int launch(const DeltaArgs& a, hipStream_t s) {
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
#define TSSM_SEQ(KR)                                                                       \
  if (vec)                                                                                 \
    delta_seq_kernel<T, CQ, KR, true><<<wgs, 256, 0, s>>>(a, (uint32_t)ncb, (uint32_t)units); \
  else                                                                                     \
    delta_seq_kernel<T, CQ, KR, false><<<wgs, 256, 0, s>>>(a, (uint32_t)ncb, (uint32_t)units)
  if (a.K <= 16) { TSSM_SEQ(kR); }
  else if (a.K <= 32) { TSSM_SEQ(2 * kR); }
  else if (a.K <= 64) { TSSM_SEQ(4 * kR); }
  else { TSSM_SEQ(8 * kR); }
#undef TSSM_SEQ
  return launch_status();
}

// 16 columns a wave while that gives at most one wave to each SIMD.
template <typename T>
int columns(const DeltaArgs& a, hipStream_t s) {
  return a.B * a.Hv * cdiv64(a.V, 16) <= 1024 ? launch<T, 4>(a, s) : launch<T, 8>(a, s);
}

}  // namespace

int delta_seq_launch(int dtype, const DeltaArgs& a, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return columns<float>(a, s);
    case TSSM_BF16: return columns<bf16_t>(a, s);
    default: return columns<f16_t>(a, s);
  }
}

}  // namespace tssm
