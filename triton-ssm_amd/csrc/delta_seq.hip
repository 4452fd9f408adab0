// Gated delta rule, step by step: decoding (one step, the state in place) and
// short sequences.
//
// A wave owns 32 columns of one head's state for the whole call: lane
// (kg, cq) = (lane / 8, lane % 8) holds rows kg KR .. kg KR + KR - 1 of columns
// 4 cq .. 4 cq + 3 in registers.  Columns never meet (S^T k, the update and
// S^T q are all per column), so waves are independent; the sums over k run in
// each lane, then over the eight row groups by lane exchanges.  The state is
// read and written once whatever L is, 128 bytes of a row at a time.
//
// One step of many streams is bound by that traffic; a few steps of one stream
// by the launch and a chain of two such sums a step.
#include "delta.h"

namespace tssm {
namespace {

// Sum over the lanes that share lane % 8.
__device__ inline float sum_kg(float v) {
  v += dpp_mov<0x128>(v);  // row_ror:8
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

template <typename T, int KR, bool VEC>
__global__ __launch_bounds__(256) void delta_seq_kernel(DeltaArgs a, uint32_t ncb, int64_t units) {
  const int lane = threadIdx.x & 63, kg = lane >> 3, cq = lane & 7;
  const int64_t unit = (int64_t)blockIdx.x * 4 +
                       __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (unit >= units) return;
  const int64_t bh = unit / ncb, b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int K = (int)a.K, k0 = kg * KR, c0 = (int)(unit - bh * ncb) * 32 + 4 * cq;
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

  float S[KR][4];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) S[i][j] = 0.0f;
    if (a.h0 && i < klim) {
      const float* p = a.h0 + sbase + (int64_t)(k0 + i) * V;
      if constexpr (VEC) {
        if (clim) {
          const float4 x = *reinterpret_cast<const float4*>(p);
          S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < clim) S[i][j] = p[j];
      }
    }
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
    for (int j = 0; j < 4; ++j) r[j] = be * (v.get(j, clim) - sum_kg(r[j]));
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
    for (int j = 0; j < 4; ++j) y[j] = a.scale * sum_kg(y[j]);
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
  if (!a.h_last) return;
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    if (i < klim) {
      float* p = a.h_last + sbase + (int64_t)(k0 + i) * V;
      if (VEC && clim) {
        *reinterpret_cast<float4*>(p) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < clim) p[j] = S[i][j];
      }
    }
  }
}

template <typename T>
int launch(const DeltaArgs& a, hipStream_t s) {
  const int64_t ncb = cdiv64(a.V, 32), units = a.B * a.Hv * ncb, wgs = cdiv64(units, 4);
  if (wgs > 0x7fffffff) return TSSM_ERR_UNSUPPORTED;
  const int E = (int)sizeof(T);
  const int kr = a.K <= 16 ? 2 : (a.K <= 32 ? 4 : (a.K <= 64 ? 8 : 16));
  // every row of every operand starts on the widest access a lane makes
  const int64_t kb = kr * E < 16 ? kr * E : 16, vb = 4 * E;
  const bool vec =
      a.K == 8 * kr && a.V % 4 == 0 && aligned(a.q, kb) && aligned(a.k, kb) && aligned(a.v, vb) &&
      aligned(a.o, vb) && (!a.h0 || aligned(a.h0, 16)) && (!a.h_last || aligned(a.h_last, 16)) &&
      (a.q_b | a.q_l | a.q_h | a.k_b | a.k_l | a.k_h) * E % kb == 0 &&
      (a.v_b | a.v_l | a.v_h | a.o_b | a.o_l | a.o_h) * E % vb == 0;
#define TSSM_SEQ(KR)                                                                          \
  if (vec) delta_seq_kernel<T, KR, true><<<(unsigned)wgs, 256, 0, s>>>(a, (uint32_t)ncb, units); \
  else delta_seq_kernel<T, KR, false><<<(unsigned)wgs, 256, 0, s>>>(a, (uint32_t)ncb, units)
  if (kr == 2) { TSSM_SEQ(2); }
  else if (kr == 4) { TSSM_SEQ(4); }
  else if (kr == 8) { TSSM_SEQ(8); }
  else { TSSM_SEQ(16); }
#undef TSSM_SEQ
  return launch_status();
}

}  // namespace

int delta_seq_launch(int dtype, const DeltaArgs& a, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return launch<float>(a, s);
    case TSSM_BF16: return launch<bf16_t>(a, s);
    default: return launch<f16_t>(a, s);
  }
}

}  // namespace tssm
