// Group norm with an activation, channels last, and its gradients.
//
// x [N, S, C], G groups of Cg = C / G neighbouring channels; mean and variance
// over a group's S x Cg elements:
//   xhat = (x - mean) rstd,  z = xhat w + b,
//   y = act(z), or z act(gate) with a gate.
// Backward, with dz = dy act'(z) (or dy act(gate)) and e = dz w:
//   dx = rstd (e - mean(e) - xhat mean(e xhat)),  dw = sum dz xhat,
//   db = sum dz,  dgate = dy z act'(gate).
// Statistics and sums are fp32; the variance is formed about the mean.
#include "common.h"

namespace tssm {
namespace {

struct GnArgs {
  const void *x, *gate, *dy;
  const float *w, *b;
  float *mean, *rstd;
  void *y, *dx, *dgate;
  float *dw, *db;
  float* lo;  // backward: what mean's rounding left, [N, G]
  int64_t N, S, G, Cg;
  int64_t x_n, x_s, gt_n, gt_s, y_n, y_s, dy_n, dy_s, dx_n, dx_s, dg_n, dg_s;
  float eps;
  int act;
};

__device__ inline float sigmoid_f(float x) {
  return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-x * kLog2e));
}
__device__ inline float act_f(float x, int act) { return act ? x * sigmoid_f(x) : x; }
// act(x) and its derivative
__device__ inline float act_df(float x, int act, float& d) {
  if (!act) {
    d = 1.0f;
    return x;
  }
  const float s = sigmoid_f(x);
  d = s * __builtin_fmaf(x, 1.0f - s, 1.0f);
  return x * s;
}

__device__ inline float block_sum(float v, float* red) {
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T>
__global__ __launch_bounds__(256) void gn_fwd_kernel(GnArgs a) {
  __shared__ float red[4];
  const int64_t n = blockIdx.x / a.G, g = blockIdx.x - n * a.G, E = a.S * a.Cg;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n + g * a.Cg;
  const T* gt = reinterpret_cast<const T*>(a.gate) + n * a.gt_n + g * a.Cg;
  T* y = reinterpret_cast<T*>(a.y) + n * a.y_n + g * a.Cg;
  float s = 0.0f;
  for (int64_t e = threadIdx.x; e < E; e += 256) s += ldf(x + e / a.Cg * a.x_s + e % a.Cg);
  const float mean = block_sum(s, red) / (float)E;
  // what mean's rounding left: groups whose values almost agree need it
  s = 0.0f;
  float t = 0.0f;
  for (int64_t e = threadIdx.x; e < E; e += 256) {
    const float d = ldf(x + e / a.Cg * a.x_s + e % a.Cg) - mean;
    t += d;
    s = __builtin_fmaf(d, d, s);
  }
  const float lo = block_sum(t, red) / (float)E;
  const float rstd = 1.0f / sqrtf(block_sum(s, red) / (float)E - lo * lo + a.eps);
  if (a.mean && threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = rstd;
  }
  for (int64_t e = threadIdx.x; e < E; e += 256) {
    const int64_t r = e / a.Cg, c = e % a.Cg;
    float z = ((ldf(x + r * a.x_s + c) - mean) - lo) * rstd;
    if (a.w) z *= a.w[g * a.Cg + c];
    if (a.b) z += a.b[g * a.Cg + c];
    stf(y + r * a.y_s + c, a.gate ? z * act_f(ldf(gt + r * a.gt_s + c), a.act) : act_f(z, a.act));
  }
}

// xhat and dz of one element; dgate is written
template <typename T>
__device__ inline float gn_dz(const GnArgs& a, int64_t n, int64_t r, int64_t c, float mean,
                              float lo, float rstd, float& xhat, bool put) {
  xhat = ((ldf(reinterpret_cast<const T*>(a.x) + n * a.x_n + r * a.x_s + c) - mean) - lo) * rstd;
  float z = xhat, d;
  if (a.w) z *= a.w[c];
  if (a.b) z += a.b[c];
  const float dy = ldf(reinterpret_cast<const T*>(a.dy) + n * a.dy_n + r * a.dy_s + c);
  if (!a.gate) {
    act_df(z, a.act, d);
    return dy * d;
  }
  const float f =
      act_df(ldf(reinterpret_cast<const T*>(a.gate) + n * a.gt_n + r * a.gt_s + c), a.act, d);
  if (put) stf(reinterpret_cast<T*>(a.dgate) + n * a.dg_n + r * a.dg_s + c, dy * z * d);
  return dy * f;
}

template <typename T>
__global__ __launch_bounds__(256) void gn_dx_kernel(GnArgs a) {
  __shared__ float red[4];
  const int64_t n = blockIdx.x / a.G, g = blockIdx.x - n * a.G, E = a.S * a.Cg;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
  float s1 = 0.0f, s2 = 0.0f, xh;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n + g * a.Cg;
  for (int64_t e = threadIdx.x; e < E; e += 256)
    s1 += ldf(x + e / a.Cg * a.x_s + e % a.Cg) - mean;
  const float lo = block_sum(s1, red) / (float)E;
  if (threadIdx.x == 0) a.lo[blockIdx.x] = lo;
  s1 = 0.0f;
  for (int64_t e = threadIdx.x; e < E; e += 256) {
    const int64_t r = e / a.Cg, c = g * a.Cg + e % a.Cg;
    float ew = gn_dz<T>(a, n, r, c, mean, lo, rstd, xh, true);
    if (a.w) ew *= a.w[c];
    s1 += ew;
    s2 = __builtin_fmaf(ew, xh, s2);
  }
  const float m1 = block_sum(s1, red) / (float)E, m2 = block_sum(s2, red) / (float)E;
  for (int64_t e = threadIdx.x; e < E; e += 256) {
    const int64_t r = e / a.Cg, c = g * a.Cg + e % a.Cg;
    float ew = gn_dz<T>(a, n, r, c, mean, lo, rstd, xh, false);
    if (a.w) ew *= a.w[c];
    stf(reinterpret_cast<T*>(a.dx) + n * a.dx_n + r * a.dx_s + c, rstd * (ew - m1 - xh * m2));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void gn_dw_kernel(GnArgs a) {
  __shared__ float red[2][4][64];
  const int64_t C = a.G * a.Cg, c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int part = threadIdx.x >> 6;
  float sw = 0.0f, sb = 0.0f, xh;
  if (c < C) {
    for (int64_t i = part; i < a.N * a.S; i += 4) {
      const int64_t n = i / a.S, r = i - n * a.S, ng = n * a.G + c / a.Cg;
      const float dz = gn_dz<T>(a, n, r, c, a.mean[ng], a.lo[ng], a.rstd[ng], xh, false);
      sb += dz;
      sw = __builtin_fmaf(dz, xh, sw);
    }
  }
  red[0][part][threadIdx.x & 63] = sw;
  red[1][part][threadIdx.x & 63] = sb;
  __syncthreads();
  if (part == 0 && c < C) {
    const int l = threadIdx.x;
    a.dw[c] = (red[0][0][l] + red[0][1][l]) + (red[0][2][l] + red[0][3][l]);
    a.db[c] = (red[1][0][l] + red[1][1][l]) + (red[1][2][l] + red[1][3][l]);
  }
}

template <typename T>
int gn_fwd(const GnArgs& a, hipStream_t s) {
  gn_fwd_kernel<T><<<(unsigned)(a.N * a.G), 256, 0, s>>>(a);
  return launch_status();
}
template <typename T>
int gn_bwd(const GnArgs& a, hipStream_t s) {
  if (a.N * a.S > 0) gn_dx_kernel<T><<<(unsigned)(a.N * a.G), 256, 0, s>>>(a);
  gn_dw_kernel<T><<<(unsigned)cdiv64(a.G * a.Cg, 64), 256, 0, s>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int64_t tssm_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t G, int64_t Cg) {
  if (N < 0 || S < 0 || G <= 0 || Cg <= 0) return TSSM_ERR_SHAPE;
  return cdiv64(N * G * 4, 256) * 256 + 256;
}

extern "C" int tssm_group_norm_act_fwd(int dtype, int act, const void* x, const float* w,
                                       const float* b, const void* gate, void* y, float* mean,
                                       float* rstd, int64_t N, int64_t S, int64_t G, int64_t Cg,
                                       int64_t sx_n, int64_t sx_s, int64_t sgt_n, int64_t sgt_s,
                                       int64_t sy_n, int64_t sy_s, float eps, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(act == TSSM_ACT_NONE || act == TSSM_ACT_SILU, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(N >= 0 && S >= 0 && G > 0 && Cg > 0, TSSM_ERR_SHAPE);
  if (N == 0 || S == 0) return TSSM_OK;
  TSSM_CHECK(x && y && !mean == !rstd, TSSM_ERR_NULL);
  TSSM_CHECK(N <= 0x7fffffff / G, TSSM_ERR_UNSUPPORTED);
  GnArgs a = {};
  a.x = x; a.w = w; a.b = b; a.gate = gate; a.y = y; a.mean = mean; a.rstd = rstd;
  a.N = N; a.S = S; a.G = G; a.Cg = Cg;
  a.x_n = sx_n; a.x_s = sx_s; a.gt_n = sgt_n; a.gt_s = sgt_s; a.y_n = sy_n; a.y_s = sy_s;
  a.eps = eps; a.act = act;
  (void)workspace;
  (void)workspace_bytes;
  switch (dtype) {
    case TSSM_F32: return gn_fwd<float>(a, as_stream(stream));
    case TSSM_BF16: return gn_fwd<bf16_t>(a, as_stream(stream));
    default: return gn_fwd<f16_t>(a, as_stream(stream));
  }
}

extern "C" int tssm_group_norm_act_bwd(int dtype, int act, const void* dy, const void* x,
                                       const float* mean, const float* rstd, const float* w,
                                       const float* b, const void* gate, void* dx, float* dw,
                                       float* db, void* dgate, int64_t N, int64_t S, int64_t G,
                                       int64_t Cg, int64_t sdy_n, int64_t sdy_s, int64_t sx_n,
                                       int64_t sx_s, int64_t sgt_n, int64_t sgt_s, int64_t sdx_n,
                                       int64_t sdx_s, int64_t sdg_n, int64_t sdg_s,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(act == TSSM_ACT_NONE || act == TSSM_ACT_SILU, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(N >= 0 && S >= 0 && G > 0 && Cg > 0, TSSM_ERR_SHAPE);
  TSSM_CHECK(dw && db, TSSM_ERR_NULL);
  TSSM_CHECK(N == 0 || S == 0 || (dy && x && mean && rstd && dx && !gate == !dgate), TSSM_ERR_NULL);
  TSSM_CHECK(N <= 0x7fffffff / G, TSSM_ERR_UNSUPPORTED);
  GnArgs a = {};
  a.dy = dy; a.x = x; a.w = w; a.b = b; a.gate = gate; a.dx = dx; a.dw = dw; a.db = db;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dgate = dgate;
  a.N = N; a.S = S; a.G = G; a.Cg = Cg;
  a.dy_n = sdy_n; a.dy_s = sdy_s; a.x_n = sx_n; a.x_s = sx_s; a.gt_n = sgt_n; a.gt_s = sgt_s;
  a.dx_n = sdx_n; a.dx_s = sdx_s; a.dg_n = sdg_n; a.dg_s = sdg_s;
  a.act = act;
  TSSM_CHECK(N == 0 || S == 0 || (workspace && workspace_bytes >= N * G * 4), TSSM_ERR_WORKSPACE);
  a.lo = reinterpret_cast<float*>(workspace);
  switch (dtype) {
    case TSSM_F32: return gn_bwd<float>(a, as_stream(stream));
    case TSSM_BF16: return gn_bwd<bf16_t>(a, as_stream(stream));
    default: return gn_bwd<f16_t>(a, as_stream(stream));
  }
}
