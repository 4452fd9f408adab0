// Group norm with an activation, channels last, and its gradients.
//
// x [N, S, C], G groups of Cg = C / G neighbouring channels; mean and variance
// over a group's S x Cg elements:
//   xhat = (x - mean) rstd,  z = xhat w + b,
//   y = act(z), or z act(gate) with a gate.
// Backward, with dz = dy act'(z) (or dy act(gate)) and e = dz w:
//   dx = rstd (e - mean(e) - xhat mean(e xhat)),  dw = sum dz xhat,
//   db = sum dz,  dgate = dy z act'(gate).
// Statistics and sums are fp32 and summed in a fixed order; the mean is kept in
// two parts (64 bits for the caller), since groups whose values almost agree
// need x - mean exactly, and the variance is formed about it.
//
// Three forms, all bound by memory where the problem is large:
// * rows (S = 1): a group in LG lanes' registers, one pass over the data (32768
//   rows of 16 x 64, gated, bf16: 43 us, 4.7 TB/s);
// * series (S > 1): blocks of positions in registers, their means and squared
//   deviations joined by Chan's formula, then a second pass over x (which the
//   last-level cache mostly serves); the backward needs only the sums of dz
//   and dz xhat of every channel, from which the group's two means follow;
// * groups wider than the registers of a wave (rows: 2048 channels, 512
//   without vector access) or rows wider than a workgroup's (series: 1024
//   accesses, 1024 channels without vector access): one workgroup a group,
//   element by element (with S = 0 the statistics of nothing, 0 / 0).  This form
//   is bound by its index arithmetic and by few workgroups: one series of 4096
//   positions of 30 groups of 50 channels, bf16, 990 us, with gradients 3550
//   (floors 5 and 10; in torch's elementary operations 220 and 680).
#include <type_traits>

#include "common.h"

namespace tssm {
namespace {

struct GnArgs {
  const void *x, *gate, *dy;
  const float *w, *b;
  double* mean;
  float* rstd;
  void *y, *dx, *dgate;
  float *dw, *db;
  float* ws;
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

// sum / count as a 32-bit value of its own: fused into the differences from it,
// the product would not be the mean that is kept (off by up to 2^-24 of it).
__device__ inline float mean_of(float sum, float inv) {
#pragma clang fp contract(off)
  return sum * inv;
}

// A variance that rounding put below 0 is 0 (NaN stays).
__device__ inline float not_below_0(float var) { return var < 0.0f ? 0.0f : var; }

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
  const int64_t ng = block_of(), n = ng / a.G, g = ng - n * a.G, E = a.S * a.Cg;
  if (n >= a.N) return;
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
  const float rstd = 1.0f / sqrtf(not_below_0(block_sum(s, red) / (float)E - lo * lo) + a.eps);
  if (a.mean && threadIdx.x == 0) {
    a.mean[ng] = (double)mean + (double)lo;
    a.rstd[ng] = rstd;
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
  const int64_t ng = block_of(), n = ng / a.G, g = ng - n * a.G, E = a.S * a.Cg;
  if (n >= a.N) return;
  const float mean = (float)a.mean[ng], rstd = a.rstd[ng];
  const float lo = (float)(a.mean[ng] - (double)mean);
  float s1 = 0.0f, s2 = 0.0f, xh;
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
  const int64_t C = a.G * a.Cg, c = (int64_t)block_of() * 64 + (threadIdx.x & 63);
  const int part = threadIdx.x >> 6;
  float sw = 0.0f, sb = 0.0f, xh;
  if (c < C) {
    for (int64_t i = part; i < a.N * a.S; i += 4) {
      const int64_t n = i / a.S, r = i - n * a.S, ng = n * a.G + c / a.Cg;
      const float mean = (float)a.mean[ng], lo = (float)(a.mean[ng] - (double)mean);
      const float dz = gn_dz<T>(a, n, r, c, mean, lo, a.rstd[ng], xh, false);
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

// ------------------------------------------------------------------ vectors
// VW elements of one access.
template <typename T, int VW>
struct Vec {
  typedef std::conditional_t<
      VW * sizeof(T) == 16, u32x4,
      std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>> word;
  union {
    word w;
    T e[VW];
  };
  __device__ inline void load(const T* p) { w = *reinterpret_cast<const word*>(p); }
  __device__ inline void store(T* p) const {
    __builtin_nontemporal_store(w, reinterpret_cast<word*>(p));
  }
  __device__ inline float get(int i) const { return ldf(&e[i]); }
  __device__ inline void set(int i, float x) { stf(&e[i], x); }
};
template <typename T> constexpr int kVw = 16 / (int)sizeof(T);

// Elements of a channel's weights, per lane: w (1 where there is none) and b.
template <int VW, int NV>
__device__ inline void gn_weights(const GnArgs& a, const int64_t (&ch)[NV], const bool (&in)[NV],
                                  float (&w)[NV][VW], float (&b)[NV][VW]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int v = 0; v < VW; ++v) {
      w[i][v] = a.w && in[i] ? a.w[ch[i] + v] : 1.0f;
      b[i][v] = a.b && in[i] ? a.b[ch[i] + v] : 0.0f;
    }
}

__device__ inline float gn_out(float z, float gate, bool gated, int act) {
  return gated ? z * act_f(gate, act) : act_f(z, act);
}
// dz of one element; dgate where there is a gate
__device__ inline float gn_dz1(float z, float dy, float gate, bool gated, int act, float& dgate) {
  float d;
  if (!gated) {
    act_df(z, act, d);
    return dy * d;
  }
  const float f = act_df(gate, act, d);
  dgate = dy * z * d;
  return dy * f;
}

// ------------------------------------------------------------------ rows
// S = 1.  A wave takes 64 / LG groups at once: GW neighbouring ones of RW rows.
template <int LG>
struct RowMap {
  int64_t g, row;  // this lane's group, and its row of the wave's first RW
  int rw;
  __device__ inline RowMap(const GnArgs& a, int gw, int64_t gb) {
    const int q = (threadIdx.x & 63) / LG;
    g = gb * gw + q % gw;
    rw = 64 / LG / gw;
    row = (int64_t)(threadIdx.x >> 6) * rw + q / gw;
  }
};

template <typename T, int VW, int LG, int NV, int U>
__global__ __launch_bounds__(256) void gn_row_fwd(GnArgs a, int gw, uint32_t ngb) {
  const uint32_t block = block_of(), rb = block / ngb;
  const RowMap<LG> m(a, gw, block - rb * ngb);
  const int l = threadIdx.x % LG;
  const int64_t step = 4 * m.rw, r0 = (int64_t)rb * U * step + m.row;
  const bool on = m.g < a.G, gated = a.gate != nullptr;
  int64_t ch[NV];
  bool in[NV];
  float w[NV][VW], b[NV][VW];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(i * LG + l) * VW;
    in[i] = on && c < a.Cg;
    ch[i] = in[i] ? m.g * a.Cg + c : 0;
  }
  gn_weights<VW, NV>(a, ch, in, w, b);
  Vec<T, VW> x[U][NV], gt[U][NV];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * step < a.N ? r0 + u * step : a.N - 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[u][i].load(reinterpret_cast<const T*>(a.x) + r * a.x_n + ch[i]);
      if (gated) gt[u][i].load(reinterpret_cast<const T*>(a.gate) + r * a.gt_n + ch[i]);
    }
  }
  const float inv = 1.0f / (float)a.Cg;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * step;
    float d[NV][VW], s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        d[i][v] = x[u][i].get(v);
        s += in[i] ? d[i][v] : 0.0f;
      }
    const float mean = mean_of(group_sum<LG>(s), inv);
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        d[i][v] = in[i] ? d[i][v] - mean : 0.0f;
        s += d[i][v];
        t = __builtin_fmaf(d[i][v], d[i][v], t);
      }
    const float lo = group_sum<LG>(s) * inv;
    const float var = __builtin_fmaf(-lo, lo, group_sum<LG>(t) * inv);
    const float rstd = __builtin_amdgcn_rsqf(not_below_0(var) + a.eps);
    if (r >= a.N) continue;
    if (a.mean && l == 0 && on) {
      a.mean[r * a.G + m.g] = (double)mean + (double)lo;
      a.rstd[r * a.G + m.g] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec<T, VW> y;
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        const float z = __builtin_fmaf((d[i][v] - lo) * rstd, w[i][v], b[i][v]);
        y.set(v, gn_out(z, gated ? gt[u][i].get(v) : 0.0f, gated, a.act));
      }
      if (in[i]) y.store(reinterpret_cast<T*>(a.y) + r * a.y_n + ch[i]);
    }
  }
}

// dw and db of the workgroup's rows go to ws[row block][2][C].
template <typename T, int VW, int LG, int NV>
__global__ __launch_bounds__(256) void gn_row_bwd(GnArgs a, int gw, uint32_t ngb, uint32_t nrb) {
  constexpr int kB = NV > 1 ? 4 : 2;  // sums of VW channels that meet at once
  __shared__ float red[kB][256][VW + 1];
  const uint32_t block = block_of(), rb = block / ngb;
  if (rb >= nrb) return;
  const RowMap<LG> m(a, gw, block - rb * ngb);
  const int l = threadIdx.x % LG;
  const int64_t step = 4 * m.rw;
  const bool on = m.g < a.G, gated = a.gate != nullptr;
  int64_t ch[NV];
  bool in[NV];
  float w[NV][VW], b[NV][VW], sw[NV][VW], sb[NV][VW];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (int64_t)(i * LG + l) * VW;
    in[i] = on && c < a.Cg;
    ch[i] = in[i] ? m.g * a.Cg + c : 0;
#pragma unroll
    for (int v = 0; v < VW; ++v) sw[i][v] = sb[i][v] = 0.0f;
  }
  gn_weights<VW, NV>(a, ch, in, w, b);
  struct In {
    Vec<T, VW> x[NV], dy[NV], gt[NV];
    double mean;
    float rstd;
  };
  const int64_t gs = on ? m.g : 0;
  auto load = [&](In& q, int64_t r) {
    if (r >= a.N) r = a.N - 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      q.x[i].load(reinterpret_cast<const T*>(a.x) + r * a.x_n + ch[i]);
      q.dy[i].load(reinterpret_cast<const T*>(a.dy) + r * a.dy_n + ch[i]);
      if (gated) q.gt[i].load(reinterpret_cast<const T*>(a.gate) + r * a.gt_n + ch[i]);
    }
    q.mean = a.mean[r * a.G + gs];
    q.rstd = a.rstd[r * a.G + gs];
  };
  const float inv = 1.0f / (float)a.Cg;
  auto row = [&](const In& q, int64_t r) {
    const float hi = (float)q.mean, lo = (float)(q.mean - (double)hi);
    const bool live = r < a.N;
    float e[NV][VW], xh[NV][VW], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec<T, VW> dg;
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        xh[i][v] = ((q.x[i].get(v) - hi) - lo) * q.rstd;
        const float z = __builtin_fmaf(xh[i][v], w[i][v], b[i][v]);
        float dgate = 0.0f;
        const float dz = gn_dz1(z, q.dy[i].get(v), gated ? q.gt[i].get(v) : 0.0f, gated, a.act,
                                dgate);
        dg.set(v, dgate);
        if (live) {
          sw[i][v] = __builtin_fmaf(dz, xh[i][v], sw[i][v]);
          sb[i][v] += dz;
        }
        e[i][v] = in[i] ? dz * w[i][v] : 0.0f;
        s1 += e[i][v];
        s2 = __builtin_fmaf(e[i][v], in[i] ? xh[i][v] : 0.0f, s2);
      }
      if (gated && in[i] && live) dg.store(reinterpret_cast<T*>(a.dgate) + r * a.dg_n + ch[i]);
    }
    const float m1 = group_sum<LG>(s1) * inv, m2 = group_sum<LG>(s2) * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec<T, VW> dx;
#pragma unroll
      for (int v = 0; v < VW; ++v)
        dx.set(v, q.rstd * ((e[i][v] - m1) - xh[i][v] * m2));
      if (in[i] && live) dx.store(reinterpret_cast<T*>(a.dx) + r * a.dx_n + ch[i]);
    }
  };
  In q0, q1;
  const int64_t hop = (int64_t)nrb * step;
  load(q0, (int64_t)rb * step + m.row);
  for (int64_t base = (int64_t)rb * step; base < a.N; base += 2 * hop) {
    load(q1, base + hop + m.row);
    row(q0, base + m.row);
    load(q0, base + 2 * hop + m.row);
    if (base + hop < a.N) row(q1, base + hop + m.row);
  }
  // sum i of w or b, 2 i or 2 i + 1, is one wave's of kB: a workgroup's lanes
  // that hold the same (group, place) are `lanes` <= 64 apart
  const int t = threadIdx.x, lanes = gw * LG, mine = t >> 6;
  const int64_t C = a.G * a.Cg;
  const bool head = mine < kB && (t & 63) < lanes;
#pragma unroll
  for (int q = 0; q < 2 * NV; q += kB) {
    if (q) __syncthreads();
#pragma unroll
    for (int k = 0; k < kB; ++k)
#pragma unroll
      for (int v = 0; v < VW; ++v)
        red[k][t][v] = k & 1 ? sb[(q + k) / 2][v] : sw[(q + k) / 2][v];
    __syncthreads();
    const int64_t c = (int64_t)((q + mine) / 2 * LG + l) * VW;
    if (head && on && c < a.Cg) {
      float x[VW] = {};
      for (int p = t & 63; p < 256; p += lanes)
#pragma unroll
        for (int v = 0; v < VW; ++v) x[v] += red[mine][p][v];
      float* part = a.ws + (int64_t)rb * 2 * C + (mine & 1) * C + m.g * a.Cg + c;
      if constexpr (VW % 4 == 0) {
#pragma unroll
        for (int v = 0; v < VW; v += 4)
          *reinterpret_cast<float4*>(part + v) = make_float4(x[v], x[v + 1], x[v + 2], x[v + 3]);
      } else {
#pragma unroll
        for (int v = 0; v < VW; ++v) part[v] = x[v];
      }
    }
  }
}

// out0, out1 [C] = sums of ws [np][2][C] over np, in a fixed order; for every
// blockIdx.z, np 2 C floats and out_step apart.
__global__ __launch_bounds__(256) void gn_sum_kernel(const float* ws, float* out0, float* out1,
                                                     int64_t C, int64_t np, int64_t out_step) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, p = threadIdx.x >> 4;
  const int64_t i = (int64_t)block_of() * 16 + c;
  ws += (int64_t)blockIdx.z * np * 2 * C;
  // eight loads in flight: np is in the hundreds and the workgroups few
  float s[8] = {};
  if (i < 2 * C) {
    int64_t k = p;
    for (; k + 112 < np; k += 128)
#pragma unroll
      for (int q = 0; q < 8; ++q) s[q] += ws[(k + 16 * q) * 2 * C + i];
    for (; k < np; k += 16) s[0] += ws[k * 2 * C + i];
  }
  red[p][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (p == 0 && i < 2 * C) {
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) all += red[k][c];
    if (i < C) out0[blockIdx.z * out_step + i] = all;
    else out1[blockIdx.z * out_step + i - C] = all;
  }
}

// ------------------------------------------------------------------ series
// tpr threads of a workgroup read a row, nc accesses each, 256 / tpr rows at
// once; a series is cut into nb blocks of `per` rows.
struct SeriesPlan {
  int tpr, nc;
  int64_t nb, per;
};
inline SeriesPlan series_plan(int64_t N, int64_t S, int64_t C, int vw) {
  SeriesPlan p;
  const int64_t acc = cdiv64(C, vw);
  p.tpr = 1;
  while (p.tpr < 256 && p.tpr < acc) p.tpr *= 2;
  p.nc = (int)cdiv64(acc, p.tpr);
  if (p.nc == 3) p.nc = 4;
  // about 1024 workgroups, each with 8 rows for every thread at least
  const int64_t rows = 256 / p.tpr, most = cdiv64(S, rows * 8), want = cdiv64(1024, N);
  p.nb = most < want ? most : want;
  p.per = cdiv64(cdiv64(S, p.nb), rows) * rows;
  p.nb = cdiv64(S, p.per);
  return p;
}

template <int VW, int NC>
struct Columns {
  int row;  // of the rows read at once
  int64_t ch[NC];
  bool in[NC];
  __device__ inline Columns(int64_t C, int tpr) {
    row = threadIdx.x / tpr;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int64_t c = (int64_t)(i * tpr + threadIdx.x % tpr) * VW;
      in[i] = c < C;
      ch[i] = in[i] ? c : 0;
    }
  }
};

// Sums over the workgroup of one value of each (thread, access), by group.
template <int VW, int NC>
__device__ inline void group_totals(const float (&x)[NC], float* red, float* sums,
                                    const GnArgs& a, int tpr) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NC; ++i) red[i * 256 + threadIdx.x] = x[i];
  __syncthreads();
  const int acc = (int)(a.Cg / VW), part = threadIdx.x & 15;  // 16 threads a group
  for (int g = threadIdx.x >> 4; g < a.G; g += 16) {
    float s = 0.0f;
    for (int k = part; k < acc * (256 / tpr); k += 16) {
      const int r = k / acc, p = g * acc + k - r * acc;  // row, access of the row
      s += red[p / tpr * 256 + r * tpr + p % tpr];
    }
    s = group_sum<16>(s);
    if (part == 0) sums[g] = s;
  }
  __syncthreads();
}

// Means and squared deviations of a row block's groups: ws [n][block][2][G], 64 bits.
template <typename T, int VW, int NC, int R>
__global__ __launch_bounds__(256) void gn_series_stats(GnArgs a, int tpr, int64_t nb,
                                                       int64_t per) {
  __shared__ float red[NC * 256];
  extern __shared__ double dyn[];
  double *mean = dyn, *sq = dyn + a.G;
  float *t0 = reinterpret_cast<float*>(dyn + 2 * a.G), *t1 = t0 + a.G, *t2 = t1 + a.G;
  const int64_t block = block_of(), n = block / nb, blk = block - n * nb;
  if (n >= a.N) return;
  const Columns<VW, NC> m(a.G * a.Cg, tpr);
  const int rows = 256 / tpr;
  const int64_t s0 = blk * per, s1 = s0 + per < a.S ? s0 + per : a.S;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n;
  for (int64_t at = s0; at < s1; at += R * rows) {
    const int64_t cnt = at + R * rows < s1 ? R * rows : s1 - at;  // rows of this turn
    Vec<T, VW> v[R][NC];
    float s[NC], d1[NC], d2[NC];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int64_t r = at + u * rows + m.row;
#pragma unroll
      for (int i = 0; i < NC; ++i) v[u][i].load(x + (r < s1 ? r : s0) * a.x_s + m.ch[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int k = 0; k < VW; ++k)
          s[i] += m.in[i] && u * rows + m.row < cnt ? v[u][i].get(k) : 0.0f;
    }
    group_totals<VW, NC>(s, red, t0, a, tpr);
    const float inv = 1.0f / (float)(cnt * a.Cg);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float mu = mean_of(t0[m.ch[i] / a.Cg], inv);
      d1[i] = d2[i] = 0.0f;
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int k = 0; k < VW; ++k) {
          const float d = m.in[i] && u * rows + m.row < cnt ? v[u][i].get(k) - mu : 0.0f;
          d1[i] += d;
          d2[i] = __builtin_fmaf(d, d, d2[i]);
        }
    }
    group_totals<VW, NC>(d1, red, t1, a, tpr);
    group_totals<VW, NC>(d2, red, t2, a, tpr);
    const double before = (double)((at - s0) * a.Cg), now = (double)(cnt * a.Cg);
    for (int g = threadIdx.x; g < a.G; g += 256) {
      const double mu = (double)mean_of(t0[g], inv), c = (double)t1[g] / now;
      const double q = (double)t2[g] - c * c * now;  // about the mean mu + c
      if (at == s0) {
        mean[g] = mu + c;
        sq[g] = q;
      } else {
        const double d = (mu + c) - mean[g];
        sq[g] += q + d * d * (before * now / (before + now));
        mean[g] += d * (now / (before + now));
      }
    }
  }
  double* out = reinterpret_cast<double*>(a.ws) + (n * nb + blk) * 2 * a.G;
  for (int g = threadIdx.x; g < a.G; g += 256) {  // (each its own)
    out[g] = mean[g];
    out[a.G + g] = sq[g];
  }
}

__device__ inline double sum16(double v) {
#pragma unroll
  for (int s = 1; s < 16; s *= 2) v += __shfl_xor(v, s);
  return v;
}

template <typename T, int VW, int NC>
__global__ __launch_bounds__(256) void gn_series_fwd(GnArgs a, int tpr, int64_t nb, int64_t per) {
  extern __shared__ double dyn[];
  float *hi = reinterpret_cast<float*>(dyn), *lo = hi + a.G, *rs = lo + a.G;
  const int64_t block = block_of(), n = block / nb, blk = block - n * nb;
  if (n >= a.N) return;
  {  // the blocks' statistics join, 16 threads a group
    const double* st = reinterpret_cast<const double*>(a.ws) + n * nb * 2 * a.G;
    const int part = threadIdx.x & 15;
    const double all = (double)(a.S * a.Cg);
    for (int g = threadIdx.x >> 4; g < a.G; g += 16) {
      double s = 0.0, q = 0.0;
      for (int64_t k = part; k < nb; k += 16) {
        const int64_t cnt = (k + 1) * per < a.S ? per : a.S - k * per;
        s += (double)(cnt * a.Cg) * st[k * 2 * a.G + g];
      }
      const double mean = sum16(s) / all;
      for (int64_t k = part; k < nb; k += 16) {
        const int64_t cnt = (k + 1) * per < a.S ? per : a.S - k * per;
        const double d = st[k * 2 * a.G + g] - mean;
        q += st[(k * 2 + 1) * a.G + g] + d * d * (double)(cnt * a.Cg);
      }
      const float rstd = 1.0f / sqrtf(not_below_0((float)(sum16(q) / all)) + a.eps);
      if (part == 0) {
        hi[g] = (float)mean;
        lo[g] = (float)(mean - (double)(float)mean);
        rs[g] = rstd;
        if (a.mean && blk == 0) {
          a.mean[n * a.G + g] = mean;
          a.rstd[n * a.G + g] = rstd;
        }
      }
    }
  }
  __syncthreads();
  const Columns<VW, NC> m(a.G * a.Cg, tpr);
  const bool gated = a.gate != nullptr;
  float w[NC][VW], b[NC][VW], h[NC], l[NC], r_[NC];
  gn_weights<VW, NC>(a, m.ch, m.in, w, b);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t g = m.ch[i] / a.Cg;
    h[i] = hi[g];
    l[i] = lo[g];
    r_[i] = rs[g];
  }
  const int64_t s1 = (blk + 1) * per < a.S ? (blk + 1) * per : a.S;
  const int rows = 256 / tpr;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n;
  const T* gt = reinterpret_cast<const T*>(a.gate) + n * a.gt_n;
  T* y = reinterpret_cast<T*>(a.y) + n * a.y_n;
#pragma unroll 4
  for (int64_t r = blk * per + m.row; r < s1; r += rows) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      Vec<T, VW> xv, gv, o;
      xv.load(x + r * a.x_s + m.ch[i]);
      if (gated) gv.load(gt + r * a.gt_s + m.ch[i]);
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const float z = __builtin_fmaf(((xv.get(k) - h[i]) - l[i]) * r_[i], w[i][k], b[i][k]);
        o.set(k, gn_out(z, gated ? gv.get(k) : 0.0f, gated, a.act));
      }
      if (m.in[i]) o.store(y + r * a.y_s + m.ch[i]);
    }
  }
}

// The row block's sums of dz xhat and dz for every channel: part [n][block][2][C].
template <typename T, int VW, int NC>
__global__ __launch_bounds__(256) void gn_series_sums(GnArgs a, int tpr, int64_t nb, int64_t per,
                                                      float* part) {
  __shared__ float red[256][VW + 1];
  const int64_t block = block_of(), n = block / nb, blk = block - n * nb, C = a.G * a.Cg;
  if (n >= a.N) return;
  const Columns<VW, NC> m(C, tpr);
  const bool gated = a.gate != nullptr;
  float w[NC][VW], b[NC][VW], h[NC], l[NC], r_[NC], sw[NC][VW], sb[NC][VW];
  gn_weights<VW, NC>(a, m.ch, m.in, w, b);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t g = n * a.G + m.ch[i] / a.Cg;
    h[i] = (float)a.mean[g];
    l[i] = (float)(a.mean[g] - (double)h[i]);
    r_[i] = a.rstd[g];
#pragma unroll
    for (int k = 0; k < VW; ++k) sw[i][k] = sb[i][k] = 0.0f;
  }
  const int64_t s1 = (blk + 1) * per < a.S ? (blk + 1) * per : a.S;
  const int rows = 256 / tpr;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n;
  const T* gt = reinterpret_cast<const T*>(a.gate) + n * a.gt_n;
  const T* dy = reinterpret_cast<const T*>(a.dy) + n * a.dy_n;
#pragma unroll 2
  for (int64_t r = blk * per + m.row; r < s1; r += rows) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      Vec<T, VW> xv, gv, dv;
      xv.load(x + r * a.x_s + m.ch[i]);
      dv.load(dy + r * a.dy_s + m.ch[i]);
      if (gated) gv.load(gt + r * a.gt_s + m.ch[i]);
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const float xh = ((xv.get(k) - h[i]) - l[i]) * r_[i];
        float dgate = 0.0f;
        const float dz = gn_dz1(__builtin_fmaf(xh, w[i][k], b[i][k]), dv.get(k),
                                gated ? gv.get(k) : 0.0f, gated, a.act, dgate);
        sw[i][k] = __builtin_fmaf(dz, xh, sw[i][k]);
        sb[i][k] += dz;
      }
    }
  }
  part += (n * nb + blk) * 2 * C;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VW; ++v) red[threadIdx.x][v] = k ? sb[i][v] : sw[i][v];
      __syncthreads();
      if (m.row == 0 && m.in[i]) {
#pragma unroll
        for (int v = 0; v < VW; ++v) {
          float s = 0.0f;
          for (int p = threadIdx.x; p < 256; p += tpr) s += red[p][v];
          part[k * C + m.ch[i] + v] = s;
        }
      }
    }
}

// dx (and dgate) from chan [n][2][C], the channels' sums of dz xhat and dz.
template <typename T, int VW, int NC>
__global__ __launch_bounds__(256) void gn_series_dx(GnArgs a, int tpr, int64_t nb, int64_t per,
                                                    const float* chan) {
  extern __shared__ double dyn[];
  float *m1 = reinterpret_cast<float*>(dyn), *m2 = m1 + a.G;
  const int64_t block = block_of(), n = block / nb, blk = block - n * nb, C = a.G * a.Cg;
  if (n >= a.N) return;
  {
    const float* cs = chan + n * 2 * C;
    const int part = threadIdx.x & 15;
    const float inv = 1.0f / (float)(a.S * a.Cg);
    for (int g = threadIdx.x >> 4; g < a.G; g += 16) {
      float s1 = 0.0f, s2 = 0.0f;
      for (int64_t k = part; k < a.Cg; k += 16) {
        const int64_t c = g * a.Cg + k;
        const float w = a.w ? a.w[c] : 1.0f;
        s2 = __builtin_fmaf(w, cs[c], s2);
        s1 = __builtin_fmaf(w, cs[C + c], s1);
      }
      s1 = group_sum<16>(s1);
      s2 = group_sum<16>(s2);
      if (part == 0) {
        m1[g] = s1 * inv;
        m2[g] = s2 * inv;
      }
    }
  }
  __syncthreads();
  const Columns<VW, NC> m(C, tpr);
  const bool gated = a.gate != nullptr;
  float w[NC][VW], b[NC][VW], h[NC], l[NC], r_[NC], e1[NC], e2[NC];
  gn_weights<VW, NC>(a, m.ch, m.in, w, b);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int64_t g = m.ch[i] / a.Cg;
    h[i] = (float)a.mean[n * a.G + g];
    l[i] = (float)(a.mean[n * a.G + g] - (double)h[i]);
    r_[i] = a.rstd[n * a.G + g];
    e1[i] = m1[g];
    e2[i] = m2[g];
  }
  const int64_t s1 = (blk + 1) * per < a.S ? (blk + 1) * per : a.S;
  const int rows = 256 / tpr;
  const T* x = reinterpret_cast<const T*>(a.x) + n * a.x_n;
  const T* gt = reinterpret_cast<const T*>(a.gate) + n * a.gt_n;
  const T* dy = reinterpret_cast<const T*>(a.dy) + n * a.dy_n;
  T* dx = reinterpret_cast<T*>(a.dx) + n * a.dx_n;
  T* dg = reinterpret_cast<T*>(a.dgate) + n * a.dg_n;
#pragma unroll 2
  for (int64_t r = blk * per + m.row; r < s1; r += rows) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      Vec<T, VW> xv, gv, dv, o, og;
      xv.load(x + r * a.x_s + m.ch[i]);
      dv.load(dy + r * a.dy_s + m.ch[i]);
      if (gated) gv.load(gt + r * a.gt_s + m.ch[i]);
#pragma unroll
      for (int k = 0; k < VW; ++k) {
        const float xh = ((xv.get(k) - h[i]) - l[i]) * r_[i];
        float dgate = 0.0f;
        const float dz = gn_dz1(__builtin_fmaf(xh, w[i][k], b[i][k]), dv.get(k),
                                gated ? gv.get(k) : 0.0f, gated, a.act, dgate);
        o.set(k, r_[i] * ((dz * w[i][k] - e1[i]) - xh * e2[i]));
        og.set(k, dgate);
      }
      if (m.in[i]) {
        o.store(dx + r * a.dx_s + m.ch[i]);
        if (gated) og.store(dg + r * a.dg_s + m.ch[i]);
      }
    }
  }
}

// ------------------------------------------------------------------ choice
// Whether every row of every operand is whole VW-wide accesses.
template <typename T>
bool gn_vector(const GnArgs& a) {
  constexpr int vw = kVw<T>;
  const void* ps[] = {a.x, a.gate, a.dy, a.y, a.dx, a.dgate};
  for (const void* p : ps)
    if (p && !aligned(p, 16)) return false;
  return a.Cg % vw == 0 && (a.x_n | a.x_s | a.gt_n | a.gt_s | a.y_n | a.y_s | a.dy_n | a.dy_s |
                            a.dx_n | a.dx_s | a.dg_n | a.dg_s) % vw == 0;
}
inline bool row_fits(int64_t S, int64_t Cg, int vw) {
  return S == 1 && cdiv64(Cg, vw) <= (vw == 8 ? 256 : 512);
}
inline bool series_fits(int64_t C, int64_t G, int vw) {
  return cdiv64(C, vw) <= 1024 && G <= 2048;
}
// Row blocks of the rows' backward: two workgroups on each CU, with two rows of
// every lane in flight (N = 8192 and 32768 of 16 x 64 channels, gated, bf16: 27
// and 64 us; with four 32 and 74, with one 29 and 81).
inline int64_t row_blocks(int64_t N, int64_t step, int64_t ngb) {
  const int64_t all = cdiv64(N, step), want = cdiv64(512, ngb);
  return all < want ? all : want;
}
struct RowPlan {
  int lg, nv, gw;
  int64_t ngb, step;  // group blocks of a row, rows of a workgroup
};
inline RowPlan row_plan(int64_t G, int64_t Cg, int vw) {
  RowPlan p;
  const int64_t acc = cdiv64(Cg, vw);
  p.lg = 1;
  while (p.lg < 64 && p.lg < acc) p.lg *= 2;
  p.nv = 1;
  while (p.nv * p.lg < acc) p.nv *= 2;
  p.gw = 1;
  while (p.gw < 64 / p.lg && p.gw < G) p.gw *= 2;
  p.ngb = cdiv64(G, p.gw);
  p.step = 4 * (64 / p.lg / p.gw);
  return p;
}
inline int64_t gn_ws_bytes(int64_t N, int64_t S, int64_t G, int64_t Cg) {
  if (N == 0 || S == 0) return 0;
  int64_t most = 0;
  const int vws[] = {1, 4, 8};
  for (const int vw : vws) {
    if (Cg % vw) continue;
    int64_t b = 0;
    if (row_fits(S, Cg, vw)) {
      const RowPlan p = row_plan(G, Cg, vw);
      b = row_blocks(N, p.step, p.ngb) * 2 * G * Cg * 4;
    } else if (series_fits(G * Cg, G, vw)) {
      const SeriesPlan p = series_plan(N, S, G * Cg, vw);
      const int64_t stats = N * p.nb * 2 * G * 8, sums = N * (p.nb + 1) * 2 * G * Cg * 4;
      b = stats > sums ? stats : sums;
    }
    most = b > most ? b : most;
  }
  return most;
}

template <typename T, int VW, typename F>
void row_dispatch(const RowPlan& p, F&& f) {
  using std::integral_constant;
#define TSSM_GN_ROW(LG, NV) f(integral_constant<int, LG>(), integral_constant<int, NV>())
  switch (p.lg) {
    case 1: TSSM_GN_ROW(1, 1); return;
    case 2: TSSM_GN_ROW(2, 1); return;
    case 4: TSSM_GN_ROW(4, 1); return;
    case 8: TSSM_GN_ROW(8, 1); return;
    case 16: TSSM_GN_ROW(16, 1); return;
    case 32: TSSM_GN_ROW(32, 1); return;
    default: break;
  }
  if (p.nv == 1) TSSM_GN_ROW(64, 1);
  else if (p.nv == 2) TSSM_GN_ROW(64, 2);
  else if (p.nv == 4) TSSM_GN_ROW(64, 4);
  else if constexpr (VW < 8) TSSM_GN_ROW(64, 8);
#undef TSSM_GN_ROW
}
template <typename F>
void series_dispatch(const SeriesPlan& p, F&& f) {
  if (p.nc == 1) f(std::integral_constant<int, 1>());
  else if (p.nc == 2) f(std::integral_constant<int, 2>());
  else f(std::integral_constant<int, 4>());
}

template <typename T, int VW>
int gn_fwd_vw(const GnArgs& a, hipStream_t s) {
  const int64_t C = a.G * a.Cg;
  if (row_fits(a.S, a.Cg, VW)) {
    const RowPlan p = row_plan(a.G, a.Cg, VW);
    row_dispatch<T, VW>(p, [&](auto lg, auto nv) {
      constexpr int LG = decltype(lg)::value, NV = decltype(nv)::value;
      // rows in flight: where a row is one access of a lane, one is too few
      constexpr int U = NV == 1 ? 4 : (NV == 2 ? 2 : 1);
      gn_row_fwd<T, VW, LG, NV, U>
          <<<grid_of(p.ngb * cdiv64(a.N, U * p.step)), 256, 0, s>>>(a, p.gw, (uint32_t)p.ngb);
    });
  } else if (a.S && series_fits(C, a.G, VW)) {
    const SeriesPlan p = series_plan(a.N, a.S, C, VW);
    series_dispatch(p, [&](auto nc) {
      constexpr int NC = decltype(nc)::value, R = VW * NC >= 16 ? 2 : (VW * NC >= 8 ? 4 : 8);
      const dim3 wgs = grid_of(a.N * p.nb);
      gn_series_stats<T, VW, NC, R><<<wgs, 256, (size_t)a.G * 28, s>>>(a, p.tpr, p.nb, p.per);
      gn_series_fwd<T, VW, NC><<<wgs, 256, (size_t)a.G * 12 + 8, s>>>(a, p.tpr, p.nb, p.per);
    });
  } else {
    gn_fwd_kernel<T><<<grid_of(a.N * a.G), 256, 0, s>>>(a);
  }
  return launch_status();
}
template <typename T>
int gn_fwd(const GnArgs& a, hipStream_t s) {
  return gn_vector<T>(a) ? gn_fwd_vw<T, kVw<T>>(a, s) : gn_fwd_vw<T, 1>(a, s);
}

template <typename T, int VW>
int gn_bwd_vw(const GnArgs& a, hipStream_t s) {
  const int64_t C = a.G * a.Cg;
  const dim3 sums = grid_of(cdiv64(2 * C, 16));
  if (a.N * a.S == 0) {
    gn_sum_kernel<<<sums, 256, 0, s>>>(nullptr, a.dw, a.db, C, 0, 0);
  } else if (row_fits(a.S, a.Cg, VW)) {
    const RowPlan p = row_plan(a.G, a.Cg, VW);
    const int64_t nrb = row_blocks(a.N, p.step, p.ngb);
    row_dispatch<T, VW>(p, [&](auto lg, auto nv) {
      gn_row_bwd<T, VW, decltype(lg)::value, decltype(nv)::value>
          <<<grid_of(p.ngb * nrb), 256, 0, s>>>(a, p.gw, (uint32_t)p.ngb, (uint32_t)nrb);
    });
    gn_sum_kernel<<<sums, 256, 0, s>>>(a.ws, a.dw, a.db, C, nrb, 0);
  } else if (series_fits(C, a.G, VW)) {
    const SeriesPlan p = series_plan(a.N, a.S, C, VW);
    float* chan = a.ws + a.N * p.nb * 2 * C;
    series_dispatch(p, [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      const dim3 wgs = grid_of(a.N * p.nb);
      gn_series_sums<T, VW, NC><<<wgs, 256, 0, s>>>(a, p.tpr, p.nb, p.per, a.ws);
      for (int64_t n = 0; n < a.N; n += 65535) {
        const unsigned ns = (unsigned)(a.N - n < 65535 ? a.N - n : 65535);
        gn_sum_kernel<<<dim3(sums.x, sums.y, ns), 256, 0, s>>>(a.ws + n * p.nb * 2 * C, chan + n * 2 * C,
                                                       chan + n * 2 * C + C, C, p.nb, 2 * C);
      }
      gn_series_dx<T, VW, NC><<<wgs, 256, (size_t)a.G * 8 + 8, s>>>(a, p.tpr, p.nb, p.per, chan);
    });
    gn_sum_kernel<<<sums, 256, 0, s>>>(chan, a.dw, a.db, C, a.N, 0);
  } else {
    gn_dx_kernel<T><<<grid_of(a.N * a.G), 256, 0, s>>>(a);
    gn_dw_kernel<T><<<grid_of(cdiv64(C, 64)), 256, 0, s>>>(a);
  }
  return launch_status();
}
template <typename T>
int gn_bwd(const GnArgs& a, hipStream_t s) {
  return gn_vector<T>(a) ? gn_bwd_vw<T, kVw<T>>(a, s) : gn_bwd_vw<T, 1>(a, s);
}

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int64_t tssm_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t G, int64_t Cg) {
  if (N < 0 || S < 0 || G <= 0 || Cg <= 0) return TSSM_ERR_SHAPE;
  return gn_ws_bytes(N, S, G, Cg) + 256;
}

extern "C" int tssm_group_norm_act_fwd(int dtype, int act, const void* x, const float* w,
                                       const float* b, const void* gate, void* y, double* mean,
                                       float* rstd, int64_t N, int64_t S, int64_t G, int64_t Cg,
                                       int64_t sx_n, int64_t sx_s, int64_t sgt_n, int64_t sgt_s,
                                       int64_t sy_n, int64_t sy_s, float eps, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(act == TSSM_ACT_NONE || act == TSSM_ACT_SILU, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(N >= 0 && S >= 0 && G > 0 && Cg > 0, TSSM_ERR_SHAPE);
  if (N == 0) return TSSM_OK;
  TSSM_CHECK((S == 0 || (x && y)) && !mean == !rstd, TSSM_ERR_NULL);
  if (S == 0 && !mean) return TSSM_OK;
  TSSM_CHECK(N <= 0x7fffffff / G && G * Cg <= 0x7fffffff, TSSM_ERR_UNSUPPORTED);
  GnArgs a = {};
  a.x = x; a.w = w; a.b = b; a.gate = gate; a.y = y; a.mean = mean; a.rstd = rstd;
  a.N = N; a.S = S; a.G = G; a.Cg = Cg;
  a.x_n = sx_n; a.x_s = sx_s; a.gt_n = sgt_n; a.gt_s = sgt_s; a.y_n = sy_n; a.y_s = sy_s;
  a.eps = eps; a.act = act;
  TSSM_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= gn_ws_bytes(N, S, G, Cg),
             TSSM_ERR_WORKSPACE);
  a.ws = reinterpret_cast<float*>(workspace);
  switch (dtype) {
    case TSSM_F32: return gn_fwd<float>(a, as_stream(stream));
    case TSSM_BF16: return gn_fwd<bf16_t>(a, as_stream(stream));
    default: return gn_fwd<f16_t>(a, as_stream(stream));
  }
}

extern "C" int tssm_group_norm_act_bwd(int dtype, int act, const void* dy, const void* x,
                                       const double* mean, const float* rstd, const float* w,
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
  TSSM_CHECK(N <= 0x7fffffff / G && G * Cg <= 0x7fffffff, TSSM_ERR_UNSUPPORTED);
  GnArgs a = {};
  a.dy = dy; a.x = x; a.w = w; a.b = b; a.gate = gate; a.dx = dx; a.dw = dw; a.db = db;
  a.mean = const_cast<double*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dgate = dgate;
  a.N = N; a.S = S; a.G = G; a.Cg = Cg;
  a.dy_n = sdy_n; a.dy_s = sdy_s; a.x_n = sx_n; a.x_s = sx_s; a.gt_n = sgt_n; a.gt_s = sgt_s;
  a.dx_n = sdx_n; a.dx_s = sdx_s; a.dg_n = sdg_n; a.dg_s = sdg_s;
  a.act = act;
  TSSM_CHECK(N == 0 || S == 0 || (workspace && aligned(workspace, 256) &&
                                  workspace_bytes >= gn_ws_bytes(N, S, G, Cg)),
             TSSM_ERR_WORKSPACE);
  a.ws = reinterpret_cast<float*>(workspace);
  switch (dtype) {
    case TSSM_F32: return gn_bwd<float>(a, as_stream(stream));
    case TSSM_BF16: return gn_bwd<bf16_t>(a, as_stream(stream));
    default: return gn_bwd<f16_t>(a, as_stream(stream));
  }
}
