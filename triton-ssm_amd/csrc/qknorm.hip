// Norm of queries and keys for each head and rotation by their positions, in one
// pass, and its gradients.
//
// A row x of K channels, r = (sum x^2 / K + eps)^-1/2, (sum x^2 + eps)^-1/2 or 1:
//   n = r x w,   (n_a, n_b) -> amplitude (n_a c - n_b s, n_a s + n_b c)
// for the R/2 pairs of the first R channels, (j, j + R/2) or (2 j, 2 j + 1), with
// c, s of the angle pos freq_j; the other channels stay n.  Gradients, with d the
// output's gradient turned back by the same angle and m = 1/K, 1 or 0:
//   dw = sum d r x,   e = d w,   dx = r (e - m r^2 x sum(e x)).
//
// All of it is bound by HBM: every row is read once and written once.  The angles,
// whose product and reduction to one turn take 64 bits (a position of 10^6 at a
// rate of 1 leaves 20 bits of an fp32 angle before the point), are formed once
// for a token by the workgroup and shared by its heads through LDS.
//
// The forward reaches 4.3 to 4.8 TB/s (B=8 L=4096, 16 + 16 heads of 64, bf16: 56 us;
// B=4 L=4096, 16 + 8 of 128: 47), a copy 5.15.  It is waves in flight that decide: rows
// are asked for before the angles are formed, and the weights, which both would hold 32
// registers, are in LDS (with them in registers and the next rows ahead, 200 registers
// and two waves a SIMD, 65 us each).
//
// A workgroup has TB tokens; a group of LG lanes holds one row, TB groups beside
// each other take tokens, the others heads, so a lane keeps its token's cosines in
// registers over the heads it goes through.  A lane holds both members of its
// pairs: two vectors of 16 (8, 4) bytes R/2 apart (or next to each other), or, where sizes
// or alignment do not fit those, single elements.
#include "planes.h"

namespace tssm {
namespace {

struct QkArgs {
  const void *q, *k;       // inputs (the forward's in the backward too)
  const void *dq, *dk;     // backward: gradients of the outputs
  void *yq, *yk;           // outputs, or gradients of the inputs
  const void* pos;
  const double* freq;
  const float *wq, *wk;
  float* part;             // backward with weights: [workgroups][2][K]
  float *dwq, *dwk;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, dq_b, dq_l, dq_h, dk_b, dk_l, dk_h;
  int64_t yq_b, yq_l, yq_h, yk_b, yk_l, yk_h, p_b, p_l;
  uint32_t tokens, L;
  int Hq, H, K, R, TB, HS;  // H: heads of q and k; HS: heads side by side
  int norm, interleaved, pos_type;
  uint32_t blocks;          // blocks of TB tokens
  float eps, amplitude;
};

enum { kHalf, kNeighbours, kSingle };  // how a lane's elements lie

__device__ inline double position(const QkArgs& a, int64_t at) {
  switch (a.pos_type) {
    case TSSM_POS_F32: return (double)reinterpret_cast<const float*>(a.pos)[at];
    case TSSM_POS_F64: return reinterpret_cast<const double*>(a.pos)[at];
    case TSSM_POS_I32: return (double)reinterpret_cast<const int32_t*>(a.pos)[at];
    default: return (double)reinterpret_cast<const int64_t*>(a.pos)[at];
  }
}

// Lanes, pairs of a lane (NS) and the elements' places for one form.
template <typename T, int FORM, int LG_, int NS>
struct Form {
  // (single elements: that a Part has 32 bytes keeps 16-bit ones from being packed by two
  // in registers, 142 against 112 us for 190 MB of rows of 100)
  static constexpr int LG = LG_, VE = FORM == kSingle ? 16 / (int)sizeof(T) : NS, NP = NS;
  // first and second element of a lane's pair i; the second may be past K
  static __device__ inline void places(const QkArgs& a, int l, int i, int& ea, int& eb) {
    const int half = a.R / 2;
    if constexpr (FORM == kSingle) {
      const int s = l + LG * i;
      const bool rot = s < half;
      ea = rot ? (a.interleaved ? 2 * s : s) : 2 * s;
      eb = rot && !a.interleaved ? s + half : 2 * s + 1;
    } else if constexpr (FORM == kNeighbours) {
      ea = 2 * (l * VE + i);
      eb = ea + 1;
    } else {
      const bool rot = l * VE < half;
      ea = rot ? l * VE + i : 2 * l * VE + i;
      eb = rot ? ea + half : ea + VE;
    }
  }
};

// A lane's part of a row, as it lies in memory.
template <typename T, int FORM, int LG, int NS>
struct Part {
  typedef Form<T, FORM, LG, NS> F;
  typedef std::conditional_t<F::VE * sizeof(T) == 16, u32x4,
                             std::conditional_t<F::VE * sizeof(T) == 8, u32x2v, uint32_t>> word;
  union {
    word v[2];
    T e[FORM == kSingle ? 2 * NS : 2 * F::VE];
  };
  __device__ inline void load(const QkArgs& a, const T* p, int l, bool on) {
    if constexpr (FORM == kSingle) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        int ea, eb;
        F::places(a, l, i, ea, eb);
        e[2 * i] = p[ea < a.K ? ea : 0];
        e[2 * i + 1] = p[eb < a.K ? eb : 0];
      }
    } else {
      int ea, eb, x;
      F::places(a, l, 0, ea, x);
      if constexpr (FORM == kHalf) eb = x;
      else eb = ea + F::VE;
      v[0] = *reinterpret_cast<const word*>(p + (on ? ea : 0));
      v[1] = *reinterpret_cast<const word*>(p + (on ? eb : 0));
    }
  }
  // pairs as floats, zero past K
  __device__ inline void get(const QkArgs& a, int l, bool on, float* x, float* y) const {
#pragma unroll
    for (int i = 0; i < F::NP; ++i) {
      if constexpr (FORM == kSingle) {
        int ea, eb;
        F::places(a, l, i, ea, eb);
        x[i] = ea < a.K ? ldf(&e[2 * i]) : 0.0f;
        y[i] = eb < a.K ? ldf(&e[2 * i + 1]) : 0.0f;
      } else {
        x[i] = on ? ldf(&e[FORM == kHalf ? i : 2 * i]) : 0.0f;
        y[i] = on ? ldf(&e[FORM == kHalf ? F::VE + i : 2 * i + 1]) : 0.0f;
      }
    }
  }
  __device__ inline void put(const QkArgs& a, T* p, int l, bool on, const float* x,
                             const float* y) {
#pragma unroll
    for (int i = 0; i < F::NP; ++i) {
      const bool pairs = FORM != kHalf;
      stf(&e[pairs ? 2 * i : i], x[i]);
      stf(&e[pairs ? 2 * i + 1 : F::VE + i], y[i]);
    }
    if constexpr (FORM == kSingle) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        int ea, eb;
        F::places(a, l, i, ea, eb);
        if (ea < a.K) p[ea] = e[2 * i];
        if (eb < a.K) p[eb] = e[2 * i + 1];
      }
    } else if (on) {
      int ea, eb, x0;
      F::places(a, l, 0, ea, x0);
      if constexpr (FORM == kHalf) eb = x0;
      else eb = ea + F::VE;
      *reinterpret_cast<word*>(p + ea) = v[0];
      *reinterpret_cast<word*>(p + eb) = v[1];
    }
  }
};

// Sum over a group's lanes.
template <int LG>
__device__ inline float row_sum(float v) { return group_sum<LG>(v); }

constexpr int kThreads = 256, kTable = 1024;  // entries of the table of angles

template <typename T, int FORM, int LG, int NS, bool BACK>
__global__ __launch_bounds__(kThreads, BACK ? 3 : 1) void qk_kernel(QkArgs a) {
  typedef Part<T, FORM, LG, NS> P;
  typedef Form<T, FORM, LG, NS> F;
  constexpr int NP = F::NP, NI = BACK ? 1 : 4;  // rows that a lane has in flight
  __shared__ float2 table[kTable];
  __shared__ __attribute__((aligned(16))) float weights[2 * LG * 2 * NP];
  __shared__ float sums[BACK ? 2 * LG * 2 * NP * 4 : 1];
  const int g = threadIdx.x / LG, l = threadIdx.x % LG, half = a.R / 2;
  const int t = g / a.HS, h0 = g % a.HS;
  const bool on = FORM == kSingle || l * 2 * F::VE < a.K;   // this lane has elements
  float sq[BACK ? 2 * NP : 1], sk[BACK ? 2 * NP : 1];
  // both weights, as a lane reads them: [q, k][lane][2 NP]
  for (int i = threadIdx.x; i < 2 * LG * 2 * NP; i += kThreads) {
    const int e = i % (2 * NP), ll = i / (2 * NP) % LG, isk = i / (2 * NP * LG);
    int ea, eb;
    F::places(a, ll, e / 2, ea, eb);
    const int at = e & 1 ? eb : ea;
    const float* w = isk ? a.wk : a.wq;
    weights[i] = w && at < a.K ? w[at] : 1.0f;
  }
  if constexpr (BACK) {
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) sq[i] = sk[i] = 0.0f;
  }
  const float m = a.norm == TSSM_NORM_RMS ? 1.0f / (float)a.K : (a.norm == TSSM_NORM_L2 ? 1.0f : 0.0f);
  for (uint32_t block = block_of(); block < a.blocks; block += gridDim.x * gridDim.y) {
    const uint32_t first = block * (uint32_t)a.TB;
    const uint32_t tok = first + (uint32_t)t;
    const bool live = tok < a.tokens;
    const uint32_t tk = live ? tok : a.tokens - 1, b = tk / a.L, at = tk - b * a.L;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_b + at * a.q_l;
    const T* k = reinterpret_cast<const T*>(a.k) + b * a.k_b + at * a.k_l;
    T* yq = reinterpret_cast<T*>(a.yq) + b * a.yq_b + at * a.yq_l;
    T* yk = reinterpret_cast<T*>(a.yk) + b * a.yk_b + at * a.yk_l;
    const T* dq = reinterpret_cast<const T*>(a.dq) + (BACK ? b * a.dq_b + at * a.dq_l : 0);
    const T* dk = reinterpret_cast<const T*>(a.dk) + (BACK ? b * a.dk_b + at * a.dk_l : 0);
    P x[NI], d[BACK ? NI : 1];
    // rows past the last head are this lane's first ones again (no branch: it would
    // make every load wait)
    const auto fetch = [&](int hb) {
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        int h = hb + n * a.HS + h0;
        h = h < a.H ? h : (h0 < a.H ? h0 : 0);
        x[n].load(a, h < a.Hq ? q + h * a.q_h : k + (h - a.Hq) * a.k_h, l, on);
        if constexpr (BACK)
          d[n].load(a, h < a.Hq ? dq + h * a.dq_h : dk + (h - a.Hq) * a.dk_h, l, on);
      }
    };
    fetch(0);  // in flight while the angles are formed
    // the table of this block's angles
    for (int i = threadIdx.x; i < a.TB * half; i += kThreads) {
      const int tt = i / half, j = i - tt * half;
      const uint32_t tok2 = first + (uint32_t)tt < a.tokens ? first + (uint32_t)tt : a.tokens - 1;
      const uint32_t b2 = tok2 / a.L, at2 = tok2 - b2 * a.L;
      const double turns =
          position(a, b2 * a.p_b + at2 * a.p_l) * a.freq[j] * 0.15915494309189535;
      float s, c;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
      table[i] = make_float2(a.amplitude * c, a.amplitude * s);
    }
    lds_barrier();
    float c[NP], s[NP];
    bool rot[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int j = FORM == kSingle ? l + LG * i : l * F::VE + i;
      rot[i] = j < half;
      const float2 y = table[t * half + (rot[i] ? j : 0)];
      c[i] = rot[i] ? y.x : 1.0f;
      s[i] = rot[i] ? y.y : 0.0f;
    }
    for (int hb = 0; hb < a.H; hb += NI * a.HS) {
      if (hb) fetch(hb);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int h = hb + n * a.HS + h0;
        if (h >= a.H || !live) continue;   // (whole groups)
        const bool isq = h < a.Hq;
        float u[NP], v[NP], sum = 0.0f, r = 1.0f;
        x[n].get(a, l, on, u, v);
        if (a.norm != TSSM_NORM_NONE) {
#pragma unroll
          for (int i = 0; i < NP; ++i) sum = __builtin_fmaf(u[i], u[i], __builtin_fmaf(v[i], v[i], sum));
          r = 1.0f / sqrtf(__builtin_fmaf(row_sum<LG>(sum), m, a.eps));
        }
        float w[2 * NP];
        const float* wp = &weights[((isq ? 0 : LG) + l) * 2 * NP];
#pragma unroll
        for (int i = 0; i < 2 * NP; ++i) w[i] = wp[i];
        T* out = isq ? yq + h * a.yq_h : yk + (h - a.Hq) * a.yk_h;
        if constexpr (!BACK) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float f = u[i] * r * w[2 * i];
            const float e = v[i] * r * w[2 * i + 1];
            u[i] = rot[i] ? f * c[i] - e * s[i] : f;
            v[i] = rot[i] ? f * s[i] + e * c[i] : e;
          }
        } else {
          float f[NP], e[NP], dot = 0.0f;
          d[n].get(a, l, on, f, e);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const float x0 = rot[i] ? f[i] * c[i] + e[i] * s[i] : f[i];
            const float x1 = rot[i] ? e[i] * c[i] - f[i] * s[i] : e[i];
            const float g0 = x0 * (u[i] * r), g1 = x1 * (v[i] * r);
            if (isq) {
              sq[2 * i] += g0;
              sq[2 * i + 1] += g1;
            } else {
              sk[2 * i] += g0;
              sk[2 * i + 1] += g1;
            }
            f[i] = x0 * w[2 * i];
            e[i] = x1 * w[2 * i + 1];
            dot = __builtin_fmaf(f[i], u[i], __builtin_fmaf(e[i], v[i], dot));
          }
          if (a.norm != TSSM_NORM_NONE) dot = row_sum<LG>(dot) * (m * r * r);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            u[i] = r * (a.norm != TSSM_NORM_NONE ? f[i] - u[i] * dot : f[i]);
            v[i] = r * (a.norm != TSSM_NORM_NONE ? e[i] - v[i] * dot : e[i]);
          }
        }
        x[n].put(a, out, l, on, u, v);
      }
    }
    lds_barrier();  // the table is read
  }
  if constexpr (BACK) {
    if (!a.part) return;
    // sums over the groups of a wave, then over the waves
    float* part = a.part + (int64_t)block_of() * 2 * a.K;
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 2 * NP; ++i) {
#pragma unroll
      for (int x = LG; x < 64; x *= 2) {
        sq[i] += __shfl_xor(sq[i], x);
        sk[i] += __shfl_xor(sk[i], x);
      }
      if ((threadIdx.x & 63) < LG) {
        sums[((wave * 2 + 0) * LG + l) * 2 * NP + i] = sq[i];
        sums[((wave * 2 + 1) * LG + l) * 2 * NP + i] = sk[i];
      }
    }
    __syncthreads();
    for (int n = threadIdx.x; n < 2 * LG; n += kThreads) {
      const int ll = n % LG, which = n / LG;
      if (FORM != kSingle && ll * 2 * F::VE >= a.K) continue;
      for (int i = 0; i < 2 * NP; ++i) {
        float y = 0.0f;
        for (int w = 0; w < kThreads / 64; ++w) y += sums[((w * 2 + which) * LG + ll) * 2 * NP + i];
        int ea, eb;
        F::places(a, ll, i / 2, ea, eb);
        const int e = i & 1 ? eb : ea;
        if (e < a.K) part[which * a.K + e] = y;
      }
    }
  }
}

// dw = sum of the workgroups' parts, in order: 16 columns of [rows][n] a workgroup, 64
// rows at a time, eight loads in flight (768 rows of 2 x 128: 4.5 us).
__global__ __launch_bounds__(1024) void qk_sum_kernel(const float* part, int rows, int n, int K,
                                                      float* dwq, float* dwk) {
  __shared__ float sums[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  const float* p = part + (col < n ? col : 0);
  float s = 0.0f;
  for (int i = r; i < rows; i += 8 * 64) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[(int64_t)(i + 64 * e < rows ? i + 64 * e : i) * n];
#pragma unroll
    for (int e = 0; e < 8; ++e) s += i + 64 * e < rows ? x[e] : 0.0f;
  }
  sums[r][c] = s;
  __syncthreads();
  if (r == 0 && col < n) {
    for (int i = 1; i < 64; ++i) s += sums[i][c];
    if (col < K && dwq) dwq[col] = s;
    if (col >= K && dwk) dwk[col - K] = s;
  }
}

// Workgroups of the gradients: the three that a CU holds, each with blocks of its own
// to go through, so that few sums of the weights' gradients are left to join (16384
// tokens of 16 + 8 heads of 128, bf16: 68 us; 82 with 1024, which leaves a third of the
// CUs a workgroup more than the others, 100 with one for each of 4096 blocks).
constexpr int64_t kBackGroups = 768;

int sum_parts(const QkArgs& a, int rows, hipStream_t st) {
  qk_sum_kernel<<<(unsigned)cdiv64(2 * a.K, 16), 1024, 0, st>>>(a.part, rows, 2 * a.K, a.K, a.dwq,
                                                             a.dwk);
  return launch_status();
}

// The widest pieces, of 16, 8 or 4 bytes, that rows and their pairs are made of (0:
// single elements), in elements.  Narrow ones for up to 16 lanes a row: 190 MB of rows
// of 40 channels in bf16 98 against 153 us (all turned, 8 bytes), 162 against 176 (half of
// them, 4 bytes); of 72, which take 18 lanes, 179 against 158.
template <typename T>
int pieces(const QkArgs& a, bool back) {
  const int E = (int)sizeof(T);
  int64_t s = a.q_b | a.q_l | a.q_h | a.k_b | a.k_l | a.k_h | a.yq_b | a.yq_l | a.yq_h | a.yk_b |
              a.yk_l | a.yk_h;
  if (back) s |= a.dq_b | a.dq_l | a.dq_h | a.dk_b | a.dk_l | a.dk_h;
  for (int VE = 16 / E; VE > 1; VE /= 2) {
    const int64_t n = VE * E;
    if (a.K % (2 * VE) || a.R % (2 * VE) || s * E % n || a.K / (2 * VE) > (n == 16 ? 32 : 16))
      continue;
    if (aligned(a.q, n) && aligned(a.k, n) && aligned(a.yq, n) && aligned(a.yk, n) &&
        (!back || (aligned(a.dq, n) && aligned(a.dk, n))))
      return VE;
  }
  return 0;
}

template <typename T, int FORM, int LG, int NS, bool BACK>
int launch(QkArgs a, hipStream_t st) {
  constexpr int kGroups = kThreads / LG;
  // tokens beside each other: all heads of one token at once where that fills the
  // chip, several rows for a lane otherwise, within the table
  int TB = 1;
  while (TB < kGroups && (int64_t)TB * 2 * (a.R / 2) <= kTable &&
         cdiv64(a.H, kGroups / (TB * 2)) <= 4 && a.tokens / (TB * 2) >= 1024)
    TB *= 2;
  a.TB = TB;
  a.HS = kGroups / TB;
  a.blocks = (uint32_t)cdiv64(a.tokens, TB);
  int64_t wgs = a.blocks;
  if (BACK && wgs > kBackGroups) wgs = kBackGroups;
  qk_kernel<T, FORM, LG, NS, BACK><<<grid_of(wgs), kThreads, 0, st>>>(a);
  if (BACK && a.part) return sum_parts(a, (int)wgs, st);
  return launch_status();
}

template <typename T, int FORM, int VE, bool BACK>
int by_lanes(const QkArgs& a, hipStream_t st) {
  const int64_t lanes = a.K / (2 * VE);
  if constexpr (VE * sizeof(T) == 16) {
    if (lanes <= 1) return launch<T, FORM, 1, VE, BACK>(a, st);
    if (lanes <= 2) return launch<T, FORM, 2, VE, BACK>(a, st);
    if (lanes <= 4) return launch<T, FORM, 4, VE, BACK>(a, st);
  }
  if (lanes <= 8) return launch<T, FORM, 8, VE, BACK>(a, st);
  if constexpr (VE * sizeof(T) == 16)
    if (lanes > 16) return launch<T, FORM, 32, VE, BACK>(a, st);
  return launch<T, FORM, 16, VE, BACK>(a, st);
}

template <typename T, int VE, bool BACK>
int by_order(const QkArgs& a, hipStream_t st) {
  return a.interleaved ? by_lanes<T, kNeighbours, VE, BACK>(a, st)
                       : by_lanes<T, kHalf, VE, BACK>(a, st);
}

template <typename T, bool BACK>
int by_form(const QkArgs& a, hipStream_t st) {
  constexpr int W = 16 / (int)sizeof(T);
  const int VE = pieces<T>(a, BACK);
  if (VE == W) return by_order<T, W, BACK>(a, st);
  if (VE == W / 2) return by_order<T, W / 2, BACK>(a, st);
  if constexpr (W == 8)
    if (VE == 2) return by_order<T, 2, BACK>(a, st);
  const int slots = a.R / 2 + (a.K - a.R + 1) / 2;
  if (slots <= 16) return launch<T, kSingle, 16, 1, BACK>(a, st);
  if (slots <= 32) return launch<T, kSingle, 16, 2, BACK>(a, st);
  if (slots <= 64) return launch<T, kSingle, 16, 4, BACK>(a, st);
  return launch<T, kSingle, 16, 8, BACK>(a, st);
}

template <bool BACK>
int by_type(int dtype, const QkArgs& a, hipStream_t st) {
  switch (dtype) {
    case TSSM_F32: return by_form<float, BACK>(a, st);
    case TSSM_BF16: return by_form<bf16_t, BACK>(a, st);
    default: return by_form<f16_t, BACK>(a, st);
  }
}

// What both directions ask for.
int checks(int dtype, int norm, int pos_type, int64_t nbatch, int64_t L, int64_t Hq, int64_t Hk,
           int64_t K, int64_t R, const void* pos, const double* freq) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(pos_type >= TSSM_POS_F32 && pos_type <= TSSM_POS_I64, TSSM_ERR_DTYPE);
  TSSM_CHECK(norm >= TSSM_NORM_NONE && norm <= TSSM_NORM_L2, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(nbatch >= 0 && L >= 0 && Hq > 0 && Hk > 0 && K > 0 && R >= 0 && R <= K && R % 2 == 0,
             TSSM_ERR_SHAPE);
  // one channel's norm is its sign, and its gradient what rounding leaves
  TSSM_CHECK(norm == TSSM_NORM_NONE || K > 1, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(K <= 256 && Hq <= 65536 && Hk <= 65536, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(L == 0 || nbatch <= 0x7fffffff / L, TSSM_ERR_UNSUPPORTED);
  TSSM_CHECK(R == 0 || nbatch * L == 0 || (pos && freq), TSSM_ERR_NULL);
  return TSSM_OK;
}

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int tssm_qk_norm_rotary_fwd(
    int dtype, int norm, int interleaved, const void* q, const void* k, const void* pos,
    int pos_type, const double* freq, const float* wq, const float* wk, void* yq, void* yk,
    int64_t nbatch, int64_t L, int64_t Hq, int64_t Hk, int64_t K, int64_t R, int64_t sq_b,
    int64_t sq_l, int64_t sq_h, int64_t sk_b, int64_t sk_l, int64_t sk_h, int64_t sp_b,
    int64_t sp_l, int64_t syq_b, int64_t syq_l, int64_t syq_h, int64_t syk_b, int64_t syk_l,
    int64_t syk_h, float eps, float amplitude, void* stream) {
  const int rc = checks(dtype, norm, pos_type, nbatch, L, Hq, Hk, K, R, pos, freq);
  if (rc) return rc;
  if (nbatch == 0 || L == 0) return TSSM_OK;
  TSSM_CHECK(q && k && yq && yk, TSSM_ERR_NULL);
  QkArgs a = {};
  a.q = q; a.k = k; a.yq = yq; a.yk = yk; a.pos = pos; a.freq = freq; a.wq = wq; a.wk = wk;
  a.q_b = sq_b; a.q_l = sq_l; a.q_h = sq_h; a.k_b = sk_b; a.k_l = sk_l; a.k_h = sk_h;
  a.p_b = sp_b; a.p_l = sp_l;
  a.yq_b = syq_b; a.yq_l = syq_l; a.yq_h = syq_h; a.yk_b = syk_b; a.yk_l = syk_l; a.yk_h = syk_h;
  a.tokens = (uint32_t)(nbatch * L); a.L = (uint32_t)L;
  a.Hq = (int)Hq; a.H = (int)(Hq + Hk); a.K = (int)K; a.R = (int)R;
  a.norm = norm; a.interleaved = interleaved; a.pos_type = pos_type;
  a.eps = eps; a.amplitude = amplitude;
  return by_type<false>(dtype, a, as_stream(stream));
}

extern "C" int64_t tssm_qk_norm_rotary_workspace_bytes(int64_t K) {
  if (K <= 0) return TSSM_ERR_SHAPE;
  if (K > 256) return TSSM_ERR_UNSUPPORTED;
  return kBackGroups * 2 * K * 4;
}

extern "C" int tssm_qk_norm_rotary_bwd(
    int dtype, int norm, int interleaved, const void* dyq, const void* dyk, const void* q,
    const void* k, const void* pos, int pos_type, const double* freq, const float* wq,
    const float* wk, void* dq, void* dk, float* dwq, float* dwk, int64_t nbatch, int64_t L,
    int64_t Hq, int64_t Hk, int64_t K, int64_t R, int64_t sdyq_b, int64_t sdyq_l, int64_t sdyq_h,
    int64_t sdyk_b, int64_t sdyk_l, int64_t sdyk_h, int64_t sq_b, int64_t sq_l, int64_t sq_h,
    int64_t sk_b, int64_t sk_l, int64_t sk_h, int64_t sp_b, int64_t sp_l, int64_t sdq_b,
    int64_t sdq_l, int64_t sdq_h, int64_t sdk_b, int64_t sdk_l, int64_t sdk_h, float eps,
    float amplitude, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = checks(dtype, norm, pos_type, nbatch, L, Hq, Hk, K, R, pos, freq);
  if (rc) return rc;
  const bool weights = dwq || dwk, none = nbatch == 0 || L == 0;
  if (weights)
    TSSM_CHECK(workspace && workspace_bytes >= tssm_qk_norm_rotary_workspace_bytes(K) &&
                   aligned(workspace, 16),
               TSSM_ERR_WORKSPACE);
  QkArgs a = {};
  a.K = (int)K;
  a.part = weights ? reinterpret_cast<float*>(workspace) : nullptr;
  a.dwq = dwq; a.dwk = dwk;
  if (none) return weights ? sum_parts(a, 0, as_stream(stream)) : TSSM_OK;
  TSSM_CHECK(dyq && dyk && q && k && dq && dk, TSSM_ERR_NULL);
  a.q = q; a.k = k; a.dq = dyq; a.dk = dyk; a.yq = dq; a.yk = dk; a.pos = pos; a.freq = freq;
  a.wq = wq; a.wk = wk;
  a.q_b = sq_b; a.q_l = sq_l; a.q_h = sq_h; a.k_b = sk_b; a.k_l = sk_l; a.k_h = sk_h;
  a.dq_b = sdyq_b; a.dq_l = sdyq_l; a.dq_h = sdyq_h;
  a.dk_b = sdyk_b; a.dk_l = sdyk_l; a.dk_h = sdyk_h;
  a.p_b = sp_b; a.p_l = sp_l;
  a.yq_b = sdq_b; a.yq_l = sdq_l; a.yq_h = sdq_h; a.yk_b = sdk_b; a.yk_l = sdk_l; a.yk_h = sdk_h;
  a.tokens = (uint32_t)(nbatch * L); a.L = (uint32_t)L;
  a.Hq = (int)Hq; a.H = (int)(Hq + Hk); a.R = (int)R;
  a.norm = norm; a.interleaved = interleaved; a.pos_type = pos_type;
  a.eps = eps; a.amplitude = amplitude;
  return by_type<true>(dtype, a, as_stream(stream));
}
