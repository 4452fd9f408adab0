// Gated delta rule, chunked: the segments of a long sequence, walked from zero
// and joined.
#include "delta_walk.h"

namespace tssm {
namespace {

// entry[seg + 1] = M_seg entry[seg] + N_seg, segment after segment (forward:
// entry[0] is a.h0), or, with REV, the gradient's way back: entry[seg - 1] =
// M_seg^T entry[seg] + N_seg, from dh_last.  M_seg and forward N_seg lie in
// transfer [bh][nseg][Vp + KP][KP] (columns of N, then of M), N of the way back
// in back [bh][nseg][Vp][KP].  A workgroup owns 16 columns, a wave of it one
// tile of 16 rows; the state goes round through LDS, the next three segments'
// M and N are in flight meanwhile, products take three planes each.
struct FoldArgs {
  const float *first, *transfer, *back;
  float* entry;
  int64_t heads, V;
  int K, nseg, nvb;
};

template <int NS, bool REV>
__global__ __launch_bounds__(128 * NS) void delta_fold_kernel(FoldArgs f) {
  constexpr int KP = 32 * NS;
  __shared__ f32x4 tiles[2][2 * NS][64];
  const int lane = threadIdx.x & 63, j = lane >> 4, c = lane & 15, ar = 8 * (c >> 2) + (c & 3);
  const int x = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));  // the wave's tile
  const int64_t bh = blockIdx.x / f.nvb, col = (int64_t)(blockIdx.x - bh * f.nvb) * 16 + c;
  const int64_t Vp = (int64_t)f.nvb * 16;
  const int row = 32 * (x >> 1) + 4 * (x & 1);  // of the state: + ar (M), + 8 j + r (tile)
  struct In {
    float m[NS][8];
    f32x4 N;
  };
  auto load = [&](In& g, int i) {
    if (i > f.nseg - 2) i = f.nseg - 2;
    const int seg = REV ? f.nseg - 1 - i : i;
    const float* tr = f.transfer + (bh * f.nseg + seg) * (Vp + KP) * KP;
    const float* M = tr + Vp * KP;  // M[k'][k] at M + k KP + k'
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = 32 * s + 8 * j + e;  // summed over
        g.m[s][e] = M[REV ? (row + ar) * KP + k : k * KP + row + ar];
      }
    const float* n = REV ? f.back + (bh * f.nseg + seg) * Vp * KP : tr;
    g.N = *reinterpret_cast<const f32x4*>(n + col * KP + row + 8 * j);
  };
  f32x4 S[2 * NS];
  get_state<NS>(f.first ? f.first + bh * f.K * f.V : nullptr, S, col, f.V, f.K, j);
  auto step = [&](int i, In& g) {
    u32x4 sp[NS][3], mp[NS][3];
    f32x4 o = g.N;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      split_tiles<3>(S[2 * s], S[2 * s + 1], sp[s]);
      split8<3>(g.m[s], mp[s]);
    }
    load(g, i + 3);
#pragma unroll
    for (int s = 0; s < NS; ++s) o = mfma_planes<3, 3, 3>(mp[s], sp[s], o);
    tiles[i & 1][x][lane] = o;
    const int seg = REV ? f.nseg - 2 - i : i + 1;
    *reinterpret_cast<f32x4*>(f.entry + ((bh * f.nseg + seg) * Vp + col) * KP + row + 8 * j) = o;
    lds_barrier();
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) S[t] = tiles[i & 1][t][lane];
  };
  // the first entry state too: the walks then read no buffer that they write
  // (h0 may be h_last)
#pragma unroll
  for (int t = 0; t < 2 * NS; ++t)
    if (t == x)
      *reinterpret_cast<f32x4*>(f.entry + ((bh * f.nseg + (REV ? f.nseg - 1 : 0)) * Vp + col) * KP +
                                row + 8 * j) = S[t];
  In g0, g1, g2;
  load(g0, 0);
  load(g1, 1);
  load(g2, 2);
  for (int i = 0; i < f.nseg - 1; i += 3) {
    step(i, g0);
    if (i + 1 < f.nseg - 1) step(i + 1, g1);
    if (i + 2 < f.nseg - 1) step(i + 2, g2);
  }
}

template <bool REV>
int fold(const FoldArgs& f, hipStream_t s) {
  const unsigned wgs = (unsigned)(f.heads * f.nvb);
  if (f.K <= 32) delta_fold_kernel<1, REV><<<wgs, 128, 0, s>>>(f);
  else if (f.K <= 64) delta_fold_kernel<2, REV><<<wgs, 256, 0, s>>>(f);
  else delta_fold_kernel<4, REV><<<wgs, 512, 0, s>>>(f);
  return launch_status();
}

}  // namespace

int delta_fold(const DeltaArgs& a, const DeltaPlan& p, hipStream_t s) {
  const FoldArgs f = {a.h0, p.transfer, nullptr, p.entry, a.B * a.Hv, a.V, (int)a.K, p.nseg,
                      (int)cdiv64(a.V, 16)};
  return fold<false>(f, s);
}

int delta_fold_back(const DeltaArgs& a, const DeltaPlan& p, hipStream_t s) {
  const FoldArgs f = {a.h0, p.transfer, p.back, p.gentry, a.B * a.Hv, a.V, (int)a.K, p.nseg,
                      (int)cdiv64(a.V, 16)};
  return fold<true>(f, s);
}

int delta_transfer_launch(int dtype, const DeltaArgs& a, bool vec, const DeltaPlan& p,
                          hipStream_t s) {
  WalkArgs g = {};
  g.a = a;
  g.ws = reinterpret_cast<const ChunkWs*>(p.chunks);
  g.nch = p.nch;
  g.per = p.per;
  g.nseg = p.nseg;
  g.walked = p.nseg - 1;
  g.states = p.transfer;
  const int rc = walk_mode<kTransfer>(dtype, g, vec, s);
  return rc ? rc : delta_fold(a, p, s);
}

}  // namespace tssm
