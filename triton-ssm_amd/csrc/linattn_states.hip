// Linear attention, chunked: the segments of a long sequence and how they are joined.
#include "linattn_walk.h"

namespace tssm {
namespace {

// ends[bh][seg], the state at a segment's end from zero, becomes the state that it
// starts from: entry[0] is a.h0 and entry[seg + 1] = e^(sum of g) entry[seg] + end[seg];
// backwards (rev) the same from the last segment on.  Elements do not meet: a lane has
// four of them and goes through the segments, whose loads run four ahead.
struct LinFoldArgs {
  const float* first;  // [bh][K][V] or null
  float* ends;
  const double* sums;
  int64_t heads, V, elems;
  int K, KP, nseg, rev;
};

__global__ __launch_bounds__(256) void lin_fold_kernel(LinFoldArgs f) {
  const int64_t at = (int64_t)block_of() * 256 + threadIdx.x, quads = f.elems / 4;
  if (at >= f.heads * quads) return;
  const int64_t bh = at / quads, q = at - bh * quads;
  const int lane = (int)(q & 63), tile = (int)(q >> 6), KT = f.KP / 16, kt = tile % KT;
  const int64_t col = (int64_t)(tile / KT) * 16 + (lane & 15);
  f32x4 e = get_tile(f.first ? f.first + bh * f.K * f.V : nullptr, kt, col, f.V, f.K, lane >> 4);
  float* p = f.ends + bh * f.nseg * f.elems + q * 4;
  const double* sums = f.sums + bh * f.nseg;
  const auto seg = [&](int i) { return f.rev ? f.nseg - 1 - i : i; };
  for (int i = 0; i < f.nseg; i += 4) {
    f32x4 x[4];
    float d[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int s = seg(i + n < f.nseg ? i + n : f.nseg - 1);
      x[n] = *reinterpret_cast<const f32x4*>(p + s * f.elems);
      d[n] = (float)sums[s];
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (i + n >= f.nseg) break;
      *reinterpret_cast<f32x4*>(p + seg(i + n) * f.elems) = e;
      const float last = exp2_fast(d[n]);
#pragma unroll
      for (int r = 0; r < 4; ++r) e[r] = __builtin_fmaf(e[r], last, x[n][r]);
    }
  }
}

int fold(const LinArgs& a, float* ends, const double* sums, int nseg, int rev, hipStream_t s) {
  LinFoldArgs f = {a.h0, ends, sums, a.B * a.Hv, a.V, 0, (int)a.K,
                   a.K <= 32 ? 32 : (a.K <= 64 ? 64 : 128), nseg, rev};
  f.elems = lin_state_elems(f.KP, a.V);
  lin_fold_kernel<<<grid_of(cdiv64(f.heads * f.elems / 4, 256)), 256, 0, s>>>(f);
  return launch_status();
}

}  // namespace

int lin_entry_launch(int dtype, const LinArgs& a, bool vec, const LinPlan& p, hipStream_t s) {
  LinWalkArgs g = {};
  g.a = a;
  g.steps = p.steps;
  g.nseg = (int)p.nseg;
  g.walked = g.nseg - 1;
  g.states = p.ends;
  g.sums = p.sums;
  const int rc = lin_walk_mode<kEnds>(dtype, g, vec, s);
  return rc ? rc : fold(a, p.ends, p.sums, g.nseg, 0, s);
}

}  // namespace tssm
