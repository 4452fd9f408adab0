// Linear attention, chunked: the segments of a long sequence and how they are joined,
// and for the gradients the states before the chunks and the gradients after them.
//
// The gradients' two walks run side by side (B=4 L=4096 H=16 64 x 64 bf16: 73 us for 134
// MB read and 134 MB of states written, 3.7 TB/s; 64 chunks one after the other, of 2200
// cycles that the loads take to arrive).  The shorter pass over the segments of B=1
// L=65536 H=8 takes 40 us for 130 MB (3.3 TB/s), joining its 31 ends 8 us.
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

template <typename T, int MODE>
int by_keys(const LinWalkArgs& f, const LinWalkArgs& b, LinRows rows, hipStream_t s) {
#define TSSM_WALK(KP) \
  (rows == kAllRows   ? lin_states_run<T, KP, kAllRows, MODE>(f, b, s) \
   : rows == kKeyRows ? lin_states_run<T, KP, kKeyRows, MODE>(f, b, s) \
                      : lin_states_run<T, KP, kNoRows, MODE>(f, b, s))
  if (f.a.K <= 32) return TSSM_WALK(32);
  if (f.a.K <= 64) return TSSM_WALK(64);
  return TSSM_WALK(128);
#undef TSSM_WALK
}

template <int MODE>
int walk(int dtype, const LinWalkArgs& f, const LinWalkArgs& b, LinRows rows, hipStream_t s) {
  switch (dtype) {
    case TSSM_F32: return by_keys<float, MODE>(f, b, rows, s);
    case TSSM_BF16: return by_keys<bf16_t, MODE>(f, b, rows, s);
    default: return by_keys<f16_t, MODE>(f, b, rows, s);
  }
}

// The walk of all segments but the last one (forward) or the first (back).
LinWalkArgs ends_of(const LinArgs& a, const LinPlan& p, bool rev) {
  LinWalkArgs g = {};
  g.a = a;
  g.steps = p.steps;
  g.nseg = (int)p.nseg;
  g.walked = g.nseg - 1;
  g.first = rev ? 1 : 0;
  g.states = rev ? p.back : p.ends;
  g.sums = rev ? p.back_sums : p.sums;
  return g;
}

}  // namespace

int lin_entry_launch(int dtype, const LinArgs& a, LinRows rows, const LinPlan& p, hipStream_t s) {
  LinWalkArgs none = ends_of(a, p, false);
  none.walked = 0;
  const int rc = walk<kEnds>(dtype, ends_of(a, p, false), none, rows, s);
  return rc ? rc : fold(a, p.ends, p.sums, (int)p.nseg, 0, s);
}

int lin_states_launch(int dtype, const LinArgs& a, const LinArgs& way, LinRows rows, const LinPlan& p,
                      hipStream_t s) {
  LinWalkArgs f = ends_of(a, p, false), b = ends_of(way, p, true);
  if (p.nseg > 1) {
    int rc = walk<kEnds>(dtype, f, b, rows, s);
    if (!rc) rc = fold(a, p.ends, p.sums, (int)p.nseg, 0, s);
    if (!rc) rc = fold(way, p.back, p.back_sums, (int)p.nseg, 1, s);
    if (rc) return rc;
  }
  f.walked = b.walked = (int)p.nseg;
  b.first = 0;
  f.entry = p.ends;
  b.entry = p.back;
  f.states = p.states;
  b.states = p.grads;
  return walk<kStates>(dtype, f, b, rows, s);
}

}  // namespace tssm
