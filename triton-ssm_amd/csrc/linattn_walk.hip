// Linear attention, chunked: the outputs (linattn_walk.h).
#include "linattn_walk.h"

namespace tssm {
namespace {

template <typename T>
int by_keys(const LinWalkArgs& g, LinRows rows, hipStream_t s) {
#define TSSM_WALK(KP)                                                \
  (rows == kAllRows   ? lin_walk_run<T, KP, kAllRows>(g, s)          \
   : rows == kKeyRows ? lin_walk_run<T, KP, kKeyRows>(g, s)          \
                      : lin_walk_run<T, KP, kNoRows>(g, s))
  if (g.a.K <= 32) return TSSM_WALK(32);
  if (g.a.K <= 64) return TSSM_WALK(64);
  return TSSM_WALK(128);
#undef TSSM_WALK
}

}  // namespace

int lin_walk_launch(int dtype, const LinArgs& a, LinRows rows, const LinPlan& p, hipStream_t s) {
  LinWalkArgs g = {};
  g.a = a;
  g.steps = p.steps;
  g.nseg = g.walked = (int)p.nseg;
  g.entry = p.ends;
  switch (dtype) {
    case TSSM_F32: return by_keys<float>(g, rows, s);
    case TSSM_BF16: return by_keys<bf16_t>(g, rows, s);
    default: return by_keys<f16_t>(g, rows, s);
  }
}

}  // namespace tssm
