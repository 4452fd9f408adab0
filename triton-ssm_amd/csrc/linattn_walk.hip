// Linear attention, chunked: the outputs (linattn_walk.h).
#include "linattn_walk.h"

namespace tssm {

int lin_walk_launch(int dtype, const LinArgs& a, bool vec, const LinPlan& p, hipStream_t s) {
  LinWalkArgs g = {};
  g.a = a;
  g.steps = p.steps;
  g.nseg = g.walked = (int)p.nseg;
  g.entry = p.ends;
  return lin_walk_mode<kOutputs>(dtype, g, vec, s);
}

}  // namespace tssm
