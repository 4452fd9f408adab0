// Gated delta rule, chunked: the walk that forms the outputs.
#include "delta_walk.h"

namespace tssm {

int delta_walk_launch(int dtype, const DeltaArgs& a, bool vec, const DeltaPlan& p, hipStream_t s) {
  WalkArgs g = {};
  g.a = a;
  g.ws = reinterpret_cast<const ChunkWs*>(p.chunks);
  g.nch = p.nch;
  g.per = p.per;
  g.nseg = g.walked = p.nseg;
  g.entry = p.entry;
  return walk_mode<kOutputs>(dtype, g, vec, s);
}

int64_t delta_chunk_ws_bytes() { return (int64_t)sizeof(ChunkWs); }

}  // namespace tssm
