// Shared argument block of linear attention's kernels (linattn.hip and its
// translation units).  Per batch b, value head h (key head h / per):
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t,   S [K, V] fp32.
#pragma once

#include "common.h"

namespace tssm {

struct LinArgs {
  const void *q, *k, *v;
  const float *g, *h0;
  void* o;
  float* h_last;
  int64_t B, L, Hk, Hv, K, V;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h;
  int64_t g_b, g_l, g_h, o_b, o_l, o_h;
  float scale;
};

// Batch, value head and key head of one of the B Hv heads, which are fewer than
// 2^32 (a 64-bit division is some 150 instructions, and kernels begin with it).
struct LinHead {
  int64_t b, h, hk;
};
__device__ inline LinHead lin_head(const LinArgs& a, uint32_t bh) {
  const uint32_t Hv = (uint32_t)a.Hv, b = bh / Hv, h = bh - b * Hv;
  return {b, h, h / (Hv / (uint32_t)a.Hk)};
}

// linattn_seq.hip: one step after another, the state in registers.
int lin_seq_launch(int dtype, const LinArgs& a, hipStream_t s);

// Chunked form.  Sequences of few heads are walked in segments: each one's end
// state from zero, joined to its entry state (ends, in place) by the sums of g.  For
// the gradients also the states before the chunks, and the gradients of those after
// them (`back`: the same of the way back).
struct LinPlan {
  int64_t steps, nseg;       // steps of a segment, segments
  float *ends, *back;        // nseg > 1
  double *sums, *back_sums;
  float *states, *grads;     // gradients only
  int64_t split;             // workgroups that share the value heads of a chunk's key head
  float* part;               // split > 1: [dQ, dK][split][B, L, Hk, K]
  int64_t bytes;
};
// rows: what whole 16-byte accesses make up.
enum LinRows { kNoRows, kKeyRows, kAllRows };  // none, the rows of q and k, those of v and o too
int lin_walk_launch(int dtype, const LinArgs& a, LinRows rows, const LinPlan& p, hipStream_t s);
// The segments' entry states, forward.
int lin_entry_launch(int dtype, const LinArgs& a, LinRows rows, const LinPlan& p, hipStream_t s);
// The states before the chunks and the gradients of those after them (way: q for k, dO
// for v, dh_last for h0, dh0 for h_last), segments included.
int lin_states_launch(int dtype, const LinArgs& a, const LinArgs& way, LinRows rows, const LinPlan& p,
                      hipStream_t s);
constexpr int kLinChunk = 64;  // steps of such a chunk
// Gradients of the inputs; outputs contiguous, dO with strides.
struct LinGrads {
  const void* dout;
  int64_t d_b, d_l, d_h;
  void *dq, *dk, *dv;
  float* dg;
};
int lin_grads_launch(int dtype, const LinArgs& a, const LinGrads& d, LinRows rows, const LinPlan& p,
                     hipStream_t s);

}  // namespace tssm
