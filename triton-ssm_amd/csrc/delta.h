// Shared argument block of the gated delta rule's kernels (delta.hip and
// its translation units).  Per batch b, value head h (key head h / per):
//   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),  S_t = e^{g_t} S_{t-1} + k_t u_t^T,
//   o_t = scale S_t^T q_t,   S [K, V] fp32.
#pragma once

#include <type_traits>

#include "common.h"

namespace tssm {

struct DeltaArgs {
  const void *q, *k, *v;
  const float *g, *beta, *h0;
  void* o;
  float* h_last;
  int64_t B, L, Hk, Hv, K, V;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h;
  int64_t g_b, g_l, g_h, be_b, be_l, be_h, o_b, o_l, o_h;
  float scale;
};

// Batch, value head and key head of one of the B Hv heads, which are fewer than
// 2^32 (a 64-bit division is some 150 instructions, and kernels begin with it).
struct HeadOf {
  int64_t b, h, hk;
};
__device__ inline HeadOf head_of(const DeltaArgs& a, uint32_t bh) {
  const uint32_t Hv = (uint32_t)a.Hv, b = bh / Hv, h = bh - b * Hv;
  return {b, h, h / (Hv / (uint32_t)a.Hk)};
}

// delta_seq.hip: one step after another, the state in registers.
int delta_seq_launch(int dtype, const DeltaArgs& a, hipStream_t s);

// Chunked form.  Workspace of one call: what the preparing pass leaves of each
// chunk and, for sequences walked in segments, the segments' transfer
// matrices and entry states; for the gradients also the states before the
// chunks, and the gradients of the states after them.
struct DeltaPlan {
  void* chunks;
  float *transfer, *entry;     // nseg > 1
  float *states, *grads;       // gradients only: of the state before, the gradient after each chunk
  float *back, *gentry;        // gradients only, nseg > 1: like transfer's N and entry
  int nch, per, nseg;          // chunks, chunks of a segment, segments
  int64_t bytes;
};

// vec: the rows of q, k and v are whole 16-byte accesses.
int delta_prep_launch(int dtype, const DeltaArgs& a, bool vec, void* chunks, hipStream_t s);
int delta_walk_launch(int dtype, const DeltaArgs& a, bool vec, const DeltaPlan& p, hipStream_t s);
// The segments' transfer matrices, then their entry states.
int delta_transfer_launch(int dtype, const DeltaArgs& a, bool vec, const DeltaPlan& p,
                          hipStream_t s);
int delta_fold(const DeltaArgs& a, const DeltaPlan& p, hipStream_t s);
int delta_fold_back(const DeltaArgs& a, const DeltaPlan& p, hipStream_t s);
// The states before the chunks and the gradients of those after them (way.v:
// dO, way.h0: dh_last, way.h_last: dh0), segments included.
int delta_both_launch(int dtype, const DeltaArgs& a, const DeltaArgs& way, bool vec,
                      const DeltaPlan& p, hipStream_t s);
// Gradients of the inputs; outputs contiguous, dO with strides.
struct DeltaGrads {
  const void* dout;
  int64_t d_b, d_l, d_h;
  void *dq, *dk, *dv;
  float *dg, *dbeta;
};
int delta_grads_launch(int dtype, const DeltaArgs& a, const DeltaGrads& d, bool vec,
                       const DeltaPlan& p, hipStream_t s);
int64_t delta_chunk_ws_bytes();  // of one chunk of one value head

}  // namespace tssm
