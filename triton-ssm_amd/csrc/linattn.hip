// Entry points of linear attention: argument checks and the choice of kernels.
#include "linattn.h"

namespace tssm {
namespace {

bool sizes_ok(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V) {
  return B >= 0 && L >= 0 && Hk > 0 && Hv > 0 && Hv % Hk == 0 && K > 0 && V > 0;
}
// A head's state takes 31 bits.
bool takes(int64_t K, int64_t V) { return K <= 128 && V <= (INT64_C(1) << 21); }

// Few steps go one by one: a step takes 0.4 us, a chunk 7.5 whatever it holds, once for
// every 256 workgroups.  Us a call, one by one against a chunk, bf16 with a state in and
// out: 8 heads of 64 x 64, 12 steps 7.1 against 7.5, 16 steps 8.7 against 7.5; 256 heads,
// 24 steps 12.7 against 14.9, 32 steps 16.0 against 14.8; 512 heads, 48 steps 28 against
// 28; 1024 heads, 48 steps 42 against 62, 96 steps 76 against 64.
bool by_steps(int64_t heads, int64_t L, int64_t V) {
  const int64_t most = heads * cdiv64(V, 32) / 20;
  return L <= (most < 12 ? 12 : (most < 64 ? most : 64));
}

// Segments of a sequence, which are walked side by side once a shorter pass (the states
// alone) has the state that each starts from: as many as give every CU a workgroup, of
// 192 steps at least and 768 in all, or 512 and 1536 with gradients.  Us a call, whole
// against segments (B=1 64 x 64 bf16): 8 heads L=8192 107 against 28, L=2048 30 against
// 20, 16 heads L=4096 56 against 27; 48 workgroups, L=777, fp32 33 against 29, L=300 13
// against 19; with gradients 117 against 66, 36 against 38, 75 against 63.  Segments of
// 2048 steps and more are halved, as the shorter pass has several workgroups on a CU: 8
// heads L=65536 124 against 139, with gradients 365 against 388 (but L=8192 35 against
// 28).  Two segments cost what they save (B=4 L=4096 H=16 64 x 64: whole 63, in two 67;
// with gradients 170 and 199) but for K > 64, where the outputs are the larger part of a
// walk: B=2 L=4096 H=16 128 x 128 whole 104, in two 97; with gradients 345 and 396.
int64_t segments(int64_t heads, int64_t L, int64_t K, int64_t V, bool grads) {
  const int64_t wgs = heads * cdiv64(V, 32), most = L / (grads ? 512 : 192);
  const int64_t fill = wgs > 0 ? 256 / wgs : 1, n = fill < most ? fill : most;
  if (n < 3 || L < 768) return n >= 2 && K > 64 && !grads ? 2 : 1;
  return n < fill || L < n * 2048 ? n : 512 / wgs;
}

// Workgroups that share the value heads of a key head in the gradients of the inputs,
// by the workgroups that there are without: one for each head, and a sum of their dQ
// and dK, while that fills CUs.  Us a call (64 x 64, 8 value heads, B=2), shared against
// one after the other: 16 workgroups of 8 heads 34 against 94 (fp32), 64 of 4 31 against
// 44 (bf16), 128 of 2 31 against 33, of 8 70 against 85; 256 of 2 46 against 43, of 8 111
// against 103.
int64_t shared(int64_t wgs, int64_t heads) { return wgs < 192 ? heads : 1; }

// The chunked form's plan over a workspace at base (which may be null: sizes).  chunk:
// steps between the states that the gradients keep, 0 for the forward.
LinPlan lin_plan(char* base, int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V,
                 int64_t chunk) {
  LinPlan p = {};
  const int64_t heads = B * Hv, elems = (K <= 32 ? 32 : (K <= 64 ? 64 : 128)) * cdiv64(V, 32) * 32;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    char* q = base + at;
    at += cdiv64(bytes, 256) * 256;
    return q;
  };
  const int64_t nseg = segments(heads, L, K, V, chunk > 0);
  p.steps = cdiv64(cdiv64(L, nseg), 128) * 128;
  p.nseg = cdiv64(L, p.steps);
  if (p.nseg > 1) {
    p.ends = reinterpret_cast<float*>(take(heads * p.nseg * elems * 4));
    p.sums = reinterpret_cast<double*>(take(heads * p.nseg * 8));
    if (chunk) {
      p.back = reinterpret_cast<float*>(take(heads * p.nseg * elems * 4));
      p.back_sums = reinterpret_cast<double*>(take(heads * p.nseg * 8));
    }
  }
  if (chunk) {
    p.states = reinterpret_cast<float*>(take(heads * cdiv64(L, chunk) * elems * 4));
    p.grads = reinterpret_cast<float*>(take(heads * cdiv64(L, chunk) * elems * 4));
    p.split = shared(B * Hk * cdiv64(L, chunk), Hv / Hk);
    if (p.split > 1) p.part = reinterpret_cast<float*>(take(2 * p.split * B * L * Hk * K * 4));
  }
  p.bytes = at;
  return p;
}

// Which rows are whole 16-byte accesses (B=1 L=35201 2 heads 128 x 11 fp16: 57 us with
// those of q and k alone, 122 element by element).
LinRows whole_rows(int dtype, const LinArgs& a) {
  const int64_t E = dtype == TSSM_F32 ? 4 : 2;
  if (a.K % 8 || !aligned(a.q, 16) || !aligned(a.k, 16) ||
      (a.q_b | a.q_l | a.q_h | a.k_b | a.k_l | a.k_h) * E % 16)
    return kNoRows;
  if (a.V % 8 || !aligned(a.v, 16) || !aligned(a.o, 16) ||
      (a.v_b | a.v_l | a.v_h | a.o_b | a.o_l | a.o_h) * E % 16)
    return kKeyRows;
  return kAllRows;
}

bool fits(int dtype, int64_t stride, int64_t cols) {
  const int64_t most = (INT64_C(1) << 31) / (129 * (dtype == TSSM_F32 ? 4 : 2));
  return stride >= cols && stride < most;
}

// What the chunked kernels' buffer accesses ask for: the rows of q, k, v and o
// do not overlap, and a chunk's lie within 31 bits of its first.
bool chunk_rows(int dtype, const LinArgs& a) {
  return fits(dtype, a.q_l, a.K) && fits(dtype, a.k_l, a.K) && fits(dtype, a.v_l, a.V) &&
         fits(dtype, a.o_l, a.V);
}

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int64_t tssm_linear_attention_workspace_bytes(int64_t nbatch, int64_t L, int64_t Hk,
                                                         int64_t Hv, int64_t K, int64_t V) {
  if (!sizes_ok(nbatch, L, Hk, Hv, K, V)) return TSSM_ERR_SHAPE;
  if (!takes(K, V)) return TSSM_ERR_UNSUPPORTED;
  if (nbatch == 0 || by_steps(nbatch * Hv, L, V)) return 0;
  return lin_plan(nullptr, nbatch, L, Hk, Hv, K, V, 0).bytes;
}

extern "C" int tssm_linear_attention_forward(
    int dtype, const void* q, const void* k, const void* v, const float* g, const float* h0,
    void* o, float* h_last, int64_t nbatch, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V,
    int64_t sq_b, int64_t sq_l, int64_t sq_h, int64_t sk_b, int64_t sk_l, int64_t sk_h,
    int64_t sv_b, int64_t sv_l, int64_t sv_h, int64_t sg_b, int64_t sg_l, int64_t sg_h,
    int64_t so_b, int64_t so_l, int64_t so_h, float scale, void* workspace,
    int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(nbatch, L, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(takes(K, V), TSSM_ERR_UNSUPPORTED);
  if (nbatch == 0) return TSSM_OK;
  TSSM_CHECK(L == 0 || (q && k && v && g && o), TSSM_ERR_NULL);
  const LinArgs a = {q, k, v, g, h0, o, h_last, nbatch, L, Hk, Hv, K, V,
                     sq_b, sq_l, sq_h, sk_b, sk_l, sk_h, sv_b, sv_l, sv_h,
                     sg_b, sg_l, sg_h, so_b, so_l, so_h, scale};
  hipStream_t st = as_stream(stream);
  if (by_steps(nbatch * Hv, L, V) || !chunk_rows(dtype, a)) return lin_seq_launch(dtype, a, st);
  TSSM_CHECK(L < (INT64_C(1) << 31) && nbatch <= 0x7fffffff / Hv, TSSM_ERR_UNSUPPORTED);
  const LinPlan p = lin_plan(reinterpret_cast<char*>(workspace), nbatch, L, Hk, Hv, K, V, 0);
  TSSM_CHECK(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 256)),
             TSSM_ERR_WORKSPACE);
  const LinRows rows = whole_rows(dtype, a);
  const int rc = p.nseg > 1 ? lin_entry_launch(dtype, a, rows, p, st) : TSSM_OK;
  return rc ? rc : lin_walk_launch(dtype, a, rows, p, st);
}

extern "C" int tssm_linear_attention_step(int dtype, const void* q, const void* k, const void* v,
                                          const float* g, float* state, void* o, int64_t S,
                                          int64_t Hk, int64_t Hv, int64_t K, int64_t V,
                                          int64_t sq_s, int64_t sq_h, int64_t sk_s, int64_t sk_h,
                                          int64_t sv_s, int64_t sv_h, int64_t sg_s, int64_t sg_h,
                                          int64_t so_s, int64_t so_h, float scale, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(S, 1, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(takes(K, V), TSSM_ERR_UNSUPPORTED);
  if (S == 0) return TSSM_OK;
  TSSM_CHECK(q && k && v && g && state && o, TSSM_ERR_NULL);
  const LinArgs a = {q, k, v, g, state, o, state, S, 1, Hk, Hv, K, V,
                     sq_s, 0, sq_h, sk_s, 0, sk_h, sv_s, 0, sv_h,
                     sg_s, 0, sg_h, so_s, 0, so_h, scale};
  return lin_seq_launch(dtype, a, as_stream(stream));
}

extern "C" int64_t tssm_linear_attention_backward_workspace_bytes(int dtype, int64_t nbatch,
                                                                  int64_t L, int64_t Hk,
                                                                  int64_t Hv, int64_t K,
                                                                  int64_t V) {
  if (dtype < TSSM_F32 || dtype > TSSM_F16) return TSSM_ERR_DTYPE;
  if (!sizes_ok(nbatch, L, Hk, Hv, K, V)) return TSSM_ERR_SHAPE;
  if (!takes(K, V)) return TSSM_ERR_UNSUPPORTED;
  if (L == 0 || nbatch == 0) return 256;
  return lin_plan(nullptr, nbatch, L, Hk, Hv, K, V, kLinChunk).bytes;
}

extern "C" int tssm_linear_attention_backward(
    int dtype, const void* q, const void* k, const void* v, const float* g, const float* h0,
    const void* dout, const float* dh_last, void* dq, void* dk, void* dv, float* dg, float* dh0,
    int64_t nbatch, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V, int64_t sq_b,
    int64_t sq_l, int64_t sq_h, int64_t sk_b, int64_t sk_l, int64_t sk_h, int64_t sv_b,
    int64_t sv_l, int64_t sv_h, int64_t sg_b, int64_t sg_l, int64_t sg_h, int64_t sd_b,
    int64_t sd_l, int64_t sd_h, float scale, void* workspace, int64_t workspace_bytes,
    void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(nbatch, L, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(takes(K, V), TSSM_ERR_UNSUPPORTED);
  if (nbatch == 0 || L == 0) return TSSM_OK;
  TSSM_CHECK(q && k && v && g && dout && dq && dk && dv && dg, TSSM_ERR_NULL);
  TSSM_CHECK(L < (INT64_C(1) << 31) && nbatch <= 0x7fffffff / Hv, TSSM_ERR_UNSUPPORTED);
  // (no outputs: o stands for dV in the checks of rows, as they are read)
  LinArgs a = {q, k, v, g, h0, dv, nullptr, nbatch, L, Hk, Hv, K, V,
               sq_b, sq_l, sq_h, sk_b, sk_l, sk_h, sv_b, sv_l, sv_h,
               sg_b, sg_l, sg_h, V, V, V, scale};
  if (L == 1) {  // the strides of one step say nothing: those that chunks are read by
    a.q_l = a.k_l = K;
    a.v_l = sd_l = V;
  }
  TSSM_CHECK(chunk_rows(dtype, a) && fits(dtype, sd_l, V), TSSM_ERR_STRIDE);
  const LinPlan p = lin_plan(reinterpret_cast<char*>(workspace), nbatch, L, Hk, Hv, K, V, kLinChunk);
  TSSM_CHECK(workspace && workspace_bytes >= p.bytes && aligned(workspace, 256),
             TSSM_ERR_WORKSPACE);
  LinArgs way = a;  // the way back reads queries for keys and dO for v
  way.k = q;
  way.k_b = sq_b;
  way.k_l = a.q_l;
  way.k_h = sq_h;
  way.v = dout;
  way.v_b = sd_b;
  way.v_l = sd_l;
  way.v_h = sd_h;
  way.h0 = dh_last;
  way.h_last = dh0;
  const LinGrads d = {dout, sd_b, sd_l, sd_h, dq, dk, dv, dg};
  // (the gradients of the inputs are written as the inputs are read)
  const LinRows here = whole_rows(dtype, a), back = whole_rows(dtype, way);
  const LinRows rows =
      !aligned(dq, 16) || !aligned(dk, 16) ? kNoRows : (here < back ? here : back);
  hipStream_t st = as_stream(stream);
  const int rc = lin_states_launch(dtype, a, way, rows, p, st);
  return rc ? rc : lin_grads_launch(dtype, a, d, rows, p, st);
}
