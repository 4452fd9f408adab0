// Entry points of the gated delta rule: argument checks and the choice of
// kernels.
#include "delta.h"

namespace tssm {
namespace {

bool sizes_ok(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V) {
  return B >= 0 && L >= 0 && Hk > 0 && Hv > 0 && Hv % Hk == 0 && K > 0 && V > 0;
}

// Sequences up to here go step by step.  That takes 3 us and 0.6 us a step (B =
// 1, 8 heads of 64 x 64: 5.3, 7.6 and 12.3 us at L = 4, 8 and 16); one chunk's
// way through the chunked kernels takes 10.5 us at any L, and 23 us once the
// chip has more than two heads on each CU (512 heads: 10.3, 16.4, 21.7 and 26.8
// us step by step at L = 8, 16, 24 and 32).  That is 64 x 64 in bf16; the two
// ways meet at 10 tokens for 12 heads of 40 x 72 in fp32, at 16 to 19 for 16 and 32
// of 128 x 128, and beyond 32 for 512 of 128 x 128 (25 tokens: 47 us step by step,
// 100 in chunks) and 1024 of 40 x 72.
bool by_steps(int64_t heads, int64_t L) { return L <= (heads >= 512 ? 24 : 12); }

// How many segments a sequence of nch chunks is walked in, by the times that the
// walks take (in tenths of a chunk's time of one workgroup on each CU, a
// microsecond): the outputs' walk fills a CU with one workgroup of 32 columns;
// the walk from zero over V + KP columns, which s > 1 segments add, takes 1.5
// and 2 times as long a chunk with two and four workgroups on a CU; joining
// takes a chunk's time a segment, the two launches more twelve.  B = 1, L = 65536,
// H = 8, K = V = 64, bf16: 1780 us in one segment; with 8, 16, 32 and 64: 513, 375,
// 332 and 406.  The rule compares times only, and other sizes keep about these
// proportions: with 128 x 128 and 40 x 72, in fp32 and fp16, and in the gradients,
// whose two walks go side by side, seven more calls took at most 7% more than
// with the best of ten counts.
int64_t segments(int64_t heads, int64_t nch, int64_t KP, int64_t V) {
  const int64_t out = heads * cdiv64(V, 32), all = heads * (cdiv64(V, 32) + KP / 32);
  int64_t best = 1, least = nch * 10 * cdiv64(out, 256);
  for (int64_t s = 2; s <= 512 && s <= nch / 4; s = s < 8 ? s + 1 : s + s / 8) {
    const int64_t per = cdiv64(nch, s), w = (s - 1) * all;
    const int64_t zero = w <= 256 ? 10 : (w <= 512 ? 15 : 20 * cdiv64(w, 1024));
    const int64_t cost = per * (zero + 10 * cdiv64(cdiv64(nch, per) * out, 256)) + 10 * s + 120;
    if (cost < least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

// The chunked form's plan over a workspace at base (which may be null: sizes).
DeltaPlan delta_plan(char* base, int64_t B, int64_t L, int64_t Hv, int64_t K, int64_t V,
                     bool gradients) {
  DeltaPlan p = {};
  const int64_t nch = cdiv64(L, 32), heads = B * Hv, KP = K <= 32 ? 32 : (K <= 64 ? 64 : 128);
  const int64_t Vp = cdiv64(V, 16) * 16;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    char* q = base + at;
    at += cdiv64(bytes, 256) * 256;
    return q;
  };
  p.nch = (int)nch;
  p.per = (int)cdiv64(nch, segments(heads, nch, KP, V));
  p.nseg = (int)cdiv64(nch, p.per);
  p.chunks = take(heads * nch * delta_chunk_ws_bytes());
  if (p.nseg > 1) {
    p.transfer = reinterpret_cast<float*>(take(heads * p.nseg * (Vp + KP) * KP * 4));
    p.entry = reinterpret_cast<float*>(take(heads * p.nseg * Vp * KP * 4));
  }
  if (gradients) {
    if (p.nseg > 1) {
      p.back = reinterpret_cast<float*>(take(heads * p.nseg * Vp * KP * 4));
      p.gentry = reinterpret_cast<float*>(take(heads * p.nseg * Vp * KP * 4));
    }
    p.states = reinterpret_cast<float*>(take(heads * nch * Vp * KP * 4));
    p.grads = reinterpret_cast<float*>(take(heads * nch * Vp * KP * 4));
  }
  p.bytes = at;
  return p;
}

// The rows of q, k and v are whole 16-byte accesses.
bool vec_rows(int dtype, const DeltaArgs& a) {
  const int64_t E = dtype == TSSM_F32 ? 4 : 2;
  return a.K % 8 == 0 && a.V % 8 == 0 && aligned(a.q, 16) && aligned(a.k, 16) &&
         aligned(a.v, 16) &&
         (a.q_b | a.q_l | a.q_h | a.k_b | a.k_l | a.k_h | a.v_b | a.v_l | a.v_h) * E % 16 == 0;
}

bool fits(int dtype, int64_t stride, int64_t cols) {
  const int64_t most = (INT64_C(1) << 31) / (33 * (dtype == TSSM_F32 ? 4 : 2));
  return stride >= cols && stride < most;
}

// What the chunked kernels' buffer accesses ask for: the rows of q, k, v and o
// do not overlap, and a chunk's lie within 31 bits of its first.
bool chunk_rows(int dtype, const DeltaArgs& a) {
  return fits(dtype, a.q_l, a.K) && fits(dtype, a.k_l, a.K) && fits(dtype, a.v_l, a.V) &&
         fits(dtype, a.o_l, a.V);
}

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int tssm_gated_delta_forward(
    int dtype, const void* q, const void* k, const void* v, const float* g, const float* beta,
    const float* h0, void* o, float* h_last, int64_t nbatch, int64_t L, int64_t Hk, int64_t Hv,
    int64_t K, int64_t V, int64_t sq_b, int64_t sq_l, int64_t sq_h, int64_t sk_b, int64_t sk_l,
    int64_t sk_h, int64_t sv_b, int64_t sv_l, int64_t sv_h, int64_t sg_b, int64_t sg_l,
    int64_t sg_h, int64_t sbe_b, int64_t sbe_l, int64_t sbe_h, int64_t so_b, int64_t so_l,
    int64_t so_h, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(nbatch, L, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(K <= 128, TSSM_ERR_UNSUPPORTED);
  if (nbatch == 0) return TSSM_OK;
  TSSM_CHECK(L == 0 || (q && k && v && g && beta && o), TSSM_ERR_NULL);
  const DeltaArgs a = {q, k, v, g, beta, h0, o, h_last, nbatch, L, Hk, Hv, K, V,
                       sq_b, sq_l, sq_h, sk_b, sk_l, sk_h, sv_b, sv_l, sv_h,
                       sg_b, sg_l, sg_h, sbe_b, sbe_l, sbe_h, so_b, so_l, so_h, scale};
  if (by_steps(nbatch * Hv, L) || !chunk_rows(dtype, a))
    return delta_seq_launch(dtype, a, as_stream(stream));
  TSSM_CHECK(nbatch * Hv <= 0x7fffffff / cdiv64(L, 32), TSSM_ERR_UNSUPPORTED);
  const DeltaPlan p = delta_plan(reinterpret_cast<char*>(workspace), nbatch, L, Hv, K, V, false);
  TSSM_CHECK(workspace && workspace_bytes >= p.bytes && aligned(workspace, 256),
             TSSM_ERR_WORKSPACE);
  const bool vec = vec_rows(dtype, a);
  hipStream_t st = as_stream(stream);
  int rc = delta_prep_launch(dtype, a, vec, p.chunks, st);
  if (!rc && p.nseg > 1) rc = delta_transfer_launch(dtype, a, vec, p, st);
  return rc ? rc : delta_walk_launch(dtype, a, vec, p, st);
}

extern "C" int tssm_gated_delta_step(int dtype, const void* q, const void* k, const void* v,
                                     const float* g, const float* beta, float* state, void* o,
                                     int64_t S, int64_t Hk, int64_t Hv, int64_t K, int64_t V,
                                     int64_t sq_s, int64_t sq_h, int64_t sk_s, int64_t sk_h,
                                     int64_t sv_s, int64_t sv_h, int64_t sg_s, int64_t sg_h,
                                     int64_t sbe_s, int64_t sbe_h, int64_t so_s, int64_t so_h,
                                     float scale, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(S, 1, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(K <= 128, TSSM_ERR_UNSUPPORTED);
  if (S == 0) return TSSM_OK;
  TSSM_CHECK(q && k && v && g && beta && state && o, TSSM_ERR_NULL);
  const DeltaArgs a = {q, k, v, g, beta, state, o, state, S, 1, Hk, Hv, K, V,
                       sq_s, 0, sq_h, sk_s, 0, sk_h, sv_s, 0, sv_h,
                       sg_s, 0, sg_h, sbe_s, 0, sbe_h, so_s, 0, so_h, scale};
  return delta_seq_launch(dtype, a, as_stream(stream));
}

extern "C" int64_t tssm_gated_delta_workspace_bytes(int64_t nbatch, int64_t L, int64_t Hk,
                                                    int64_t Hv, int64_t K, int64_t V) {
  if (!sizes_ok(nbatch, L, Hk, Hv, K, V)) return TSSM_ERR_SHAPE;
  if (K > 128) return TSSM_ERR_UNSUPPORTED;
  if (nbatch == 0 || by_steps(nbatch * Hv, L)) return 0;
  return delta_plan(nullptr, nbatch, L, Hv, K, V, false).bytes;
}

extern "C" int64_t tssm_gated_delta_backward_workspace_bytes(int64_t nbatch, int64_t L, int64_t Hk,
                                                             int64_t Hv, int64_t K, int64_t V) {
  if (!sizes_ok(nbatch, L, Hk, Hv, K, V)) return TSSM_ERR_SHAPE;
  if (K > 128) return TSSM_ERR_UNSUPPORTED;
  if (L == 0 || nbatch == 0) return 256;
  return delta_plan(nullptr, nbatch, L, Hv, K, V, true).bytes;
}

extern "C" int tssm_gated_delta_backward(
    int dtype, const void* q, const void* k, const void* v, const float* g, const float* beta,
    const float* h0, const void* dout, const float* dh_last, void* dq, void* dk, void* dv,
    float* dg, float* dbeta, float* dh0, int64_t nbatch, int64_t L, int64_t Hk, int64_t Hv,
    int64_t K, int64_t V, int64_t sq_b, int64_t sq_l, int64_t sq_h, int64_t sk_b, int64_t sk_l,
    int64_t sk_h, int64_t sv_b, int64_t sv_l, int64_t sv_h, int64_t sg_b, int64_t sg_l,
    int64_t sg_h, int64_t sbe_b, int64_t sbe_l, int64_t sbe_h, int64_t sd_b, int64_t sd_l,
    int64_t sd_h, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  TSSM_CHECK(dtype >= TSSM_F32 && dtype <= TSSM_F16, TSSM_ERR_DTYPE);
  TSSM_CHECK(sizes_ok(nbatch, L, Hk, Hv, K, V), TSSM_ERR_SHAPE);
  TSSM_CHECK(K <= 128, TSSM_ERR_UNSUPPORTED);
  if (nbatch == 0 || L == 0) return TSSM_OK;
  TSSM_CHECK(q && k && v && g && beta && dout && dq && dk && dv && dg && dbeta, TSSM_ERR_NULL);
  TSSM_CHECK(nbatch * Hv <= 0x7fffffff / cdiv64(L, 32), TSSM_ERR_UNSUPPORTED);
  DeltaArgs a = {q, k, v, g, beta, h0, nullptr, nullptr, nbatch, L, Hk, Hv, K, V,
                 sq_b, sq_l, sq_h, sk_b, sk_l, sk_h, sv_b, sv_l, sv_h,
                 sg_b, sg_l, sg_h, sbe_b, sbe_l, sbe_h, V, V, V, scale};
  TSSM_CHECK(V <= (INT64_C(1) << 21), TSSM_ERR_UNSUPPORTED);  // a state takes 31 bits
  if (L == 1) {  // the strides of one step say nothing: those that chunks are read by
    a.q_l = a.k_l = K;
    a.v_l = sd_l = V;
  }
  TSSM_CHECK(chunk_rows(dtype, a) && fits(dtype, sd_l, V), TSSM_ERR_STRIDE);
  const DeltaPlan p = delta_plan(reinterpret_cast<char*>(workspace), nbatch, L, Hv, K, V, true);
  TSSM_CHECK(workspace && workspace_bytes >= p.bytes && aligned(workspace, 256),
             TSSM_ERR_WORKSPACE);
  DeltaArgs way = a;  // the way back reads dO where the walk reads v
  way.v = dout;
  way.v_b = sd_b;
  way.v_l = sd_l;
  way.v_h = sd_h;
  way.h0 = dh_last;
  way.h_last = dh0;
  const DeltaGrads d = {dout, sd_b, sd_l, sd_h, dq, dk, dv, dg, dbeta};
  // (the gradients of the inputs are written as the inputs are read)
  const bool vec = vec_rows(dtype, a) && vec_rows(dtype, way) && aligned(dq, 16) &&
                   aligned(dk, 16) && aligned(dv, 16);
  hipStream_t st = as_stream(stream);
  int rc = delta_prep_launch(dtype, a, vec, p.chunks, st);
  if (!rc) rc = delta_both_launch(dtype, a, way, vec, p, st);
  return rc ? rc : delta_grads_launch(dtype, a, d, vec, p, st);
}
