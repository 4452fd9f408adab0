// Entry points of linear attention: argument checks and the choice of kernels.
#include "linattn.h"

namespace tssm {
namespace {

bool sizes_ok(int64_t B, int64_t L, int64_t Hk, int64_t Hv, int64_t K, int64_t V) {
  return B >= 0 && L >= 0 && Hk > 0 && Hv > 0 && Hv % Hk == 0 && K > 0 && V > 0;
}
// A head's state takes 31 bits.
bool takes(int64_t K, int64_t V) { return K <= 128 && V <= (INT64_C(1) << 21); }

}  // namespace
}  // namespace tssm

using namespace tssm;

extern "C" int64_t tssm_linear_attention_workspace_bytes(int64_t nbatch, int64_t L, int64_t Hk,
                                                         int64_t Hv, int64_t K, int64_t V) {
  if (!sizes_ok(nbatch, L, Hk, Hv, K, V)) return TSSM_ERR_SHAPE;
  if (!takes(K, V)) return TSSM_ERR_UNSUPPORTED;
  return 0;
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
  (void)workspace;
  (void)workspace_bytes;
  return lin_seq_launch(dtype, a, as_stream(stream));
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
