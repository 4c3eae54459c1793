// tl_logits.cuh -- operators over vocabulary rows (logits [N][V]): what the
// entry points of tl_logits.cu and the model paths share.
#pragma once
#include "tl_common.cuh"

namespace tl {

// A call's logits: N rows of V values of one type, row n at p + n * ld.
struct LogitRows {
  const void *p;
  int dtype;        // TL_F32, TL_BF16 or TL_F16
  long long ld;
  int N, V;
};

// The launches behind tl_token_logprobs, tl_token_logprobs_bwd and
// tl_distill_topk, arguments already checked.  loss64: the same row losses in
// double, for loss_sum (either may be nullptr).
int k_token_logprobs(DeviceCtx *c, const LogitRows &z, const int *ids, float temperature, float *logp,
                     float *entropy, float *stats, int K, int *top_ids, float *top_logp);
int k_token_logprobs_bwd(DeviceCtx *c, void *dlogits, long long ldd, const LogitRows &z, const int *ids,
                         float temperature, const float *stats, const float *entropy, const float *dlogp,
                         const float *dentropy);
int k_distill_topk(DeviceCtx *c, const LogitRows &z, const int *t_ids, const float *t_vals, int K,
                   float temperature, int tail, const float *weight, float scale, float *loss, double *loss64,
                   void *dlogits, long long ldd);

// Argument checks shared with the model paths.
int check_temperature(float t);
int check_topk(int K, int V);
// TL_EINVAL for memory of another device, TL_EPTR for host memory, TL_EALIGN
// where p is not a multiple of `align` bytes.
int check_ptr_here(DeviceCtx *c, const void *p, const char *name, size_t align);

}  // namespace tl
