// tl_logits.cu -- entry points over vocabulary rows (tl_token_logprobs,
// tl_token_logprobs_bwd, tl_distill_topk): argument checks and how rows are
// laid over the GPU.  The kernels are in tl_logits_score.cu and
// tl_logits_grad.cu.
//
// With y = z / temperature, m = max z, e_v = exp((z_v - m) / temperature) and
// s = sum e_v:  log p_v = (z_v - m) / temperature - log s  and
// H = log s - (1/s) sum e_v (z_v - m) / temperature.  Everything is taken
// relative to the row's largest logit, so rows of a type's lowest value (every
// token masked) and very large logits keep their distribution.
#include <algorithm>
#include <cmath>
#include "tl_logits_dev.cuh"

namespace tl {

// The choices below, each with what it was measured against (B200, us; "scaled"
// is 16384 x 8192 fp32, "50k" 2047 x 50001 fp16 or 4096 x 50000 bf16, "131k" N x
// 131072 bf16).  Both sides of a choice are of one build; figures of this build
// stand first where it is another.
//
//  * A row longer than one piece of 2048 chunks is split over a cluster where
//    there are no more rows than SMs: 131k scores with K = 20 take 8 instead of
//    29 us for 1 row, 16 against 30 for 74 and 24 against 31 for 148, but 36
//    against 35 for 296.  So many blocks a row that they fill the SMs once, two
//    at least: 74 rows of 32768 fp32 take 5.6, 5.9 and 7.7 us with 2, 4 and 8.
//    A row of one piece gains nothing from it (6.9 against 6.2 us for a
//    distilled row of 8192 fp32, 7.3 now).
//  * Alternatives: pieces of 2048 chunks, one stage, 128 threads (5 blocks an
//    SM): scaled K = 64 takes 211 us; 205, with two stages (3 blocks) 235, with
//    256 threads 272, with pieces of 1024 chunks 250.  Above K = 64 rows of more
//    than 1024 chunks have 256 threads: K = 128 takes 510 us with them and 2069
//    with 128, whose four warps' maxima are too few for a threshold.  Rows of up
//    to 1024 chunks keep 128 threads at any K, and there it is not always high
//    enough: K above 124 takes all 32 maxima of each warp, and 50 to 90 % of
//    random rows of 800 to 8192 logits overflow their list and go to select_row;
//    16-bit rows of 32 to 127 chunks have no threshold where K is above 32 a full
//    warp, and overflow with more logits than the list holds (320, above K = 64
//    512).  Below that one warp sorts 2 K and more a row: 16384 x 1000 fp32, K =
//    100 takes 271 us, 20 without alternatives.
//  * No alternatives: pieces of 1024 chunks, two stages, 128 threads: 83 us
//    scaled; 86 and for 50k 81, one stage of 2048 and 256 threads 92 and 100.
//  * Distillation: 256 threads, pieces of 2048 chunks, two stages: 223 us scaled
//    and 111 for 50k; two stages against one, in an earlier build, 207 against
//    224 and 104 against 123.  Rows of six pieces or more, which come twice, three
//    stages: so two blocks an SM, whose rows stay in L2 in between, 221 us for
//    2048 rows of 131k; 218 against 242.
//  * Short rows, up to 256 chunks, have one computing warp, if its 32 maxima are
//    enough for a threshold (K <= 16).
RowPlan plan_rows(const DeviceCtx *c, const LogitRows &z, int K, bool twice) {
  const int es = z.dtype == TL_F32 ? 4 : 2, ev = 16 / es;
  // chunks of a row: its own alignment where all rows share it, else the worst
  const bool one = (z.ld * es) % 16 == 0 || z.N == 1;
  const int mis = one ? (int)(reinterpret_cast<uintptr_t>(z.p) & 15) / es : ev - 1;
  const int nch = (z.V + mis + ev - 1) / ev;
  constexpr int kPiece = 2048, kMostPerBlock = 6144;           // of a cluster: 96 KB in one stage
  RowPlan p{256, 1, {z.p, z.ld, z.N, z.V, nch, 1, 1, 0, 0, c->copy_wait_ns}};
  if (nch > kPiece && z.N <= c->num_sms) {
    p.blocks = 2;
    while (z.N * p.blocks * 2 <= c->num_sms && p.blocks < 8) p.blocks *= 2;
    p.blocks = std::max(p.blocks, (nch + kMostPerBlock - 1) / kMostPerBlock);
    p.l.per = (nch + p.blocks - 1) / p.blocks;
    p.l.pieces = p.blocks;
    p.threads = p.l.per <= 512 ? 128 : p.l.per <= 2048 ? 256 : 512;
  } else {
    p.threads = nch <= 256 && K <= 16 ? 32 : nch <= 1024 ? 128 : twice || K > 64 ? 256 : 128;
    p.l.per = std::min(nch, twice || K > 0 ? kPiece : kPiece / 2);
    p.l.pieces = (nch + p.l.per - 1) / p.l.per;
    p.l.stages = p.threads == 32 ? 4 : !twice && K > 0 ? 1 : twice && p.l.pieces >= 6 ? 3 : 2;
  }
  p.l.chunks = (p.l.per + 7) / 8 * 8;
  p.l.ragged = !one || mis || (z.V % ev) != 0;
  return p;
}

int launch_rows(const void *kernel, DeviceCtx *c, const RowPlan &p, int more_threads, int more_smem, Resident *seen, void *args) {
  constexpr int kMaxDynamic = 212 * 1024;          // of 227 KB a block may have, less the kernels' static part
  const int smem = p.l.stages * p.l.chunks * 16 + more_smem;
  if (smem > kMaxDynamic) return set_error(TL_EINVAL, "rows need %d bytes of shared memory a block", smem);
  cudaLaunchConfig_t cfg = {};
  const int threads = p.threads + more_threads;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = c->stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)p.blocks;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  if (p.blocks > 1) {
    cfg.attrs = &at;
    cfg.numAttrs = 1;
  }
  if (!seen->ready) {
    TL_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamic));
    TL_TRY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    seen->ready = 1;
  }
  int fit = 0;
  for (const Resident::Shape &s : seen->of)
    if (s.threads == threads && s.blocks == p.blocks && s.smem == smem) fit = s.fit;
  if (!fit) {
    if (p.blocks == 1) {
      TL_TRY_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, (size_t)smem));
      fit *= c->num_sms;
    } else {
      cfg.gridDim = dim3((unsigned)p.blocks);
      TL_TRY_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
    }
    if (fit < 1) return set_error(TL_ECUDA, "%d blocks of %d threads and %d bytes do not fit", p.blocks, threads, smem);
    seen->of[seen->next] = Resident::Shape{threads, p.blocks, smem, fit};
    seen->next = (seen->next + 1) % Resident::N;
  }
  cfg.gridDim = dim3((unsigned)((p.l.N < fit ? p.l.N : fit) * p.blocks));
  void *argv[1] = {args};
  TL_TRY_CUDA(cudaLaunchKernelExC(&cfg, kernel, argv));
  return TL_OK;
}

int check_temperature(float t) {
  if (!(t >= 1e-6f && t <= 1e6f)) return set_error(TL_EINVAL, "temperature %g outside [1e-6, 1e6]", (double)t);
  return TL_OK;
}
int check_topk(int K, int V) {
  if (K < 0 || K > TL_TOPK_MAX || K > V)
    return set_error(TL_EINVAL, "K = %d outside [0, min(%d, V = %d)]", K, TL_TOPK_MAX, V);
  return TL_OK;
}
int check_ptr_here(DeviceCtx *c, const void *p, const char *name, size_t align) {
  if (!p) return set_error(TL_EINVAL, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % align)
    return set_error(TL_EALIGN, "%s is not aligned to its %zu-byte elements", name, align);
  cudaPointerAttributes a;
  const cudaError_t e = cudaPointerGetAttributes(&a, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(TL_EPTR, "%s: not a CUDA pointer (%s)", name, cudaGetErrorString(e));
  }
  if (a.type == cudaMemoryTypeManaged) return TL_OK;
  if (a.type != cudaMemoryTypeDevice)
    return set_error(TL_EPTR, "%s is a host pointer; the library computes on device memory only", name);
  if (a.device != c->device)
    return set_error(TL_EINVAL, "%s is memory of device %d, the call runs on device %d", name, a.device, c->device);
  return TL_OK;
}

namespace {

size_t dtype_size(int dtype) { return dtype == TL_F32 ? 4 : 2; }

int check_rows(int dtype, long long ld, int N, int V, const char *what) {
  if (dtype != TL_F32 && dtype != TL_BF16 && dtype != TL_F16)
    return set_error(TL_EINVAL, "dtype %d is none of TL_F32, TL_BF16, TL_F16", dtype);
  if (N < 0 || N > (1 << 30) || V < 1 || V > TL_VOCAB_MAX)
    return set_error(TL_EINVAL, "N = %d, V = %d: 0 <= N <= 2^30 and 1 <= V <= %d are taken", N, V, TL_VOCAB_MAX);
  if (ld < V || ld > (1LL << 40)) return set_error(TL_EINVAL, "row stride of %s %lld below V = %d", what, ld, V);
  return TL_OK;
}

// A gradient may take its logits' own place (the same rows), or rows that share
// no element with them: other memory, or, with the same stride, the space
// between them.
int check_in_place(const void *dz, long long ldd, const LogitRows &z) {
  if (dz == z.p && (ldd == z.ld || z.N == 1)) return TL_OK;
  const long long es = (long long)dtype_size(z.dtype);
  const uintptr_t a = reinterpret_cast<uintptr_t>(dz), b = reinterpret_cast<uintptr_t>(z.p);
  const uintptr_t a1 = a + ((size_t)(z.N - 1) * ldd + z.V) * es, b1 = b + ((size_t)(z.N - 1) * z.ld + z.V) * es;
  if (a >= b1 || b >= a1) return TL_OK;
  if (ldd == z.ld) {
    const long long between = (a > b ? (long long)(a - b) : (long long)(b - a)) / es % ldd;
    if (between >= z.V && between <= ldd - z.V) return TL_OK;
  }
  return set_error(TL_EINVAL, "dlogits overlaps logits without being the same rows");
}

}  // namespace
}  // namespace tl

using namespace tl;

#define TRY(x) do { int _rc = (x); if (_rc) return _rc; } while (0)

TL_API int tl_token_logprobs(const void *logits, int dtype, long long ld, const int *ids, int N, int V,
                             float temperature, float *logp, float *entropy, float *stats, int K, int *top_ids,
                             float *top_logp) {
  TRY(check_rows(dtype, ld, N, V, "logits"));
  TRY(check_temperature(temperature));
  TRY(check_topk(K, V));
  if (N > 0 && !logp && !entropy && !stats && K == 0) return set_error(TL_EINVAL, "no output asked for");
  if (N > 0 && (logp != nullptr) != (ids != nullptr)) return set_error(TL_EINVAL, "ids and logp come together");
  if (K == 0 && (top_ids || top_logp)) return set_error(TL_EINVAL, "top_ids and top_logp take K >= 1");
  TL_REQUIRE_CTX(c);
  if (N == 0) return TL_OK;
  TRY(check_ptr_here(c, logits, "logits", dtype_size(dtype)));
  if (logp) {
    TRY(check_ptr_here(c, ids, "ids", 4));
    TRY(check_ptr_here(c, logp, "logp", 4));
  }
  if (entropy) TRY(check_ptr_here(c, entropy, "entropy", 4));
  if (stats) TRY(check_ptr_here(c, stats, "stats", 4));
  if (K) {
    TRY(check_ptr_here(c, top_ids, "top_ids", 4));
    TRY(check_ptr_here(c, top_logp, "top_logp", 4));
  }
  return k_token_logprobs(c, LogitRows{logits, dtype, ld, N, V}, ids, temperature, logp, entropy, stats, K, top_ids,
                          top_logp);
}

TL_API int tl_token_logprobs_bwd(void *dlogits, long long ldd, const void *logits, int dtype, long long ld,
                                 const int *ids, int N, int V, float temperature, const float *stats,
                                 const float *entropy, const float *dlogp, const float *dentropy) {
  TRY(check_rows(dtype, ld, N, V, "logits"));
  TRY(check_rows(dtype, ldd, N, V, "dlogits"));
  TRY(check_temperature(temperature));
  if (N > 0 && !dlogp && !dentropy) return set_error(TL_EINVAL, "neither dlogp nor dentropy given");
  if (N > 0 && dlogp && !ids) return set_error(TL_EINVAL, "dlogp takes ids");
  if (N > 0 && dentropy && !entropy) return set_error(TL_EINVAL, "dentropy takes the forward pass's entropy");
  TL_REQUIRE_CTX(c);
  if (N == 0) return TL_OK;
  TRY(check_ptr_here(c, logits, "logits", dtype_size(dtype)));
  TRY(check_ptr_here(c, dlogits, "dlogits", dtype_size(dtype)));
  TRY(check_ptr_here(c, stats, "stats", 4));
  if (dlogp) {
    TRY(check_ptr_here(c, ids, "ids", 4));
    TRY(check_ptr_here(c, dlogp, "dlogp", 4));
  }
  if (dentropy) {
    TRY(check_ptr_here(c, entropy, "entropy", 4));
    TRY(check_ptr_here(c, dentropy, "dentropy", 4));
  }
  const LogitRows z{logits, dtype, ld, N, V};
  TRY(check_in_place(dlogits, ldd, z));
  return k_token_logprobs_bwd(c, dlogits, ldd, z, ids, temperature, stats, entropy, dlogp, dentropy);
}

TL_API int tl_distill_topk(const void *logits, int dtype, long long ld, const int *t_ids, const float *t_vals, int K,
                           int N, int V, float temperature, int tail, const float *weight, float scale, float *loss,
                           void *dlogits, long long ldd) {
  TRY(check_rows(dtype, ld, N, V, "logits"));
  if (dlogits) TRY(check_rows(dtype, ldd, N, V, "dlogits"));
  TRY(check_temperature(temperature));
  TRY(check_topk(K, V));
  if (K < 1) return set_error(TL_EINVAL, "K = 0: a teacher names at least one token");
  if (tail != 0 && tail != 1) return set_error(TL_EINVAL, "tail %d is neither 0 nor 1", tail);
  if (!std::isfinite(scale)) return set_error(TL_EINVAL, "scale is not finite");
  if (N > 0 && !loss && !dlogits) return set_error(TL_EINVAL, "no output asked for");
  TL_REQUIRE_CTX(c);
  if (N == 0) return TL_OK;
  TRY(check_ptr_here(c, logits, "logits", dtype_size(dtype)));
  TRY(check_ptr_here(c, t_ids, "t_ids", 4));
  TRY(check_ptr_here(c, t_vals, "t_vals", 4));
  if (weight) TRY(check_ptr_here(c, weight, "weight", 4));
  if (loss) TRY(check_ptr_here(c, loss, "loss", 4));
  const LogitRows z{logits, dtype, ld, N, V};
  if (dlogits) {
    TRY(check_ptr_here(c, dlogits, "dlogits", dtype_size(dtype)));
    TRY(check_in_place(dlogits, ldd, z));
  }
  return k_distill_topk(c, z, t_ids, t_vals, K, temperature, tail, weight, scale, loss, nullptr, dlogits, ldd);
}
