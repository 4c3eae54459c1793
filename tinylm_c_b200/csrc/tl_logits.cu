// tl_logits.cu -- operators over vocabulary rows: log probabilities of given
// tokens with the row's entropy and most likely tokens, their gradient, and
// distillation from a teacher's most likely tokens.
//
// With y = z / temperature, m = max z, e_v = exp((z_v - m) / temperature) and
// s = sum e_v:  log p_v = (z_v - m) / temperature - log s  and
// H = log s - (1/s) sum e_v (z_v - m) / temperature.  Everything is taken
// relative to the row's largest logit, so rows of a type's lowest value (every
// token masked) and very large logits keep their distribution.
#include <cfloat>
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tl_logits.cuh"
#include "tl_trace.cuh"

namespace tl {
namespace lg {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// The smallest mass that counts as a teacher's tail: below it 1 - sum q is
// the rounding of q, not probability.
constexpr float TAIL_MIN = 0x1p-20f;

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float block_max(float v, float *red) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); i++) v = fmaxf(v, red[i]);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float *red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); i++) v += red[i];
  return v;
}
__device__ __forceinline__ unsigned long long block_max64(unsigned long long v, unsigned long long *red) {
  for (int o = 16; o; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(~0u, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); i++) v = red[i] > v ? red[i] : v;
  return v;
}

// Order of the alternatives as one integer: larger logit first, then the
// lower index.  x + 0 makes -0 equal to +0.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int v) {
  return ((unsigned long long)order_of(x) << 32) | (0xFFFFFFFFu - (unsigned)v);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const unsigned u = (unsigned)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// (1/s) sum e d is taken with d bounded below, where e is 0 anyway: -inf
// would make it NaN.
__device__ __forceinline__ float bounded(float d) { return d < -1e30f ? -1e30f : d; }

// One block a row, straight from the formulas: the row is read once for its
// maximum, once for its sums and once for every alternative.
template <typename T>
__global__ void __launch_bounds__(256)
token_logprobs_kernel(const T *__restrict__ z0, long long ld, const int *__restrict__ ids, int V, float inv_t,
                      float *__restrict__ logp, float *__restrict__ entropy, float *__restrict__ stats, int K,
                      int *__restrict__ top_ids, float *__restrict__ top_logp, int *err) {
  __shared__ float red[8];
  __shared__ unsigned long long red64[8];
  const size_t n = blockIdx.x;
  const T *z = z0 + n * ld;
  float m = -FLT_MAX;
  for (int v = threadIdx.x; v < V; v += 256) m = fmaxf(m, to_f(z[v]));
  m = block_max(m, red);
  float s = 0.0f, t = 0.0f;
  for (int v = threadIdx.x; v < V; v += 256) {
    const float d = (to_f(z[v]) - m) * inv_t, e = expf(d);
    s += e;
    t += e * bounded(d);
  }
  s = block_sum(s, red);
  t = block_sum(t, red);
  const bool bad = !(s >= 0.0f);          // a NaN or an infinite logit: no distribution
  const float ls = logf(s);               // -inf where nothing is left
  if (threadIdx.x == 0) {
    if (logp) {
      const int id = ids[n];
      float lp = 0.0f;
      if (id >= 0 && id < V) lp = s == 0.0f ? -INFINITY : (to_f(z[id]) - m) * inv_t - ls;
      else if (id != -1) atomicExch(err, 100);
      logp[n] = lp;
    }
    if (entropy) {
      const float h = ls - t / s;
      entropy[n] = s == 0.0f || h < 0.0f ? 0.0f : h;
    }
    if (stats) {
      stats[2 * n] = m;
      stats[2 * n + 1] = s == 0.0f ? INFINITY : ls;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < K; k++) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < V; v += 256) {
      const float x = to_f(z[v]);
      if (x > -INFINITY) {
        const unsigned long long q = key_of(x, v);
        if (q < last && q > best) best = q;
      }
    }
    best = block_max64(best, red64);
    if (threadIdx.x == 0) {
      const bool none = bad || best == 0;
      top_ids[n * K + k] = none ? -1 : (int)(0xFFFFFFFFu - (unsigned)best);
      top_logp[n * K + k] = bad ? NAN : none ? -INFINITY : (value_of(best) - m) * inv_t - ls;
    }
    last = best ? best : 1;                // nothing left: later rounds find nothing
  }
}

// dz_v = (1/t) [ a (1[v = id] - p_v) - b p_v (log p_v + H) ]
template <typename T>
__global__ void __launch_bounds__(256)
token_logprobs_bwd_kernel(T *dz0, long long ldd, const T *z0, long long ld, const int *__restrict__ ids, int V,
                          float inv_t, const float *__restrict__ stats, const float *__restrict__ entropy,
                          const float *__restrict__ dlogp, const float *__restrict__ dentropy, int *err) {
  const size_t n = blockIdx.x;
  const T *z = z0 + n * ld;
  T *dz = dz0 + n * ldd;
  const int id = dlogp ? ids[n] : -1;
  const bool given = id >= 0 && id < V;
  if (!given && id != -1 && threadIdx.x == 0) atomicExch(err, 100);
  const float m = stats[2 * n], ls = stats[2 * n + 1];
  const bool empty = ls == INFINITY;
  const float a = given && !empty ? dlogp[n] : 0.0f;
  const float b = dentropy && !empty ? dentropy[n] : 0.0f, H = b != 0.0f ? entropy[n] : 0.0f;
  if (a == 0.0f && b == 0.0f) {            // nothing comes back to this row: it is not read
    for (int v = threadIdx.x; v < V; v += 256) dz[v] = from_f<T>(0.0f);
    return;
  }
  for (int v = threadIdx.x; v < V; v += 256) {
    const float lp = bounded((to_f(z[v]) - m) * inv_t - ls), p = expf(lp);
    float g = -p * (a + b * (lp + H));
    if (v == id) g += a;
    dz[v] = from_f<T>(g * inv_t);
  }
}

// KL(q || p) of one row a block and its gradient; see k_distill_topk.
template <typename T>
__global__ void __launch_bounds__(256)
distill_topk_kernel(const T *z0, long long ld, const int *__restrict__ t_ids, const float *__restrict__ t_vals, int K,
                    int V, float inv_t, int tail, const float *__restrict__ weight, float scale,
                    float *__restrict__ loss, double *__restrict__ loss64, T *dz0, long long ldd, int *err) {
  __shared__ float red[8];
  __shared__ int s_id[TL_TOPK_MAX];
  __shared__ float s_q[TL_TOPK_MAX], s_z[TL_TOPK_MAX];
  const size_t n = blockIdx.x;
  const T *z = z0 + n * ld;
  T *dz = dz0 ? dz0 + n * ldd : nullptr;
  const float w = weight ? weight[n] : 1.0f;
  if (w == 0.0f) {                         // a row that does not count is not read
    if (dz)
      for (int v = threadIdx.x; v < V; v += 256) dz[v] = from_f<T>(0.0f);
    if (threadIdx.x == 0) {
      if (loss) loss[n] = 0.0f;
      if (loss64) loss64[n] = 0.0;
    }
    return;
  }
  float tv = -INFINITY, tm = -FLT_MAX;
  if (threadIdx.x < K) {
    int id = t_ids[n * K + threadIdx.x];
    if (id < 0 || id >= V) {
      if (id != -1) atomicExch(err, 100);
      id = -1;
    } else {
      tv = t_vals[n * K + threadIdx.x];
    }
    s_id[threadIdx.x] = id;
    s_z[threadIdx.x] = id >= 0 ? to_f(z[id]) : -INFINITY;
    tm = fmaxf(tm, tv);
  }
  tm = block_max(tm, red);
  float q = threadIdx.x < K && s_id[threadIdx.x] >= 0 ? (tail ? expf(tv) : expf((tv - tm) * inv_t)) : 0.0f;
  float Q = block_sum(q, red);
  if (!tail) {
    q = Q == 0.0f ? 0.0f : q / Q;
    Q = Q == 0.0f ? 0.0f : Q == Q ? 1.0f : Q;   // a NaN among the values stays one
  }
  if (Q == INFINITY) Q = NAN;
  if (threadIdx.x < K) s_q[threadIdx.x] = q;
  __syncthreads();
  // entries naming one token add up; the first of them stands for it
  float qv = 0.0f;
  bool first = threadIdx.x < K && s_id[threadIdx.x] >= 0;
  if (first)
    for (int j = 0; j < K; j++)
      if (s_id[j] == s_id[threadIdx.x]) {
        qv += s_q[j];
        if (j < (int)threadIdx.x) first = false;
      }
  float m = -FLT_MAX;
  for (int v = threadIdx.x; v < V; v += 256) m = fmaxf(m, to_f(z[v]));
  m = block_max(m, red);
  float all = 0.0f, rest = 0.0f, mr = m;
  for (int v = threadIdx.x; v < V; v += 256) all += expf((to_f(z[v]) - m) * inv_t);
  all = block_sum(all, red);
  float qr = 0.0f;
  if (tail) {                              // the mass of the tokens not named, relative to their largest logit
    qr = 1.0f - Q;
    if (qr < TAIL_MIN) qr = 0.0f;
    mr = -FLT_MAX;
    for (int v = threadIdx.x; v < V; v += 256) {
      bool named = false;
      for (int j = 0; j < K; j++) named |= s_id[j] == v;
      if (!named) mr = fmaxf(mr, to_f(z[v]));
    }
    mr = block_max(mr, red);
    for (int v = threadIdx.x; v < V; v += 256) {
      bool named = false;
      for (int j = 0; j < K; j++) named |= s_id[j] == v;
      if (!named) rest += expf((to_f(z[v]) - mr) * inv_t);
    }
    rest = block_sum(rest, red);
  }
  const float ls = logf(all);
  float term = 0.0f;
  if (first && qv > 0.0f) term = qv * (logf(qv) - ((s_z[threadIdx.x] - m) * inv_t - ls));
  float L = block_sum(term, red);
  if (qr > 0.0f) L += qr * (logf(qr) - (logf(rest) + (mr - m) * inv_t - ls));
  if (all == 0.0f) L = Q + qr > 0.0f ? INFINITY : 0.0f;   // a student that allows no token
  if (all != all || Q != Q) L = NAN;
  L *= w;
  if (threadIdx.x == 0) {
    if (loss) loss[n] = L;
    if (loss64) loss64[n] = (double)L;
  }
  if (!dz) return;
  const float g = w * scale * inv_t, total = Q + qr;
  // e relative to mr: p = e f / all, the tail's share q_r e / rest
  const float f = expf(bounded((mr - m) * inv_t));
  const float coef = all == 0.0f ? 0.0f : total * f / all - (qr > 0.0f && rest > 0.0f ? qr / rest : 0.0f);
  for (int v = threadIdx.x; v < V; v += 256) {
    float d = (to_f(z[v]) - mr) * inv_t;
    bool named = false;
    if (tail && all != 0.0f)
      for (int j = 0; j < K; j++) named |= s_id[j] == v;
    if (!named) dz[v] = from_f<T>(g * coef * expf(d));
  }
  __syncthreads();
  if (first && all != 0.0f) {
    const float p = expf((s_z[threadIdx.x] - m) * inv_t) / all;
    dz[s_id[threadIdx.x]] = from_f<T>(g * (total * p - qv));
  }
}

}  // namespace lg

#define LG_LAUNCH_CHECK() TL_TRY_CUDA(cudaGetLastError())
#define LG_DISPATCH(dtype, CALL)                                  \
  do {                                                            \
    if ((dtype) == TL_F32) { using T = float; CALL; }             \
    else if ((dtype) == TL_BF16) { using T = __nv_bfloat16; CALL; } \
    else { using T = __half; CALL; }                              \
  } while (0)

int k_token_logprobs(DeviceCtx *c, const LogitRows &z, const int *ids, float temperature, float *logp,
                     float *entropy, float *stats, int K, int *top_ids, float *top_logp) {
  TraceScope ts(c, "k_token_logprobs");
  LG_DISPATCH(z.dtype, (lg::token_logprobs_kernel<T><<<z.N, 256, 0, c->stream>>>(
                           static_cast<const T *>(z.p), z.ld, ids, z.V, 1.0f / temperature, logp, entropy, stats, K,
                           top_ids, top_logp, c->err_flag)));
  LG_LAUNCH_CHECK();
  return TL_OK;
}

int k_token_logprobs_bwd(DeviceCtx *c, void *dlogits, long long ldd, const LogitRows &z, const int *ids,
                         float temperature, const float *stats, const float *entropy, const float *dlogp,
                         const float *dentropy) {
  TraceScope ts(c, "k_token_logprobs_bwd");
  LG_DISPATCH(z.dtype, (lg::token_logprobs_bwd_kernel<T><<<z.N, 256, 0, c->stream>>>(
                           static_cast<T *>(dlogits), ldd, static_cast<const T *>(z.p), z.ld, ids, z.V,
                           1.0f / temperature, stats, entropy, dlogp, dentropy, c->err_flag)));
  LG_LAUNCH_CHECK();
  return TL_OK;
}

int k_distill_topk(DeviceCtx *c, const LogitRows &z, const int *t_ids, const float *t_vals, int K,
                   float temperature, int tail, const float *weight, float scale, float *loss, double *loss64,
                   void *dlogits, long long ldd) {
  TraceScope ts(c, "k_distill_topk");
  LG_DISPATCH(z.dtype, (lg::distill_topk_kernel<T><<<z.N, 256, 0, c->stream>>>(
                           static_cast<const T *>(z.p), z.ld, t_ids, t_vals, K, z.V, 1.0f / temperature, tail, weight,
                           scale, loss, loss64, static_cast<T *>(dlogits), ldd, c->err_flag)));
  LG_LAUNCH_CHECK();
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
  if (N < 0 || V < 1 || V > TL_VOCAB_MAX)
    return set_error(TL_EINVAL, "N = %d, V = %d: N >= 0 and 1 <= V <= %d are taken", N, V, TL_VOCAB_MAX);
  if (ld < V || ld > (1LL << 40)) return set_error(TL_EINVAL, "row stride of %s %lld below V = %d", what, ld, V);
  return TL_OK;
}

// A gradient may take its logits' own place (the same rows), nothing between.
int check_in_place(const void *dz, long long ldd, const LogitRows &z) {
  if (dz == z.p && ldd == z.ld) return TL_OK;
  const size_t es = dtype_size(z.dtype);
  const uintptr_t a = reinterpret_cast<uintptr_t>(dz), b = reinterpret_cast<uintptr_t>(z.p);
  const uintptr_t a1 = a + ((size_t)(z.N - 1) * ldd + z.V) * es, b1 = b + ((size_t)(z.N - 1) * z.ld + z.V) * es;
  if (a < b1 && b < a1)
    return set_error(TL_EINVAL, "dlogits overlaps logits without being the same rows");
  return TL_OK;
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
