// tl_logits_score.cu -- log probability of a given token a row, the row's
// entropy and its most likely tokens in one pass over the logits.
//
// A row's slice is loaded once and stays in registers: its largest logit, the
// sums of e and e d relative to it, and the alternatives all come from there.
//
// The K most likely tokens.  A threshold below the K-th largest logit is found
// without sorting the row: each full warp of the row's F takes the j-th
// largest of its 32 lanes' maxima, j = ceil(K / F), and the threshold is the
// least of these.  Each of the F warps has j elements at or above it, so there
// are K.  About 1.5 K of random logits pass; they are collected in the first
// block's shared memory as 64-bit keys (logit, then the lower index), and each
// one's place is the number of larger keys.  Where more pass than the memory
// holds (many equal logits, sorted rows) the K-th largest key is found by
// bisection, counting over the registers, and exactly K are collected.
#include <cmath>
#include "tl_logits_dev.cuh"
#include "tl_trace.cuh"

namespace tl {
namespace lg {

constexpr int CAP = 512;             // candidates a row's first block holds

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

// The j-th largest of the lanes' values (1 <= j <= 32): a bitonic sort of the
// warp in descending order.
__device__ __forceinline__ float warp_nth_largest(float v, int j) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o; o >>= 1) {
      const float u = __shfl_xor_sync(FULL, v, o);
      v = ((lane & o) == 0) == ((lane & k) == 0) ? fmaxf(v, u) : fminf(v, u);
    }
  return __shfl_sync(FULL, v, j - 1);
}

// The K largest keys of the row into the first block's memory, by bisection:
// the thread's chunks x (the first holding element v0, the next TH chunks
// on), at least K of them at or above thr > -inf or thr = -inf.  Every thread
// of the row's blocks calls it.  Kept out of line, its chunks in local memory:
// it takes 2 to 50 counting passes of about a microsecond, on rows with many
// equal logits or of sorted order.
template <typename T, int TH, bool CL>
__device__ __noinline__ void select_exactly(const uint4 *x, int v0, int V, int K, float thr, unsigned *s_count,
                                            unsigned long long *s_keys) {
  using TM = Team<CL>;
  constexpr int W = TH / 32, EV = Elem<T>::EV;
  __shared__ int s_cnt[2][W], s_sum[2][MAX_CLUSTER];
  const int tid = threadIdx.x;
  const unsigned S = TM::size();
  int flip = 0;
  // elements of an order above u, and those of order u and an index below b
  auto count = [&](unsigned u, int b) {
    int k = 0;
#pragma unroll 1
    for (int i = 0; i < NV; i++) {
      float f[EV];
      Elem<T>::unpack(x[i], f);
      const int v = v0 + i * TH * EV;
#pragma unroll
      for (int e = 0; e < EV; e++) {
        const unsigned o = order_of(f[e]);
        if (f[e] > -INFINITY && (o > u || (o == u && v + e < b))) k++;
      }
    }
    k = __reduce_add_sync(FULL, k);
    if ((tid & 31) == 0) s_cnt[flip][tid >> 5] = k;
    __syncthreads();
    int sum = 0;
    for (int i = 0; i < W; i++) sum += s_cnt[flip][i];
    if constexpr (CL) {
      if (tid < (int)S) *TM::at(&s_sum[flip][TM::rank()], tid) = sum;
      TM::sync();
      sum = 0;
      for (int i = 0; i < (int)S; i++) sum += s_sum[flip][i];
    }
    flip ^= 1;
    return sum;
  };
  // invariant: at least K of order lo or above, fewer of order hi or above.
  // The first probe is the order just above the threshold: a mask of a type's
  // lowest value leaves fewer than K above it.
  unsigned lo = order_of(thr == -INFINITY ? -FLT_MAX : thr), hi = order_of(INFINITY), probe = lo + 1;
  int b = V;
  bool few = false;
  while (hi - lo > 1 && !few) {
    const int k = count(probe, V);
    if (k >= K) lo = probe; else hi = probe;
    few = k >= K && k <= CAP;
    probe = lo + (hi - lo) / 2;
  }
  for (int under = 0; !few && b - under > 1;) {   // equal logits: the lowest indices of them
    const int mid = under + (b - under) / 2;
    if (count(lo, mid) >= K) b = mid; else under = mid;
  }
  if (TM::rank() == 0 && tid == 0) *s_count = 0;  // every thread has read it before the first count
  TM::sync();
  unsigned *to = TM::at(s_count, 0);
  unsigned long long *keys = TM::at(s_keys, 0);
#pragma unroll 1
  for (int i = 0; i < NV; i++) {
    float f[EV];
    Elem<T>::unpack(x[i], f);
    const int v = v0 + i * TH * EV;
#pragma unroll
    for (int e = 0; e < EV; e++) {
      const unsigned o = order_of(f[e]);
      if (f[e] > -INFINITY && (o > lo || (o == lo && v + e < b))) {
        const unsigned at = atomicAdd(to, 1u);
        if (at < CAP) keys[at] = key_of(f[e], v + e);
      }
    }
  }
  TM::sync();
}

struct ScoreArgs {
  const void *z;
  long long ld;
  const int *ids;
  int V;
  float c, inv_t;                    // log2(e) / temperature, 1 / temperature
  float *logp, *entropy, *stats;
  int K;
  int *top_ids;
  float *top_logp;
  int *err;
};

template <typename T, int TH, bool CL, bool ENT>
__global__ void __launch_bounds__(TH, 1024 / TH) score_kernel(const ScoreArgs a) {
  using TM = Team<CL>;
  constexpr int W = TH / 32, EV = Elem<T>::EV;
  __shared__ Part s_part[W], s_from[MAX_CLUSTER];
  __shared__ unsigned s_count;
  __shared__ unsigned long long s_keys[CAP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = TM::rank(), S = TM::size();
  const size_t n = CL ? blockIdx.x / S : blockIdx.x;
  const Chunks<T> r(static_cast<const T *>(a.z) + n * a.ld, a.V);
  const int per = CL ? (r.n + (int)S - 1) / (int)S : r.n;
  const int c0 = (int)rank * per, c1 = min(r.n, c0 + per), cnt = c1 - c0;
  if (tid == 0) s_count = 0;
  TM::arrive();

  uint4 x[NV];
  load_slice<T, TH>(r, c0, c1, x);
  // the given token's logit, read by the thread that reports it
  int id = -1;
  float z_id = 0.0f;
  if (rank == 0 && tid == 0 && a.logp) {
    id = a.ids[n];
    if (id >= 0 && id < a.V) {
      z_id = Elem<T>::to_f(r.row[id]);
    } else {
      if (id != -1) atomicExch(a.err, 100);
      id = -1;
    }
  }
  const float lane_max = lane_max_of<T, TH>(x, cnt);
  float thr = INFINITY;              // a warp that is not full sets none
  if (a.K) {
    int full = 0;                    // full warps of the row
    for (int i = 0; i < (int)S; i++) full += min(max(min(per, r.n - i * per), 0), TH) >> 5;
    const int j = full ? (a.K + full - 1) / full : 33;
    if (j > 32) thr = -INFINITY;     // too few maxima: every element passes
    else if (min(cnt, TH) >= warp * 32 + 32) thr = j == 1 ? warp_max(lane_max) : warp_nth_largest(lane_max, j);
  }
  Part p = warp_part<T, TH, ENT>(x, cnt, lane_max, a.c);
  p.w = thr;
  if (lane == 0) s_part[warp] = p;
  p = join_row<CL, W, ENT>(s_part, s_from, INFINITY, a.c);
  const float ls = logf(p.s);        // -inf where nothing is left, NaN for a row without a distribution
  const bool bad = !(p.s >= 0.0f);
  if (rank == 0 && tid == 0) {
    if (a.logp)
      a.logp[n] = id < 0 ? 0.0f : p.s == 0.0f ? -INFINITY : (z_id - p.m) * a.inv_t - ls;
    if (ENT) {
      const float h = ls - p.t / p.s * LN2;
      a.entropy[n] = p.s == 0.0f || h < 0.0f ? 0.0f : h;
    }
    if (a.stats) {
      a.stats[2 * n] = p.m;
      a.stats[2 * n + 1] = p.s == 0.0f ? INFINITY : ls;
    }
  }
  if (!a.K) return;

  // ---- the alternatives
  thr = p.w;
  unsigned *count = TM::at(&s_count, 0);
  unsigned long long *keys = TM::at(s_keys, 0);
  if (lane_max >= thr && lane_max > -INFINITY) {
#pragma unroll
    for (int i = 0; i < NV; i++)
      if (i * TH < cnt && Elem<T>::max_of(x[i]) >= thr) {
        float f[EV];
        Elem<T>::unpack(x[i], f);
        const int v = r.first(c0 + i * TH + tid);
#pragma unroll
        for (int e = 0; e < EV; e++)
          if (f[e] >= thr && f[e] > -INFINITY) {
            const unsigned at = atomicAdd(count, 1u);
            if (at < CAP) keys[at] = key_of(f[e], v + e);
          }
      }
  }
  TM::sync();
  unsigned found = *count;
  if (found > CAP && !bad) {
    uint4 kept[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) kept[i] = x[i];
    select_exactly<T, TH, CL>(kept, r.first(c0 + tid), a.V, a.K, thr, &s_count, s_keys);
    found = *count;
  }
  if (CL) {                          // the first block's memory has been read by all
    TM::arrive();
    TM::wait();
  }
  if (rank != 0) return;
  const int got = bad ? 0 : (int)min(found, (unsigned)CAP);
  for (int i = tid; i < got; i += TH) {
    const unsigned long long k = s_keys[i];
    int place = 0;
    for (int j = 0; j < got; j++) place += s_keys[j] > k;
    if (place < a.K) {
      a.top_ids[n * a.K + place] = (int)(0xFFFFFFFFu - (unsigned)k);
      a.top_logp[n * a.K + place] = (value_of(k) - p.m) * a.inv_t - ls;
    }
  }
  for (int i = got + tid; i < a.K; i += TH) {
    a.top_ids[n * a.K + i] = -1;
    a.top_logp[n * a.K + i] = bad ? NAN : -INFINITY;
  }
}

}  // namespace lg

namespace {

template <typename T, int TH, bool CL, bool ENT>
int launch_score(DeviceCtx *c, int N, int S, const lg::ScoreArgs &a) {
  if constexpr (!CL) {
    lg::score_kernel<T, TH, false, ENT><<<N, TH, 0, c->stream>>>(a);
    TL_TRY_CUDA(cudaGetLastError());
    return TL_OK;
  } else {
    return launch_rows_cluster((const void *)lg::score_kernel<T, TH, true, ENT>, c, N, TH, S, const_cast<void *>(static_cast<const void *>(&a)));
  }
}
template <typename T, bool ENT> int score_typed(DeviceCtx *c, int N, const RowPlan &pl, const lg::ScoreArgs &a) {
  if (pl.blocks > 1)
    return pl.threads == 256 ? launch_score<T, 256, true, ENT>(c, N, pl.blocks, a)
                             : launch_score<T, 512, true, ENT>(c, N, pl.blocks, a);
  switch (pl.threads) {
    case 32: return launch_score<T, 32, false, ENT>(c, N, 1, a);
    case 128: return launch_score<T, 128, false, ENT>(c, N, 1, a);
    case 256: return launch_score<T, 256, false, ENT>(c, N, 1, a);
    default: return launch_score<T, 512, false, ENT>(c, N, 1, a);
  }
}

}  // namespace

int k_token_logprobs(DeviceCtx *c, const LogitRows &z, const int *ids, float temperature, float *logp,
                     float *entropy, float *stats, int K, int *top_ids, float *top_logp) {
  TraceScope ts(c, "k_token_logprobs");
  const RowPlan pl = plan_rows(c, z, K);
  const lg::ScoreArgs a{z.p, z.ld, ids, z.V, lg::LOG2E / temperature, 1.0f / temperature, logp, entropy, stats, K,
                        top_ids, top_logp, c->err_flag};
  if (z.dtype == TL_F32) return entropy ? score_typed<float, true>(c, z.N, pl, a) : score_typed<float, false>(c, z.N, pl, a);
  if (z.dtype == TL_BF16)
    return entropy ? score_typed<__nv_bfloat16, true>(c, z.N, pl, a) : score_typed<__nv_bfloat16, false>(c, z.N, pl, a);
  return entropy ? score_typed<__half, true>(c, z.N, pl, a) : score_typed<__half, false>(c, z.N, pl, a);
}

}  // namespace tl
