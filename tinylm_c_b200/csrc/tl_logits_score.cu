// tl_logits_score.cu -- log probability of a given token a row, the row's
// entropy and its most likely tokens in one pass over the logits.
//
// The K most likely tokens.  A threshold below the K-th largest logit is found
// without sorting the row.  Of the row's F full warps each takes the j-th
// largest of its 32 lanes' maxima, j about 5/4 K / F; each block takes the
// g-th largest of its F_b full warps' values, g = K F_b / (j F) rounded up;
// the threshold is the least of the blocks'.  Every one of the g warps has j
// elements at or above it, so the row has at least j sum g >= K.  Of random
// logits 1.5 to 2 K pass (5/4: with j = 1 and all warps counted it is up to
// 4.5 K, the least of many maxima being low).  They are collected in the first
// block's shared memory as 64-bit keys (logit, then the lower index), and each
// one's place is the number of larger keys.  Where more pass than the memory
// holds (many equal logits, rows in order) the K-th largest key is found by
// bisection, counting over the share, and exactly K are collected.
#include <algorithm>
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

// The K largest keys of the row into the first block's memory, by bisection:
// at least K logits are at or above thr, or thr = -inf.  `first` is the share's
// first element.  Every thread of the row's blocks calls it.  2 to 50 counting
// passes over shared memory, of about a microsecond each.
template <typename T, bool CL>
__device__ __noinline__ void select_exactly(const uint4 *st, int cnt, int first, int V, int K, float thr,
                                            unsigned *s_count, unsigned long long *s_keys) {
  using TM = Team<CL>;
  constexpr int EV = Elem<T>::EV;
  __shared__ int s_cnt[2][MAX_WARPS], s_sum[2][MAX_CLUSTER];
  const int tid = threadIdx.x, TH = blockDim.x, W = TH >> 5;
  const unsigned S = TM::size();
  int flip = 0;
  // elements of an order above u, and those of order u and an index below b
  auto count = [&](unsigned u, int b) {
    int k = 0;
#pragma unroll 1
    for (int i = tid; i < cnt; i += TH) {
      float f[EV];
      Elem<T>::unpack(st[i], f);
      const int v = first + i * EV;
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
  for (int i = tid; i < cnt; i += TH) {
    float f[EV];
    Elem<T>::unpack(st[i], f);
    const int v = first + i * EV;
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

// Keys in descending order, four a lane (lane l holds places 4l .. 4l + 3): a
// bitonic sort of 128 in one warp.
__device__ __forceinline__ void sort_128(unsigned long long (&k)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 128; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1)
      if (o >= 4) {
        const bool larger = ((lane * 4 & o) == 0) == ((lane * 4 & size) == 0);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const unsigned long long u = __shfl_xor_sync(FULL, k[r], o >> 2);
          k[r] = (u > k[r]) == larger ? u : k[r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (!(r & o)) {
            const bool down = ((lane * 4 + r) & size) == 0;
            const unsigned long long x = k[r], y = k[r | o];
            const bool swap = (y > x) == down;
            k[r] = swap ? y : x;
            k[r | o] = swap ? x : y;
          }
      }
}

struct ScoreArgs {
  Layout l;
  const int *ids;
  float c, inv_t;                    // log2(e) / temperature, 1 / temperature
  float *logp, *entropy, *stats;
  int K, j, g_full;                  // alternatives; see threshold() for j and g_full
  int *top_ids;
  float *top_logp;
  int *err;
};

template <typename T, bool CL, bool ENT>
__global__ void __launch_bounds__(MAX_THREADS, 2) score_kernel(const ScoreArgs a) {
  using TM = Team<CL>;
  constexpr int EV = Elem<T>::EV;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  __shared__ Part s_part[2][MAX_WARPS], s_from[2][MAX_CLUSTER];
  __shared__ unsigned s_count[2];
  __shared__ uint64_t s_full[MAX_STAGES];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, TH = blockDim.x, W = TH >> 5;
  const int S = (int)TM::size(), rank = (int)TM::rank();
  const Rows<T> t(a.l, rank);
  const int N = a.l.N, stride = (int)gridDim.x / S, first_row = (int)blockIdx.x / S;
  unsigned long long *s_keys = reinterpret_cast<unsigned long long *>(s_dyn + (size_t)a.l.stages * a.l.chunks * 16);
  Pipe<T> pipe{reinterpret_cast<uint4 *>(s_dyn), a.l.stages, a.l.chunks, s_full, &s_abort, a.err};
  // full warps of this block, in every row: those whose 32 lanes all hold logits
  const int mine = max(0, min(min((a.l.V + EV - 1) / EV - t.c0, t.per), TH)) >> 5;
  const int g = a.j ? (a.K * mine + a.j * a.g_full - 1) / (a.j * a.g_full) : 0;
  const bool reports = rank == 0 && tid == 0;    // the thread that writes a row's scalars
  if (tid == 0) {
    pipe.init();
    for (int i = 0; i < a.l.stages; i++)
      if (first_row + i * stride < N) pipe.issue(t, first_row + i * stride, i, true);
    s_count[0] = s_count[1] = 0;
  }
  int id_next = reports && a.logp ? a.ids[first_row] : -1;
  TM::sync();
  for (int n = first_row, flip = 0; n < N; n += stride, flip ^= 1) {
    const Share<T> sh(t, n);
    // the given token's logit, and the next row's token
    int id = id_next;
    float z_id = 0.0f;
    if (reports && a.logp) {
      if (id >= 0 && id < t.V) {
        z_id = Elem<T>::to_f(sh.r.row[id]);
      } else {
        if (id != -1) atomicExch(a.err, ERR_TOKEN);
        id = -1;
      }
      if (n + stride < N) id_next = a.ids[n + stride];
    }
    const int cnt = sh.cnt;
    const uint4 *st = pipe.stage();
    pipe.wait(t, sh);
    const float top = thread_max<T>(st, cnt);
    float w = -INFINITY;
    if (a.j && warp < mine) w = a.j == 1 ? warp_max(top) : nth_largest<32>(top, a.j);
    Part p = warp_part<T, ENT>(st, cnt, top, a.c);
    p.w = w;
    if (lane == 0) s_part[flip][warp] = p;
    if (CL) meet<ENT>(s_part[flip], s_from[flip], g, a.c);
    else __syncthreads();
    const Part *parts = CL ? s_from[flip] : s_part[flip];
    const int ahead = n + a.l.stages * stride;
    if (!a.K && tid == 0 && ahead < N) pipe.issue(t, ahead, pipe.at, true);
    unsigned found = 0;
    if (a.K) {                       // ---- the alternatives
      float thr = -INFINITY;         // too few maxima: every element passes
      if (CL) {
        if (a.j) {
          thr = (lane & 15) < S ? parts[lane & 15].w : INFINITY;
#pragma unroll
          for (int o = 8; o; o >>= 1) thr = fminf(thr, __shfl_xor_sync(FULL, thr, o));
        }
      } else if (a.j) {
        thr = W == 1 ? parts[0].w : nth_largest<16>((lane & 15) < W ? parts[lane & 15].w : -INFINITY, g);
      }
      unsigned *count = TM::at(&s_count[flip], 0);
      unsigned long long *keys = TM::at(s_keys, 0);
      if (top >= thr && top > -INFINITY) {
#pragma unroll 2
        for (int i = tid; i < cnt; i += TH) {
          const uint4 x = st[i];
          if (Elem<T>::max_of(x) >= thr) {
            float f[EV];
            Elem<T>::unpack(x, f);
            const int v = sh.r.first(sh.c0 + i);
#pragma unroll
            for (int e = 0; e < EV; e++)
              if (f[e] >= thr && f[e] > -INFINITY) {
                const unsigned at = atomicAdd(count, 1u);
                if (at < CAP) keys[at] = key_of(f[e], v + e);
              }
          }
        }
      }
      TM::sync();
      found = *count;
      if (found > CAP) {
        const Part all = join_all<false>(parts, CL ? S : W, a.c);
        if (all.s >= 0.0f) {         // a row without a distribution has no alternatives
          select_exactly<T, CL>(st, cnt, sh.r.first(sh.c0), t.V, a.K, thr, &s_count[flip], s_keys);
          found = *count;
        }
      }
      if (tid == 0 && ahead < N) pipe.issue(t, ahead, pipe.at, true);
    }
    // ---- results: the first block's first warp, and all its warps where many
    // candidates are left to put in order
    const bool crowd = found > 128;
    if (rank == 0 && (warp == 0 || crowd)) {
      p = join_all<ENT>(parts, CL ? S : W, a.c);
      const float ls = logf(p.s);    // -inf where nothing is left, NaN for a row without a distribution
      const bool bad = !(p.s >= 0.0f);
      if (tid == 0) {
        s_count[flip ^ 1] = 0;       // its readers have passed a barrier of this row
        if (a.logp) a.logp[n] = id < 0 ? 0.0f : p.s == 0.0f ? -INFINITY : (z_id - p.m) * a.inv_t - ls;
        if (ENT) {
          const float h = ls - p.t / p.s * LN2;
          a.entropy[n] = p.s == 0.0f || h < 0.0f ? 0.0f : h;
        }
        if (a.stats) {
          a.stats[2 * (size_t)n] = p.m;
          a.stats[2 * (size_t)n + 1] = p.s == 0.0f ? INFINITY : ls;
        }
      }
      if (a.K) {
        const int got = bad ? 0 : (int)min(found, (unsigned)CAP);
        int *to_id = a.top_ids + (size_t)n * a.K;
        float *to_lp = a.top_logp + (size_t)n * a.K;
        auto put = [&](int place, unsigned long long k) {
          if (place >= a.K) return;
          to_id[place] = (int)(0xFFFFFFFFu - (unsigned)k);
          to_lp[place] = (value_of(k) - p.m) * a.inv_t - ls;
        };
        if (crowd || got <= 24) {
          for (int i = tid; i < got; i += crowd ? TH : 32) {
            const unsigned long long k = s_keys[i];
            int place = 0;
            for (int q = 0; q < got; q++) place += s_keys[q] > k;
            put(place, k);
          }
        } else {
          unsigned long long k[4];
#pragma unroll
          for (int r = 0; r < 4; r++) k[r] = lane * 4 + r < got ? s_keys[lane * 4 + r] : 0;
          sort_128(k);
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (lane * 4 + r < got) put(lane * 4 + r, k[r]);
        }
        if (warp == 0)
          for (int i = got + lane; i < a.K; i += 32) {
            to_id[i] = -1;
            to_lp[i] = bad ? NAN : -INFINITY;
          }
      }
    }
    pipe.next();
  }
  if (CL) TM::sync();                // the first block's memory stays until all have read it
}

}  // namespace lg

namespace {

template <typename T, bool CL, bool ENT> int launch_score(DeviceCtx *c, const RowPlan &pl, lg::ScoreArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::score_kernel<T, CL, ENT>, c, pl, a.K ? lg::CAP * 8 : 0, &seen[c->device], &a);
}
template <typename T> int score_typed(DeviceCtx *c, const RowPlan &pl, const lg::ScoreArgs &a) {
  if (pl.blocks > 1) return a.entropy ? launch_score<T, true, true>(c, pl, a) : launch_score<T, true, false>(c, pl, a);
  return a.entropy ? launch_score<T, false, true>(c, pl, a) : launch_score<T, false, false>(c, pl, a);
}

// What the threshold goes by: the row's full warps F (g_full) and the j of
// "the j-th largest of a warp's 32 maxima", 0 where 32 F maxima are fewer than K.
void threshold(const RowPlan &pl, int ev, lg::ScoreArgs *a) {
  const int nch = (a->l.V + ev - 1) / ev;        // chunks that every row has, whatever its alignment
  int full = 0;
  for (int i = 0; i < pl.blocks; i++)
    full += std::max(0, std::min(std::min(nch - i * a->l.per, a->l.per), pl.threads)) / 32;
  a->g_full = full;
  a->j = 0;
  if (!a->K || !full) return;
  a->j = (5 * a->K + 4 * full - 1) / (4 * full);
  if (a->j > 32) a->j = (a->K + full - 1) / full;
  if (a->j > 32) a->j = 0;
}

}  // namespace

int k_token_logprobs(DeviceCtx *c, const LogitRows &z, const int *ids, float temperature, float *logp,
                     float *entropy, float *stats, int K, int *top_ids, float *top_logp) {
  TraceScope ts(c, "k_token_logprobs");
  const RowPlan pl = plan_rows(c, z, K);
  lg::ScoreArgs a{pl.l, ids, lg::LOG2E / temperature, 1.0f / temperature, logp, entropy, stats, K, 0, 0, top_ids,
                  top_logp, c->err_flag};
  threshold(pl, z.dtype == TL_F32 ? 4 : 8, &a);
  if (z.dtype == TL_F32) return score_typed<float>(c, pl, a);
  if (z.dtype == TL_BF16) return score_typed<__nv_bfloat16>(c, pl, a);
  return score_typed<__half>(c, pl, a);
}

}  // namespace tl
