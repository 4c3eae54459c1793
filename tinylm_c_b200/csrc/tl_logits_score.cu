// tl_logits_score.cu -- log probability of a given token a row, the row's
// entropy and its most likely tokens in one pass over the logits.
//
// The K most likely tokens.  A threshold below the K-th largest logit is found
// without sorting the row.  Of a block's F full warps each takes the j-th
// largest of its 32 lanes' maxima; the threshold is the g-th largest of these,
// g = K / j rounded up: every one of g warps has j elements at or above it.
// j = K / F where that is 8 or more, else 5/4 of it, so that g < F: the least
// of many maxima can be very low.  Of random logits 1.7 to 2.2 K pass where j
// stays below 32; plan_rows says where it does not.  (A cluster's blocks take g
// in proportion to their full warps, and the least of their thresholds.)  The
// elements that pass are collected in shared memory and sorted as 64-bit keys:
// logit, then the lower index.  Where more pass than the memory holds (many
// equal logits, rows in order) the K-th largest is searched, counting over the
// row, and the lowest indices of equal ones taken.
#include <algorithm>
#include <cmath>
#include "tl_logits_dev.cuh"
#include "tl_trace.cuh"

namespace tl {
namespace lg {

constexpr int CAP = 512;             // candidates a cluster's first block holds, and one block's row at most

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
template <typename T>
__device__ __noinline__ void select_exactly(const uint4 *st, int cnt, int first, int V, int K, float thr,
                                            unsigned *s_count, unsigned long long *s_keys) {
  using TM = Team;
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
    if (tid < (int)S) *TM::at(&s_sum[flip][TM::rank()], tid) = sum;
    TM::sync();
    sum = 0;
    for (int i = 0; i < (int)S; i++) sum += s_sum[flip][i];
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

// Keys of a warp in descending order, R a lane (lane l holds places R l ...):
// a bitonic sort of 32 R.
template <int R> __device__ __forceinline__ void sort_keys(unsigned long long (&k)[R]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32 * R; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1)
      if (o >= R) {
        const bool larger = ((lane * R & o) == 0) == ((lane * R & size) == 0);
#pragma unroll
        for (int r = 0; r < R; r++) {
          const unsigned long long u = __shfl_xor_sync(FULL, k[r], o / R);
          k[r] = (u > k[r]) == larger ? u : k[r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; r++)
          if (!(r & o)) {
            const bool down = ((lane * R + r) & size) == 0;
            const unsigned long long x = k[r], y = k[r | o];
            const bool swap = (y > x) == down;
            k[r] = swap ? y : x;
            k[r | o] = swap ? x : y;
          }
      }
}

// A warp's chunks whose largest logit passes, by their index in the piece, and
// then their elements that pass, as many lanes a chunk as it has elements: few
// chunks pass, and a warp that branched at each of them would run the elements'
// code once for nearly every chunk (4096 x 50000 bf16, K = 32: 223 instead of 178
// us).
struct Passing {
  unsigned short *list;                          // LIST of them
  int n = 0;
  __device__ __forceinline__ void add(bool pass, int i) {
    const unsigned m = __ballot_sync(FULL, pass);
    if (m) {
      if (pass) list[n + __popc(m & ((1u << (threadIdx.x & 31)) - 1))] = (unsigned short)i;
      n += __popc(m);
    }
  }
  // push(element, its index in the piece) for the elements at or above (equal)
  // or above thr.
  template <typename T, typename F>
  __device__ __forceinline__ void elements(const T *st, float thr, bool equal, F &&push) {
    constexpr int EV = Elem<T>::EV;
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int b = 0; b < n; b += 32 / EV) {
      const int q = b + lane / EV;
      if (q < n) {
        const int v = list[q] * EV + lane % EV;
        const float f = Elem<T>::to_f(st[v]);
        if ((f > thr || (equal && f == thr)) && f > -INFINITY) push(f, v);
      }
    }
    __syncwarp();
    n = 0;
  }
};
constexpr int LIST = 160;                        // of a warp: four chunks a lane on top of a flush limit

struct ScoreArgs {
  Layout l;
  const int *ids;
  float c, inv_t;                    // log2(e) / temperature, 1 / temperature
  float *logp, *entropy, *stats;
  int K, j, g_full, updates, cap;    // alternatives; see threshold() for the others
  int *top_ids;
  float *top_logp;
  int *err;
};

// Few rows, each split over the blocks of a cluster, a piece a block.
template <typename T, int TH, bool ENT>
__global__ void __launch_bounds__(TH, min_blocks(TH)) score_cluster_kernel(const ScoreArgs a) {
  using TM = Team;
  constexpr int EV = Elem<T>::EV, W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  __shared__ Part s_part[2][W], s_from[2][MAX_CLUSTER];
  __shared__ unsigned s_count[2];
  __shared__ unsigned short s_list[W][LIST];
  __shared__ uint64_t s_full;
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = (int)TM::size(), rank = (int)TM::rank();
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x / S, first_row = (int)blockIdx.x / S;
  unsigned long long *s_keys = reinterpret_cast<unsigned long long *>(s_dyn + (size_t)a.l.chunks * 16);
  const Pipe<T> pipe(s_dyn, a.l, 1, &s_abort, a.err);
  // full warps of this block, in every row: those whose 32 lanes all hold logits
  const int mine = max(0, min(min((a.l.V + EV - 1) / EV - rank * t.per, t.per), TH)) >> 5;
  const int g = a.j ? (a.K * mine + a.j * a.g_full - 1) / (a.j * a.g_full) : 0;
  const bool reports = rank == 0 && tid == 0;    // the thread that writes a row's scalars
  int issued = 0;                                // by thread 0
  if (tid == 0) {
    tc::mbar_init(tc::smem_u32(&s_full), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    issued += pipe.issue(t, first_row, rank, 0, &s_full, true, l2_once());
    s_count[0] = s_count[1] = 0;
  }
  int id_next = reports && a.logp ? a.ids[first_row] : -1;
  TM::sync();
  uint32_t phase = 0;
  for (int n = first_row, flip = 0; n < N; n += stride, flip ^= 1, phase ^= 1) {
    const Piece<T> sh(t, n, rank);
    // the given token's logit, and the next row's token
    int id = id_next;
    float z_id = 0.0f;
    if (reports && a.logp) {
      if (id >= 0 && id < t.V) {
        z_id = Elem<T>::to_f(sh.r.row[id]);
      } else {
        if (id != -1) report_token(a.err);
        id = -1;
      }
      if (n + stride < N) id_next = a.ids[n + stride];
    }
    const int cnt = sh.cnt;
    const uint32_t st = tc::smem_u32(s_dyn);
    pipe.wait(&s_full, phase);
    if (t.ragged) sh.mask_ends(pipe.stage(0), [&](int i) { return i % TH == tid; });
    Running run;
    add_share<T, TH, ENT>(run, st, cnt, a.c);
    const float top = run.top;
    float w = -INFINITY;
    if (a.j && warp < mine) w = a.j == 1 ? warp_max(top) : nth_largest<32>(top, a.j);
    Part p = run.warp<ENT>(a.c);
    p.w = w;
    if (lane == 0) s_part[flip][warp] = p;
    meet<ENT>(s_part[flip], s_from[flip], g, a.c);
    const Part *parts = s_from[flip];
    const int ahead = n + stride;
    if (!a.K && tid == 0 && ahead < N) issued += pipe.issue(t, ahead, rank, 0, &s_full, true, l2_once());
    unsigned found = 0;
    if (a.K) {                       // ---- the alternatives
      float thr = -INFINITY;         // too few maxima: every element passes
      if (a.j) {
        thr = (lane & 15) < S ? parts[lane & 15].w : INFINITY;
#pragma unroll
        for (int o = 8; o; o >>= 1) thr = fminf(thr, __shfl_xor_sync(FULL, thr, o));
      }
      unsigned *count = TM::at(&s_count[flip], 0);
      unsigned long long *keys = TM::at(s_keys, 0);
      Passing pass{s_list[warp]};
      auto flush = [&] {
        pass.elements<T>(reinterpret_cast<const T *>(s_dyn), thr, true, [&](float f, int v) {
          const unsigned at = atomicAdd(count, 1u);
          if (at < CAP) keys[at] = key_of(f, sh.r.first(sh.c0) + v);
        });
      };
      for_chunks<T, TH>(st, cnt, [&](const uint4 &x, int i) {
        const float m = Elem<T>::max_of(x);
        pass.add(m >= thr && m > -INFINITY, i);
        if (pass.n > LIST - 32) flush();
      });
      flush();
      TM::sync();
      found = *count;
      if (found > CAP) {
        const Part all = join_all<false>(parts, S, a.c);
        if (all.s >= 0.0f) {         // a row without a distribution has no alternatives
          select_exactly<T>(pipe.stage(0), cnt, sh.r.first(sh.c0), t.V, a.K, thr, &s_count[flip], s_keys);
          found = *count;
        }
      }
      if (tid == 0 && ahead < N) issued += pipe.issue(t, ahead, rank, 0, &s_full, true, l2_once());
    }
    // ---- results: the first block's first warp, and all its warps where many
    // candidates are left to put in order
    const bool crowd = found > 128;
    if (rank == 0 && (warp == 0 || crowd)) {
      p = join_all<ENT>(parts, S, a.c);
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
          sort_keys<4>(k);
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
  }
  if (tid == 0) pipe.drain(&s_full, 1, issued);
  TM::sync();                // the first block's memory stays until all have read it
}


// ---- rows of one block each, in pieces one after another
//
// TH threads compute; one more warp keeps the pieces coming and one writes the
// results, sorts the alternatives and looks the given tokens up, so that the
// next row is under way meanwhile.  The warps hand over through barriers in
// shared memory (a stage full, a stage free, a row's results there, taken).
//
// Alternatives over several pieces: the threshold is taken from the maxima of
// the row so far after piece 1, and after 2, 4, 8, ... until about 256 elements
// of random logits pass in all.  Every element above the threshold at hand is
// kept; in a piece whose own maxima have moved it, elements equal to it as well
// (elsewhere they cannot be among the K: the K elements at or above it come
// earlier).  A threshold of the whole row then leaves few to put in order.

// The K largest keys of a row in memory (up to cap with them), where more than
// cap elements passed: at least K are at or above thr, or thr = -inf.  By TH
// threads (barrier 1), over the row in L2: one pass counts the elements at or
// above the threshold and those above it.  Few enough are collected (the
// row's last threshold is higher than those that filled the list); fewer than
// K above it, as with a mask of a type's lowest value, leave equal logits to be
// taken in order of their index; else the K-th largest value is searched, two
// bits a pass.
template <typename T, int TH>
__device__ __noinline__ void select_row(const T *row, int V, int K, float thr, uint2 *keys, unsigned *s_count, int cap) {
  constexpr int EV = Elem<T>::EV, W = TH / 32;
  __shared__ int s_cnt[2][3][W];
  const Chunks<T> r(row, V);
  const int tid = threadIdx.x, lane = tid & 31;
  int flip = 0;
  auto chunk = [&](int c) {
    if (c >= r.full0 && c < r.full1) return __ldcg(r.base + c);
    return c < r.n ? r.load_edge(c) : make_uint4(Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL);
  };
  auto total = [&](const int (&k)[3], int (&sum)[3]) {
    bar_sync<TH>();
#pragma unroll
    for (int q = 0; q < 3; q++) {
      const int w = __reduce_add_sync(FULL, k[q]);
      if (lane == 0) s_cnt[flip][q][tid >> 5] = w;
    }
    bar_sync<TH>();
#pragma unroll
    for (int q = 0; q < 3; q++) {
      sum[q] = 0;
      for (int i = 0; i < W; i++) sum[q] += s_cnt[flip][q][i];
    }
    flip ^= 1;
  };
  // elements of order u[q] or above
  auto at_least = [&](unsigned u0, unsigned u1, unsigned u2, int (&sum)[3]) {
    int k[3] = {};
#pragma unroll 1
    for (int c = tid; c < r.n; c += 4 * TH) {
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = chunk(c + i * TH);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float f[EV];
        Elem<T>::unpack(x[i], f);
#pragma unroll
        for (int e = 0; e < EV; e++) {
          const unsigned o = f[e] > -INFINITY ? order_of(f[e]) : 0;
          k[0] += o >= u0;
          k[1] += o >= u1;
          k[2] += o >= u2;
        }
      }
    }
    total(k, sum);
  };
  // invariant: at least K of order lo or above; `above` < K of order hi or above
  unsigned lo = order_of(thr == -INFINITY ? -FLT_MAX : thr), hi = order_of(INFINITY);
  int sum[3], above = 0;
  at_least(lo, lo + 1, hi, sum);
  const bool few = sum[0] <= cap;
  if (few) {
    hi = lo;                         // all of order lo or above are collected
    above = sum[0];
  } else if (sum[1] < K) {
    hi = lo + 1;
    above = sum[1];
  }
  while (!few && hi - lo > 1) {
    const unsigned d = max((hi - lo) >> 2, 1u), u0 = lo + d, u1 = min(u0 + d, hi), u2 = min(u1 + d, hi);
    at_least(u0, u1, u2, sum);
    if (u2 < hi && sum[2] >= K) {
      lo = u2;
    } else {
      if (u2 < hi) { hi = u2; above = sum[2]; }
      if (u1 < hi && sum[1] >= K) {
        lo = u1;
      } else {
        if (u1 < hi) { hi = u1; above = sum[1]; }
        if (sum[0] >= K) lo = u0;
        else { hi = u0; above = sum[0]; }
      }
    }
  }
  if (tid == 0) *s_count = 0;
  bar_sync<TH>();
#pragma unroll 1
  for (int c = tid; above && c < r.n; c += TH) {
    float f[EV];
    Elem<T>::unpack(chunk(c), f);
#pragma unroll
    for (int e = 0; e < EV; e++)
      if (f[e] > -INFINITY && order_of(f[e]) >= hi) {
        const unsigned at = atomicAdd(s_count, 1u);            // below `above`, as long as nobody writes to the row meanwhile
        if (at < (unsigned)cap) keys[at] = make_uint2(__float_as_uint(f[e]), (unsigned)(r.first(c) + e));
      }
  }
  int have = above;
  for (int c0 = 0; have < K && c0 < r.n; c0 += TH) {
    float f[EV];
    Elem<T>::unpack(chunk(c0 + tid), f);
    int k = 0;
#pragma unroll
    for (int e = 0; e < EV; e++) k += f[e] > -INFINITY && order_of(f[e]) == lo;
    int before = k;                  // of the warp's lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(FULL, before, o);
      if (lane >= o) before += u;
    }
    const int mark = flip, mine[3] = {k, 0, 0};
    total(mine, sum);
    int at = have + before - k;
    for (int i = 0; i < tid >> 5; i++) at += s_cnt[mark][0][i];
#pragma unroll
    for (int e = 0; e < EV; e++)
      if (f[e] > -INFINITY && order_of(f[e]) == lo && at < K)
        keys[at++] = make_uint2(__float_as_uint(f[e]), (unsigned)(r.first(c0 + tid) + e));
    have += sum[0];
  }
  bar_sync<TH>();
  if (tid == 0) *s_count = few ? min(above, cap) : K;
  bar_sync<TH>();
}

// Without alternatives 56 registers a thread: six blocks of 192 an SM instead of
// five (16384 x 2048 bf16 21.9 against 24.8 us, 2047 x 50001 fp16 44.6 against
// 46.2).
template <typename T, int TH, bool ENT, bool TOP>
__global__ void __launch_bounds__(TH + 64, TOP ? min_blocks(TH + 64) : 65536 / (56 * (TH + 64))) score_kernel(const ScoreArgs a) {
  constexpr int W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  // two of each, for rows in turn
  __shared__ Part s_part[2][W];
  __shared__ float s_thr[2], s_w[2][W];
  __shared__ unsigned short s_list[TOP ? W : 1][LIST];
  __shared__ unsigned s_count[3];    // the last of nobody
  __shared__ uint64_t s_full[MAX_STAGES], s_free[MAX_STAGES], s_done[2], s_taken[2];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x, first_row = (int)blockIdx.x, stages = a.l.stages, pieces = a.l.pieces;
  const Pipe<T> pipe(s_dyn, a.l, stages, &s_abort, a.err);
  uint2 *s_keys = reinterpret_cast<uint2 *>(s_dyn + (size_t)stages * a.l.chunks * 16);     // [2][a.cap]
  if (tid == 0) {
    for (int i = 0; i < stages; i++) {
      tc::mbar_init(tc::smem_u32(&s_full[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_free[i]), W);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(tc::smem_u32(&s_done[i]), W);
      tc::mbar_init(tc::smem_u32(&s_taken[i]), 1);
      s_count[i] = 0;
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == W) {                   // ---- the pieces
    Turn put;
    int k = 0;
    for (int n = first_row; n < N; n += stride)
      for (int i = 0; i < pieces; i++, k++) {
        if (k >= stages && !pipe.wait_all(&s_free[put.s], put.phase ^ 1)) goto out;
        const bool ok = lane != 0 || pipe.issue(t, n, i, put.s, &s_full[put.s], true, l2_once());
        if (!__all_sync(FULL, ok)) goto out;
        put.next(stages);
      }
  out:
    if (lane == 0) pipe.drain(s_full, stages, k);
    return;
  }
  if (warp == W + 1) {               // ---- the results
    int id = a.logp && lane == 0 ? a.ids[first_row] : -1;
    uint32_t phase = 0;
    for (int n = first_row, flip = 0; n < N; n += stride) {
      float z_id = 0.0f;
      const int given = id;
      if (lane == 0 && a.logp) {
        if (id >= 0 && id < t.V) z_id = Elem<T>::to_f(t.z[(size_t)n * t.ld + id]);
        else if (id != -1) report_token(a.err);
        if (n + stride < N) id = a.ids[n + stride];
      }
      if (!pipe.wait_all(&s_done[flip], phase)) return;
      const Part p = join_all<ENT>(s_part[flip], W, a.c);
      const float ls = logf(p.s);    // -inf where nothing is left, NaN for a row without a distribution
      const bool bad = !(p.s >= 0.0f);
      if (lane == 0) {
        if (a.logp)
          a.logp[n] = given < 0 || given >= t.V ? 0.0f : p.s == 0.0f ? -INFINITY : (z_id - p.m) * a.inv_t - ls;
        if (ENT) {
          const float h = ls - p.t / p.s * LN2;
          a.entropy[n] = p.s == 0.0f || h < 0.0f ? 0.0f : h;
        }
        if (a.stats) {
          a.stats[2 * (size_t)n] = p.m;
          a.stats[2 * (size_t)n + 1] = p.s == 0.0f ? INFINITY : ls;
        }
      }
      if (TOP) {
        const int found = bad ? 0 : min((int)__shfl_sync(FULL, s_count[flip], 0), a.cap);
        const float thr = s_thr[flip];
        uint2 *keys = s_keys + flip * a.cap;
        int *to_id = a.top_ids + (size_t)n * a.K;
        float *to_lp = a.top_logp + (size_t)n * a.K;
        int got = 0;                 // the candidates at or above the last threshold, to the front
        for (int i = 0; i < found; i += 32) {
          const uint2 e = i + lane < found ? keys[i + lane] : make_uint2(0xFF800000u, 0);
          const unsigned m = __ballot_sync(FULL, __uint_as_float(e.x) >= thr && i + lane < found);
          __syncwarp();
          if (m >> lane & 1) keys[got + __popc(m & ((1u << lane) - 1))] = e;
          got += __popc(m);
        }
        __syncwarp();
        auto key = [&](int i) -> unsigned long long {
          if (i >= got) return 0;
          const uint2 e = keys[i];
          return key_of(__uint_as_float(e.x), (int)e.y);
        };
        auto put = [&](int place, unsigned long long k) {
          if (place >= a.K || !k) return;
          to_id[place] = (int)(0xFFFFFFFFu - (unsigned)k);
          to_lp[place] = (value_of(k) - p.m) * a.inv_t - ls;
        };
        auto in_order = [&](auto &k) {
          constexpr int R = sizeof(k) / sizeof(k[0]);
#pragma unroll
          for (int r = 0; r < R; r++) k[r] = key(lane + 32 * r);
          sort_keys<R>(k);
#pragma unroll
          for (int r = 0; r < R; r++) put(lane * R + r, k[r]);
        };
        if (got <= 16) {
          const unsigned long long k = key(lane);
          int place = 0;
          for (int q = 0; q < got; q++) place += __shfl_sync(FULL, k, q) > k;
          put(place, k);
        } else if (got <= 32) {
          unsigned long long k[1];
          in_order(k);
        } else if (got <= 128) {
          unsigned long long k[4];
          in_order(k);
        } else if (got <= 256) {
          unsigned long long k[8];
          in_order(k);
        } else {
          unsigned long long k[16];
          in_order(k);
        }
        for (int i = got + lane; i < a.K; i += 32) {
          to_id[i] = -1;
          to_lp[i] = bad ? NAN : -INFINITY;
        }
        __syncwarp();
        if (lane == 0) s_count[flip] = 0;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_taken[flip]));
      flip ^= 1;
      if (!flip) phase ^= 1;
    }
    return;
  }
  // ---- the computing warps
  Turn turn;
  int count_rows = 0, w_flip = 0;
  for (int n = first_row; n < N; n += stride, count_rows++) {
    const int flip = count_rows & 1;
    // this row's places in shared memory: the results' warp has taken the row before last from them
    const bool mine = count_rows < 2 || pipe.wait_all(&s_taken[flip], ((count_rows >> 1) - 1) & 1);
    bool ok = mine;                  // of each lane
    const int slot = mine ? flip : 2;              // else the row's places may still be another's
    const unsigned cap = mine ? a.cap : 0;
    const Chunks<T> r = t.row(n);
    uint2 *keys = s_keys + flip * a.cap;
    Running run;
    float thr = TOP && a.j ? INFINITY : -INFINITY;
    Passing pass{s_list[TOP ? warp : 0]};
    // A value that at least K logits of the row so far are at or above, from
    // the warps whose lanes all had logits in the first piece.
    auto threshold = [&] {
      float w = -INFINITY;
      if (warp < a.g_full) w = a.j == 1 ? warp_max(run.top) : nth_largest<32>(run.top, a.j);
      if (W > 1) {
        if (lane == 0) s_w[w_flip][warp] = w;
        bar_sync<TH>();
        w = nth_largest<W>(s_w[w_flip][lane & (W - 1)], (a.K + a.j - 1) / a.j);
        w_flip ^= 1;
      }
      return w;
    };
    for (int i = 0; i < pieces; i++) {
      const int c0 = i * t.per, cnt = max(0, min(r.n - c0, t.per));
      const uint32_t st = tc::smem_u32(pipe.stage(turn.s));
      bool equal = false;
      auto flush = [&] {
        pass.elements<T>(reinterpret_cast<const T *>(pipe.stage(turn.s)), thr, equal, [&](float f, int v) {
          const unsigned at = atomicAdd(&s_count[slot], 1u);
          if (at < cap) keys[at] = make_uint2(__float_as_uint(f), (unsigned)(r.first(c0) + v));
        });
      };
      ok &= pipe.wait(&s_full[turn.s], turn.phase);
      if (t.ragged) Piece<T>(t, n, i).mask_ends(pipe.stage(turn.s), [&](int k) { return k % TH == tid; });
      if (!TOP) {
        add_share<T, TH, ENT>(run, st, cnt, a.c);
      } else if (a.j && (i & (i + 1)) == 0 && i + 1 < 2 * a.updates) {
        add_share<T, TH, ENT>(run, st, cnt, a.c);
        thr = threshold();
        equal = true;
        for_chunks<T, TH>(st, cnt, [&](const uint4 (&x)[4], int k) {
          float m[4];
#pragma unroll
          for (int q = 0; q < 4; q++) m[q] = Elem<T>::max_of(x[q]);
          const float b = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
          if (__any_sync(FULL, b >= thr && b > -INFINITY)) {
#pragma unroll
            for (int q = 0; q < 4; q++) pass.add(m[q] >= thr && m[q] > -INFINITY, k + q * TH);
            if (pass.n > LIST - 4 * 32) flush();
          }
        }, [&](const uint4 (&x)[1], int k) {
          const float m = Elem<T>::max_of(x[0]);
          pass.add(m >= thr && m > -INFINITY, k);
          if (pass.n > LIST - 4 * 32) flush();
        });
      } else {
        for_chunks<T, TH>(st, cnt, [&](const uint4 (&x)[4], int k) {
          const float m = run.add<T, ENT>(x, a.c);
          if (__any_sync(FULL, m > thr)) {
#pragma unroll
            for (int q = 0; q < 4; q++) pass.add(Elem<T>::max_of(x[q]) > thr, k + q * TH);
            if (pass.n > LIST - 4 * 32) flush();
          }
        }, [&](const uint4 (&x)[1], int k) {
          pass.add(run.add<T, ENT>(x, a.c) > thr, k);
          if (pass.n > LIST - 4 * 32) flush();
        });
        run.fold<ENT>();
      }
      if (TOP) flush();
      __syncwarp();
      if (lane == 0 && ok) tc::mbar_arrive(tc::smem_u32(&s_free[turn.s]));
      turn.next(stages);
    }
    if (!TOP && !__all_sync(FULL, ok)) return;   // no barrier is left that the others wait at
    Part p = run.warp<ENT>(a.c);
    if (lane == 0 && mine) s_part[flip][warp] = p;
    if (TOP) {
      if (a.j && pieces > 1) thr = fmaxf(thr, threshold());
      if (tid == 0 && mine) s_thr[flip] = thr;
      if (bar_any<TH>(!ok)) return;  // else the results' warp leaves s_count alone until this row is done
      if (s_count[flip] > (unsigned)a.cap) {
        p = join_all<false>(s_part[flip], W, a.c);
        if (p.s >= 0.0f)             // a row without a distribution has no alternatives
          select_row<T, TH>(r.row, t.V, a.K, thr, keys, &s_count[flip], a.cap);
      }
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_done[flip]));
  }
}

}  // namespace lg

namespace {

template <typename T, int TH, bool ENT> int launch_cluster(DeviceCtx *c, const RowPlan &pl, lg::ScoreArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::score_cluster_kernel<T, TH, ENT>, c, pl, 0, a.K ? lg::CAP * 8 : 0,
                     &seen[c->device], &a);
}
template <typename T, int TH, bool ENT, bool TOP> int launch_score(DeviceCtx *c, const RowPlan &pl, lg::ScoreArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::score_kernel<T, TH, ENT, TOP>, c, pl, 64, TOP ? 2 * a.cap * 8 : 0,
                     &seen[c->device], &a);
}
template <typename T, bool ENT, bool TOP> int score_rows(DeviceCtx *c, const RowPlan &pl, const lg::ScoreArgs &a) {
  if (pl.threads == 32) return launch_score<T, 32, ENT, TOP>(c, pl, a);
  if constexpr (TOP)                 // 256 threads take more than 64 alternatives
    if (pl.threads == 256) return launch_score<T, 256, ENT, TOP>(c, pl, a);
  return launch_score<T, 128, ENT, TOP>(c, pl, a);
}
template <typename T, bool ENT> int score_typed(DeviceCtx *c, const RowPlan &pl, const lg::ScoreArgs &a) {
  if (pl.blocks > 1) {
    if (pl.threads == 128) return launch_cluster<T, 128, ENT>(c, pl, a);
    return pl.threads == 256 ? launch_cluster<T, 256, ENT>(c, pl, a) : launch_cluster<T, 512, ENT>(c, pl, a);
  }
  return a.K ? score_rows<T, ENT, true>(c, pl, a) : score_rows<T, ENT, false>(c, pl, a);
}

// What the threshold goes by: the full warps F (g_full) of the row, or of its
// first piece, and the j of "the j-th largest of a warp's 32 maxima", 0 where
// 32 F maxima are fewer than K; `updates` pieces at most go by before the last
// threshold that elements are kept by.
void threshold(const RowPlan &pl, int ev, lg::ScoreArgs *a) {
  const int nch = (a->l.V + ev - 1) / ev;        // chunks that every row has, whatever its alignment
  int full = 0;
  for (int i = 0; i < pl.blocks; i++)
    full += std::max(0, std::min(std::min(nch - i * a->l.per, a->l.per), pl.threads)) / 32;
  a->g_full = full;
  // of random logits 2 to 2.5 K of a threshold's part of the row pass, as many
  // again of each further part of that length: kept below 256
  a->cap = a->K <= 64 ? 320 : lg::CAP;
  a->updates = std::max(1, (a->K * a->l.pieces + 99) / 100);
  a->j = 0;
  if (!a->K || !full) return;
  a->j = (a->K + full - 1) / full;
  if (a->j < 8) a->j = (5 * a->K + 4 * full - 1) / (4 * full);
  if (a->j > 32) a->j = 0;
}

}  // namespace

int k_token_logprobs(DeviceCtx *c, const LogitRows &z, const int *ids, float temperature, float *logp,
                     float *entropy, float *stats, int K, int *top_ids, float *top_logp) {
  TraceScope ts(c, "k_token_logprobs");
  const RowPlan pl = plan_rows(c, z, K, false);
  lg::ScoreArgs a{pl.l, ids, lg::LOG2E / temperature, 1.0f / temperature, logp, entropy, stats, K, 0, 0, 0, 0, top_ids,
                  top_logp, c->err_flag};
  threshold(pl, z.dtype == TL_F32 ? 4 : 8, &a);
  if (z.dtype == TL_F32) return entropy ? score_typed<float, true>(c, pl, a) : score_typed<float, false>(c, pl, a);
  if (z.dtype == TL_BF16)
    return entropy ? score_typed<__nv_bfloat16, true>(c, pl, a) : score_typed<__nv_bfloat16, false>(c, pl, a);
  return entropy ? score_typed<__half, true>(c, pl, a) : score_typed<__half, false>(c, pl, a);
}

}  // namespace tl
