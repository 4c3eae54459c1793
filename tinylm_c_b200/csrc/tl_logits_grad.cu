// tl_logits_grad.cu -- gradients over vocabulary rows: of token log
// probabilities and entropies, and of the divergence from a teacher's K most
// likely tokens with the divergence itself.
#include <cmath>
#include "tl_logits_dev.cuh"
#include "tl_trace.cuh"

namespace tl {
namespace lg {

// The smallest mass that counts as a teacher's tail: below it 1 - sum q is
// the rounding of fp32 log probabilities, not probability.
constexpr float TAIL_MIN = 0x1p-20f;

// ------------------------------------------------- token log probabilities
struct GradArgs {
  void *dz;
  long long ldd;
  const void *z;
  long long ld;
  const int *ids;
  int N, V;
  float c, inv_t;                    // log2(e) / temperature, 1 / temperature
  const float *stats, *entropy, *dlogp, *dentropy;
  int *err;
};

// dz_v = (1/t) [ a (1[v = id] - p_v) - b p_v (log p_v + H) ], element by
// element from the forward pass's statistics: one read, one write.  TPR
// threads take CPT chunks each of one row, 256 / TPR rows a block.  4 chunks of
// fp32 and 8 of 16-bit types: 181 and 91 us at 16384 x 8192 fp32 and 1021 x
// 131072 bf16 (91 and 90 % of the measured copy rate), the other way round 208
// and 96.
template <typename T> constexpr int CPT = Elem<T>::EV;
template <typename T, int TPR, bool ENT>
__global__ void __launch_bounds__(256) token_logprobs_bwd_kernel(const GradArgs a, int segs) {
  constexpr int EV = Elem<T>::EV, CPT = lg::CPT<T>;
  const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int seg = blockIdx.x % segs;
  const long long n = (long long)(blockIdx.x / segs) * (256 / TPR) + sub;
  if (n >= a.N) return;
  const Chunks<T> r(static_cast<const T *>(a.z) + n * a.ld, a.V);
  const Chunks<T> o(static_cast<const T *>(a.dz) + n * a.ldd, a.V);
  const int c0 = seg * (TPR * CPT) + t;
  int id = a.dlogp ? a.ids[n] : -1;
  if (id != -1 && (unsigned)id >= (unsigned)a.V) {
    if (c0 == 0) atomicExch(a.err, ERR_TOKEN);
    id = -1;
  }
  const float m = a.stats[2 * n], ls = a.stats[2 * n + 1];
  const bool empty = ls == INFINITY;               // a row of -inf only
  const float ga = id >= 0 && !empty ? a.dlogp[n] * a.inv_t : 0.0f;
  const float gb = ENT && !empty ? a.dentropy[n] * a.inv_t : 0.0f;
  const bool unread = ga == 0.0f && gb == 0.0f;
  const float H = ENT && gb != 0.0f ? a.entropy[n] : 0.0f;
  uint4 x[CPT];
#pragma unroll
  for (int i = 0; i < CPT; i++) {
    const int c = c0 + i * TPR;
    if (!unread && c >= r.full0 && c < r.full1) x[i] = __ldcg(r.base + c);
    else if (!unread && c < r.n) x[i] = r.load_edge(c);
  }
  // log2 p = (z - m) c - ls log2(e); the factor of p: -(a + b (log p + H))
  const float nl = -ls * LOG2E, fb = -gb * LN2, fa = -fmaf(gb, H, ga);
  const f32x2 nm2 = pack2(-m, -m), c2 = pack2(a.c, a.c), nl2 = pack2(nl, nl), fb2 = pack2(fb, fb), fa2 = pack2(fa, fa);
#pragma unroll
  for (int i = 0; i < CPT; i++) {
    const int c = c0 + i * TPR;
    if (c >= r.n) break;
    float f[EV];
    Elem<T>::unpack(x[i], f);
    const int v = r.first(c);
#pragma unroll
    for (int e = 0; e < EV; e += 2) {
      const f32x2 l2 = fma2(add2(pack2(f[e], f[e + 1]), nm2), c2, nl2);
      float l0, l1;
      unpack2(l2, l0, l1);
      const f32x2 p2 = pack2(exp2_fast(l0), exp2_fast(l1));
      const f32x2 k2 = ENT ? fma2(pack2(bounded(l0), bounded(l1)), fb2, fa2) : fa2;
      unpack2(mul2(p2, k2), f[e], f[e + 1]);
    }
    if ((unsigned)(id - v) < (unsigned)EV && id >= 0) {
#pragma unroll
      for (int e = 0; e < EV; e++)
        if (v + e == id) f[e] += ga;
    }
    if (unread) {
#pragma unroll
      for (int e = 0; e < EV; e++) f[e] = 0.0f;
    }
    if (o.mis == r.mis && c >= r.full0 && c < r.full1) {
      o.base[c] = Elem<T>::pack(f);
    } else {                         // past an end, or rows of another alignment: the chunk's elements one by one
#pragma unroll
      for (int e = 0; e < EV; e++)
        if (v + e >= 0 && v + e < a.V) o.row[v + e] = Elem<T>::from_f(f[e]);
    }
  }
}

// ------------------------------------------------------------ distillation
struct DistillArgs {
  Layout l;
  const int *t_ids;
  const float *t_vals;
  int K;
  float c, inv_t;                    // log2(e) / temperature, 1 / temperature
  double per_t;                      // 1 / temperature
  const float *weight;
  float scale;
  float *loss;
  double *loss64;
  void *dz;
  long long ldd;
  int *err;
};

// L = sum_v q_v (log q_v - log p_v) over the named tokens, with the tail
// + q_r (log q_r - log p_r), p_r = sum of p over the others; Q = sum q + q_r.
//   named v:  dL/dy_v = Q p_v - q_v
//   others:   dL/dy_v = p_v (Q - q_r / p_r)
// With a tail the named tokens are taken out of the row (set to -inf in shared
// memory) before its statistics, so that p_r is summed and never 1 - sum p,
// which loses all its digits for a confident student.  All others' gradients
// are then one factor times e_v; the named tokens' are written over them at
// the end.
//
// A row's entries in shared memory, K of each: the token (-1: padding), its q
// and logit, and the mass of the token an entry stands for (-1 if it stands
// for none: entries naming one token add up, the first of them stands for it).
struct Entries {
  int *id;
  float *q, *z, *qv;
  __device__ __forceinline__ Entries(void *p, int K, int flip)
      : id(static_cast<int *>(p) + flip * 4 * K), q(static_cast<float *>(p) + (flip * 4 + 1) * K), z(q + K), qv(z + K) {}
};
constexpr int KL = TL_TOPK_MAX / 32;             // entries a lane

// Row n's entries as one warp loads them.
struct Loaded {
  int id[KL];
  float t[KL];
  __device__ __forceinline__ void load(const DistillArgs &a, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < KL; k++) {
      const int j = k * 32 + lane;
      id[k] = -1;
      t[k] = -INFINITY;
      if (j < a.K) {
        id[k] = a.t_ids[(size_t)n * a.K + j];
        t[k] = a.t_vals[(size_t)n * a.K + j];
      }
    }
  }
};
// The teacher's distribution from a row's loaded entries, by one warp: the
// entries in shared memory, sum[0] the sum of q, sum[1] the tail.
template <typename T, bool TAIL>
__device__ __forceinline__ void teach(const DistillArgs &a, const Chunks<T> &r, Loaded &l, const Entries &to, float *sum) {
  const int lane = threadIdx.x & 31;
  float z[KL], tm = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < KL; k++) {
    if ((unsigned)l.id[k] >= (unsigned)a.l.V) {
      if (l.id[k] != -1) atomicExch(a.err, ERR_TOKEN);
      l.id[k] = -1;
      l.t[k] = -INFINITY;
    }
    z[k] = l.id[k] >= 0 ? Elem<T>::to_f(r.row[l.id[k]]) : -INFINITY;
    tm = fmaxf(tm, l.t[k]);
  }
  if (!TAIL) tm = warp_max(tm);
  float q[KL];
  double mass = 0.0;                             // 1 - sum q keeps what fp32 entries say of it
#pragma unroll
  for (int k = 0; k < KL; k++) {
    q[k] = l.id[k] < 0 ? 0.0f : expf(TAIL ? l.t[k] : (l.t[k] - tm) * a.inv_t);
    mass += (double)q[k];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(FULL, mass, o);
  const float all = (float)mass;
  const float inv = TAIL ? 1.0f : all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
  for (int k = 0; k < KL; k++) {
    const int j = k * 32 + lane;
    if (j < a.K) {
      to.id[j] = l.id[k];
      to.q[j] = to.qv[j] = q[k] * inv;
      to.z[j] = z[k];
    }
  }
  if (lane == 0) {
    float Q = TAIL || all == 0.0f ? all : 1.0f;
    if (!(all < INFINITY)) Q = NAN;              // a NaN or +inf among the values
    const float qr = TAIL ? (Q == Q ? (float)(1.0 - mass) : Q) : 0.0f;
    sum[0] = Q;
    sum[1] = qr < TAIL_MIN ? 0.0f : qr;          // NaN stays
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < KL; k++) {
    const int j = k * 32 + lane;
    if (k * 32 < a.K) {
      bool again = false;
      for (int i = 0; i < a.K; i++) again |= to.id[i] == l.id[k] && i != j;
      if (l.id[k] < 0) {
        if (j < a.K) to.qv[j] = -1.0f;
      } else if (again) {
        float qv = 0.0f;
        bool first = true;
        for (int i = 0; i < a.K; i++)
          if (to.id[i] == l.id[k]) {
            qv += to.q[i];
            first = first && i >= j;
          }
        to.qv[j] = first ? qv : -1.0f;
      }
    }
  }
}
// The named tokens of a piece in shared memory set to -inf, by the warp that
// loaded the entries.
template <typename T> __device__ __forceinline__ void take_out(const Piece<T> &p, T *st, const Loaded &l) {
  constexpr int EV = Elem<T>::EV;
#pragma unroll
  for (int k = 0; k < KL; k++) {
    const int at = l.id[k] + p.r.mis - p.c0 * EV;              // element of the piece
    if (l.id[k] >= 0 && at >= 0 && at < p.cnt * EV) st[at] = Elem<T>::none();
  }
  tc::fence_proxy_async();                       // a later copy into this stage comes after these writes
}

// What the gradient and the loss of a row go by, from its statistics p (with a
// tail: of the tokens not named) and its entries; the same in every warp.
struct RowLoss {
  float m, all, f, total, qr;                    // e relative to p.m, times f, is relative to m; all: its sum
  __device__ __forceinline__ RowLoss(const Part &p, const float *sum)
      : m(p.m), all(p.s), f(1.0f), total(sum[0] + sum[1]), qr(sum[1]) {}
  template <bool TAIL>
  __device__ __forceinline__ void named(const DistillArgs &a, const Part &p, const Entries &s) {
    if (!TAIL) return;
    const int lane = threadIdx.x & 31;
    for (int j = lane; j < a.K; j += 32) m = fmaxf(m, s.z[j]);
    m = warp_max(m);
    float sum = 0.0f;
    for (int j = lane; j < a.K; j += 32)
      if (!(s.qv[j] < 0.0f)) sum += exp2f((s.z[j] - m) * a.c);
    f = exp2f(bounded((p.m - m) * a.c));
    all = fmaf(p.s, f, warp_sum(sum));
  }
  // The row's loss, by one warp.  It is small where the student is close to its
  // teacher, and a difference of terms as large as log V: these are added up in
  // double from the fp32 sums, which are good to about 1e-7 (all in fp32, the
  // rounding of log s alone, 5e-7, was 3e-5 of the loss at V = 20010,
  // temperature 2).
  template <bool TAIL>
  __device__ __forceinline__ void write_loss(const DistillArgs &a, const Part &p, const Entries &s, int n, float w) const {
    const int lane = threadIdx.x & 31;
    // the row's three logarithms, a lane each
    const double logs = log((double)(lane == 0 ? all : lane == 1 ? p.s : qr)), per = a.per_t;
    const double ls = __shfl_sync(FULL, logs, 0), lrest = __shfl_sync(FULL, logs, 1), lqr = __shfl_sync(FULL, logs, 2);
    double L = 0.0;
    for (int j = lane; j < a.K; j += 32) {
      const float qv = s.qv[j];
      if (qv > 0.0f) L += (double)qv * ((double)logf(qv) - (((double)s.z[j] - (double)m) * per - ls));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(FULL, L, o);
    if (TAIL && qr > 0.0f) L += (double)qr * (lqr - (lrest + ((double)p.m - (double)m) * per - ls));
    if (all == 0.0f) L = total > 0.0f ? INFINITY : 0.0f;       // a student that allows no token
    if (all != all || total != total) L = NAN;
    L *= (double)w;
    if (lane == 0) {
      if (a.loss) a.loss[n] = (float)L;
      if (a.loss64) a.loss64[n] = L;
    }
  }
  // The factor of e_v of the tokens not named; g = dL's factor.
  template <bool TAIL> __device__ __forceinline__ float factor(const Part &p, float g) const {
    return all == 0.0f ? 0.0f : g * (total * f / all - (TAIL && qr > 0.0f && p.s > 0.0f ? qr / p.s : 0.0f));
  }
};

// A row's gradient rows: chunks of the row's own alignment go out 16 bytes at a
// time where the gradient's rows have it too.
template <typename T> struct Out {
  static constexpr int EV = Elem<T>::EV;
  Chunks<T> o;
  const Chunks<T> &r;
  bool same;
  __device__ __forceinline__ Out(const DistillArgs &a, const Chunks<T> &r_, int n)
      : o(static_cast<const T *>(a.dz) + (a.dz ? (size_t)n * a.ldd : 0), a.l.V), r(r_), same(o.mis == r_.mis) {}
  __device__ __forceinline__ void each(int c, const float (&f)[EV]) const {
    const int v = r.first(c);
#pragma unroll
    for (int e = 0; e < EV; e++)
      if (v + e >= 0 && v + e < r.V) o.row[v + e] = Elem<T>::from_f(f[e]);
  }
  // The others' gradients of a piece in shared memory.
  // ONCE: the row's other pieces are to stay in L2 meanwhile.
  template <int TH, bool ONCE>
  __device__ __forceinline__ void piece(uint32_t st, int c0, int cnt, const Part &p, float c, float coef) const {
    const int in0 = same ? max(0, r.full0 - c0) : cnt, in1 = same ? max(in0, min(cnt, r.full1 - c0)) : cnt;
    uint4 *const out = o.base + c0;
    const f32x2 nm2 = pack2(-p.m, -p.m), c2 = pack2(c, c), k2 = pack2(coef, coef);
    for_chunks<T, TH>(st, cnt, [&](const uint4 &x, int i) {
      float v[EV];
      Elem<T>::unpack(x, v);
#pragma unroll
      for (int e = 0; e < EV; e += 2) {
        float d0, d1;
        unpack2(mul2(add2(pack2(v[e], v[e + 1]), nm2), c2), d0, d1);
        unpack2(mul2(pack2(exp2_fast(d0), exp2_fast(d1)), k2), v[e], v[e + 1]);
      }
      if ((unsigned)(i - in0) < (unsigned)(in1 - in0)) {
        if (ONCE) __stcs(out + i, Elem<T>::pack(v));
        else out[i] = Elem<T>::pack(v);
      }
      else if (i < cnt) {
        each(c0 + i, v);
      }
    });
  }
  __device__ __forceinline__ void zeros(int c0, int cnt, int t, int TH) const {
    const float f[EV] = {};
    for (int i = c0 + t; i < c0 + cnt; i += TH) {
      if (same && i >= r.full0 && i < r.full1) o.base[i] = make_uint4(0, 0, 0, 0);
      else each(i, f);
    }
  }
  // The named tokens' gradients, those in chunks [c0, c0 + cnt).
  __device__ __forceinline__ void named(const DistillArgs &a, const Entries &s, const RowLoss &l, float g, int c0, int cnt,
                                        int t, int TH) const {
    if (l.all == 0.0f) return;
    for (int j = t; j < a.K; j += TH) {
      const float q = s.qv[j];
      if (q < 0.0f) continue;
      const int id = s.id[j], at = (id + r.mis) / EV;
      if (at < c0 || at >= c0 + cnt) continue;
      const float p = exp2_fast((s.z[j] - l.m) * a.c) / l.all;
      o.row[id] = Elem<T>::from_f(g * (l.total * p - q));
    }
  }
};

// Few rows, each split over the blocks of a cluster, a piece a block.
template <typename T, int TH, bool TAIL>
__global__ void __launch_bounds__(TH, min_blocks(TH)) distill_cluster_kernel(const DistillArgs a) {
  using TM = Team;
  constexpr int W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  // two of each, for rows in turn: a barrier of the next row lies between a
  // row's last reads and the row after that's writes
  __shared__ Part s_part[2][W], s_from[2][MAX_CLUSTER];
  __shared__ float s_sum[2][2];
  __shared__ uint64_t s_full;
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = (int)TM::size(), rank = (int)TM::rank();
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x / S, first_row = (int)blockIdx.x / S;
  const Pipe<T> pipe{reinterpret_cast<uint4 *>(s_dyn), 1, a.l.chunks, &s_full, &s_abort, a.err};
  auto counts = [&](int n) { return !a.weight || a.weight[n] != 0.0f; };
  if (tid == 0) {
    tc::mbar_init(tc::smem_u32(&s_full), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pipe.issue(t, first_row, rank, 0, counts(first_row), l2_normal());
  }
  TM::sync();
  uint32_t phase = 0;
  for (int n = first_row, flip = 0; n < N; n += stride, flip ^= 1, phase ^= 1) {
    const Piece<T> pc(t, n, rank);
    const Out<T> out(a, pc.r, n);
    const float w = a.weight ? a.weight[n] : 1.0f;
    const int ahead = n + stride;
    const bool next_counts = tid == 0 && ahead < N && counts(ahead);
    const uint32_t st = tc::smem_u32(s_dyn);
    const Entries s(s_dyn + (size_t)a.l.chunks * 16, a.K, flip);
    if (w == 0.0f) {                             // a row that does not count is not read
      if (a.dz) out.zeros(pc.c0, pc.cnt, tid, TH);
      if (rank == 0 && tid == 0) {
        if (a.loss) a.loss[n] = 0.0f;
        if (a.loss64) a.loss64[n] = 0.0;
      }
      pipe.wait(&s_full, phase);
      TM::sync();
      if (tid == 0 && ahead < N) pipe.issue(t, ahead, rank, 0, next_counts, l2_normal());
      continue;
    }
    Loaded l;
    if (warp == 0) {
      l.load(a, n);
      teach<T, TAIL>(a, pc.r, l, s, s_sum[flip]);
    }
    pipe.wait(&s_full, phase);
    if (t.ragged) pc.mask_ends(pipe.stage(0), [&](int i) { return i % TH == tid; });
    if (TAIL) {
      if (warp == 0) take_out(pc, reinterpret_cast<T *>(s_dyn), l);
      __syncthreads();
    }
    Running run;
    add_share<T, TH, false>(run, st, pc.cnt, a.c);
    Part p = run.warp<false>(a.c);
    if (lane == 0) s_part[flip][warp] = p;
    meet<false>(s_part[flip], s_from[flip], 0, a.c);
    p = join_all<false>(s_from[flip], S, a.c);
    RowLoss row(p, s_sum[flip]);
    row.named<TAIL>(a, p, s);
    if (rank == 0 && warp == 0 && (a.loss || a.loss64)) row.write_loss<TAIL>(a, p, s, n, w);
    const float g = w * a.scale * a.inv_t;
    if (a.dz) out.template piece<TH, false>(st, pc.c0, pc.cnt, p, a.c, row.factor<TAIL>(p, g));
    __syncthreads();
    if (tid == 0 && ahead < N) pipe.issue(t, ahead, rank, 0, next_counts, l2_normal());
    if (a.dz) out.named(a, s, row, g, pc.c0, pc.cnt, tid, TH);
  }
  TM::sync();                                    // no block leaves while another may write to it
}

// Rows of one block each, in pieces one after another: TH threads compute, one
// more warp keeps the pieces coming and one reads the teacher's entries a row
// ahead and takes the named tokens out of the pieces.  A row of one piece is
// kept in shared memory between the statistics and the gradient, a longer one
// comes a second time, from L2 if the rows in flight fit there.
template <typename T, int TH, bool TAIL>
__global__ void __launch_bounds__(TH + 64, min_blocks(TH + 64)) distill_kernel(const DistillArgs a) {
  constexpr int W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  __shared__ Part s_part[2][W];
  __shared__ float s_sum[2][2], s_weight[2];
  __shared__ uint64_t s_full[MAX_STAGES], s_ready[MAX_STAGES], s_free[MAX_STAGES], s_taught[2], s_spent[2];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x, first_row = (int)blockIdx.x, stages = a.l.stages, pieces = a.l.pieces;
  const int passes = a.dz && pieces > 1 ? 2 : 1;
  void *const entries = s_dyn + (size_t)stages * a.l.chunks * 16;
  const Pipe<T> pipe{reinterpret_cast<uint4 *>(s_dyn), stages, a.l.chunks, s_full, &s_abort, a.err};
  if (tid == 0) {
    for (int i = 0; i < stages; i++) {
      tc::mbar_init(tc::smem_u32(&s_full[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_ready[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_free[i]), W);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(tc::smem_u32(&s_taught[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_spent[i]), W);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == W) {                               // ---- the pieces
    Turn put;
    const uint64_t first = passes == 2 ? l2_again() : l2_normal(), last = l2_once();
    int k = 0;
    float w = a.weight ? a.weight[first_row] : 1.0f;
    for (int n = first_row; n < N; n += stride) {
      const bool read = w != 0.0f;
      if (a.weight && n + stride < N) w = a.weight[n + stride];
      for (int i = 0; read && i < passes * pieces; i++, k++) {
        if (k >= stages) pipe.wait(&s_free[put.s], put.phase ^ 1);
        if (lane == 0) pipe.issue(t, n, i % pieces, put.s, true, i < pieces ? first : last);
        __syncwarp();
        put.next(stages);
      }
    }
    return;
  }
  if (warp == W + 1) {                           // ---- the teacher
    Turn get;
    Loaded next;
    next.load(a, first_row);
    float w_next = a.weight ? a.weight[first_row] : 1.0f;
    int rows = 0;
    for (int n = first_row; n < N; n += stride, rows++) {
      const int flip = rows & 1;
      Loaded l = next;
      const float w = w_next;
      if (n + stride < N) {
        next.load(a, n + stride);
        if (a.weight) w_next = a.weight[n + stride];
      }
      if (rows >= 2) pipe.wait(&s_spent[flip], ((rows >> 1) - 1) & 1);
      if (w != 0.0f) teach<T, TAIL>(a, t.row(n), l, Entries(entries, a.K, flip), s_sum[flip]);
      __syncwarp();
      if (lane == 0) {
        s_weight[flip] = w;
        tc::mbar_arrive(tc::smem_u32(&s_taught[flip]));
      }
      for (int i = 0; TAIL && w != 0.0f && i < passes * pieces; i++) {
        pipe.wait(&s_full[get.s], get.phase);
        // the second time the named tokens are written over anyway
        if (i < pieces) take_out(Piece<T>(t, n, i), reinterpret_cast<T *>(pipe.stage(get.s)), l);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_ready[get.s]));
        get.next(stages);
      }
    }
    return;
  }
  // ---- the computing warps
  Turn turn;
  auto arrived = [&] {
    pipe.wait(&s_full[turn.s], turn.phase);
    if (TAIL) pipe.wait(&s_ready[turn.s], turn.phase);
  };
  auto done = [&] {
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_free[turn.s]));
    turn.next(stages);
  };
  int rows = 0;
  for (int n = first_row; n < N; n += stride, rows++) {
    const int flip = rows & 1;
    const Entries s(entries, a.K, flip);
    const Chunks<T> r = t.row(n);
    const Out<T> out(a, r, n);
    pipe.wait(&s_taught[flip], (rows >> 1) & 1);
    const float w = s_weight[flip];
    if (w == 0.0f) {                             // a row that does not count is not read
      if (a.dz) out.zeros(0, r.n, tid, TH);
      if (tid == 0) {
        if (a.loss) a.loss[n] = 0.0f;
        if (a.loss64) a.loss64[n] = 0.0;
      }
    } else {
      Running run;
      for (int i = 0; i < pieces; i++) {
        arrived();
        if (t.ragged) Piece<T>(t, n, i).mask_ends(pipe.stage(turn.s), [&](int k) { return k % TH == tid; });
        add_share<T, TH, false>(run, tc::smem_u32(pipe.stage(turn.s)), max(0, min(r.n - i * t.per, t.per)), a.c);
        if (pieces > 1 || !a.dz) done();
      }
      Part p = run.warp<false>(a.c);
      if (lane == 0) s_part[flip][warp] = p;
      bar_sync<TH>();
      p = join_all<false>(s_part[flip], W, a.c);
      RowLoss row(p, s_sum[flip]);
      row.named<TAIL>(a, p, s);
      const float g = w * a.scale * a.inv_t;
      if (a.dz) {
        const float coef = row.factor<TAIL>(p, g);
        if (pieces == 1) {
          out.template piece<TH, false>(tc::smem_u32(pipe.stage(turn.s)), 0, r.n, p, a.c, coef);
          done();
        }
        for (int i = 0; pieces > 1 && i < pieces; i++) {
          arrived();
          out.template piece<TH, true>(tc::smem_u32(pipe.stage(turn.s)), i * t.per, max(0, min(r.n - i * t.per, t.per)),
                                       p, a.c, coef);
          done();
        }
        bar_sync<TH>();
        out.named(a, s, row, g, 0, r.n, tid, TH);
      }
      if (warp == W - 1 && (a.loss || a.loss64)) row.write_loss<TAIL>(a, p, s, n, w);
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_spent[flip]));
  }
}

}  // namespace lg

namespace {

template <typename T, int TPR>
int launch_grad(DeviceCtx *c, int nch, const lg::GradArgs &a) {
  const int segs = (nch + TPR * lg::CPT<T> - 1) / (TPR * lg::CPT<T>);
  const long long groups = ((long long)a.N * TPR + 255) / 256;
  if (groups * segs > 0x7FFFFFFFLL) return set_error(TL_EINVAL, "N = %d rows of V = %d are too many for one launch", a.N, a.V);
  const unsigned grid = (unsigned)(groups * segs);
  if (a.dentropy) lg::token_logprobs_bwd_kernel<T, TPR, true><<<grid, 256, 0, c->stream>>>(a, segs);
  else lg::token_logprobs_bwd_kernel<T, TPR, false><<<grid, 256, 0, c->stream>>>(a, segs);
  TL_TRY_CUDA(cudaGetLastError());
  return TL_OK;
}
template <typename T> int grad_typed(DeviceCtx *c, const lg::GradArgs &a) {
  constexpr int EV = lg::Elem<T>::EV;
  const int nch = (a.V + 2 * EV - 2) / EV;       // chunks of a row at the worst alignment
  if (nch <= 32 * lg::CPT<T>) return launch_grad<T, 32>(c, nch, a);
  if (nch <= 128 * lg::CPT<T>) return launch_grad<T, 128>(c, nch, a);
  return launch_grad<T, 256>(c, nch, a);
}

template <typename T, int TH, bool TAIL> int launch_cluster(DeviceCtx *c, const RowPlan &pl, lg::DistillArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::distill_cluster_kernel<T, TH, TAIL>, c, pl, 0, 32 * a.K, &seen[c->device], &a);
}
template <typename T, int TH, bool TAIL> int launch_distill(DeviceCtx *c, const RowPlan &pl, lg::DistillArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::distill_kernel<T, TH, TAIL>, c, pl, 64, 32 * a.K, &seen[c->device], &a);
}
template <typename T, bool TAIL> int distill_typed(DeviceCtx *c, const RowPlan &pl, const lg::DistillArgs &a) {
  if (pl.blocks > 1) {
    if (pl.threads == 128) return launch_cluster<T, 128, TAIL>(c, pl, a);
    return pl.threads == 256 ? launch_cluster<T, 256, TAIL>(c, pl, a) : launch_cluster<T, 512, TAIL>(c, pl, a);
  }
  if (pl.threads == 32) return launch_distill<T, 32, TAIL>(c, pl, a);
  return pl.threads == 128 ? launch_distill<T, 128, TAIL>(c, pl, a) : launch_distill<T, 256, TAIL>(c, pl, a);
}

}  // namespace

int k_token_logprobs_bwd(DeviceCtx *c, void *dlogits, long long ldd, const LogitRows &z, const int *ids,
                         float temperature, const float *stats, const float *entropy, const float *dlogp,
                         const float *dentropy) {
  TraceScope ts(c, "k_token_logprobs_bwd");
  const lg::GradArgs a{dlogits, ldd, z.p, z.ld, ids, z.N, z.V, lg::LOG2E / temperature, 1.0f / temperature, stats,
                       entropy, dlogp, dentropy, c->err_flag};
  if (z.dtype == TL_F32) return grad_typed<float>(c, a);
  if (z.dtype == TL_BF16) return grad_typed<__nv_bfloat16>(c, a);
  return grad_typed<__half>(c, a);
}

int k_distill_topk(DeviceCtx *c, const LogitRows &z, const int *t_ids, const float *t_vals, int K,
                   float temperature, int tail, const float *weight, float scale, float *loss, double *loss64,
                   void *dlogits, long long ldd) {
  TraceScope ts(c, "k_distill_topk");
  const RowPlan pl = plan_rows(c, z, 0, true);
  const lg::DistillArgs a{pl.l, t_ids, t_vals, K, lg::LOG2E / temperature, 1.0f / temperature,
                          1.0 / (double)temperature, weight, scale, loss,
                          loss64, dlogits, ldd, c->err_flag};
  if (z.dtype == TL_F32) return tail ? distill_typed<float, true>(c, pl, a) : distill_typed<float, false>(c, pl, a);
  if (z.dtype == TL_BF16)
    return tail ? distill_typed<__nv_bfloat16, true>(c, pl, a) : distill_typed<__nv_bfloat16, false>(c, pl, a);
  return tail ? distill_typed<__half, true>(c, pl, a) : distill_typed<__half, false>(c, pl, a);
}

}  // namespace tl
