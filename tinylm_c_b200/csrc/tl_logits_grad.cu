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
    if (c0 == 0) report_token(a.err);
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
  // log2 p = (z - m) c - ls log2(e); the factor of p: -(a + b (log p + H)).  A
  // token without probability has a finite factor up to |b| = 2^119.
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
      const f32x2 k2 = ENT ? fma2(pack2(bounded<-256>(l0), bounded<-256>(l1)), fb2, fa2) : fa2;
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
  int K, tail;
  float c;                           // log2(e) / temperature
  double per;                        // 1 / temperature
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
// Where the student is confident or close to its teacher these are small
// differences: Q p_v - q_v of p and q near 1, 1 - sum q, log q - log p.  So the
// K entries of a row are worked out in double by one warp, the teacher's side
// (q, the tail) a row ahead, the student's (the named tokens' e relative to
// their own largest logit) as the row arrives.  The named tokens are taken out of the row (set to -inf in shared
// memory) before its statistics, so these are of the others alone, in fp32.
// An error of theirs (about 1e-7) is then one factor 1 + delta of p_r, and
// moves p_n = 1 - p_r by delta p_r p_n only.  Of 600 small fp32 cases
// (temperatures 0.5, 1 and 2) loss and gradient are 5e-6 of themselves off at
// most; all in fp32 46 were over 1e-5, up to 2e-1.  All others' gradients are
// one factor times e_v; the named tokens' are written over them at the end.
//
// A row's entries in shared memory, K of each in places that rows take in turn:
// the token (-1: padding), its share of the teacher's mass before it is
// normalised (entries naming one token add up, the first of them stands for it;
// -1 for the others of them and for padding) and its e.
constexpr int PLACES = 2;
struct Entries {
  static constexpr int BITS = 9;
  double *q, *e;
  int *id;
  unsigned char *table;                          // of the warp that works them out, see teach()
  static __host__ __device__ __forceinline__ int even(int K) { return (K + 1) & ~1; }
  static __host__ __device__ __forceinline__ int bytes(int K) { return PLACES * even(K) * (2 * 8 + 4) + (1 << BITS); }
  __device__ __forceinline__ Entries(void *p, int K, int place)
      : q(static_cast<double *>(p) + place * even(K)), e(q + PLACES * even(K)),
        id(reinterpret_cast<int *>(static_cast<double *>(p) + 2 * PLACES * even(K)) + place * even(K)),
        table(reinterpret_cast<unsigned char *>(static_cast<double *>(p) + 2 * PLACES * even(K)) + PLACES * even(K) * 4) {}
};
// What else of a row's teacher, and of the student's side of its tokens.
struct Taught {
  double named, tail;                            // sum of q over the named tokens, q_r
  double mass;                                   // sum of the entries' shares
  double own;                                    // sum of share (log share - (z - m) / temperature)
  double s;                                      // sum of e over the named tokens
  float m;                                       // the named tokens' largest logit, what e is relative to
  // q of an entry is its share times this
  __device__ __forceinline__ double norm(bool tail) const { return tail || mass == 0.0 ? 1.0 : 1.0 / mass; }
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
// The teacher's distribution from a row's loaded entries, by one warp; `own` of
// the result still lacks the student's logits.
__device__ __forceinline__ Taught teach(const DistillArgs &a, Loaded &l, const Entries &to) {
  const int lane = threadIdx.x & 31;
  float tm = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < KL; k++) {
    const int j = k * 32 + lane;
    if ((unsigned)l.id[k] >= (unsigned)a.l.V) {
      if (l.id[k] != -1) report_token(a.err);
      l.id[k] = -1;
      l.t[k] = -INFINITY;
    }
    tm = fmaxf(tm, l.t[k]);
    if (j < a.K) to.id[j] = l.id[k];
  }
  tm = warp_max(tm);
  double mass = 0.0, own = 0.0;
#pragma unroll
  for (int k = 0; k < KL; k++)
    if (k * 32 + lane < a.K) to.q[k * 32 + lane] = a.tail ? (double)l.t[k] : ((double)l.t[k] - (double)tm) * a.per;
#pragma unroll 1                       // one copy of the code: unrolled, 16384 x 8192 fp32, K = 64 takes 230 instead of 218 us
  for (int j = lane; j < a.K; j += 32) {
    const double u = to.q[j], x = exp(u);
    const bool is = to.id[j] >= 0;
    to.q[j] = is ? x : -1.0;
    if (is) {
      mass += x;
      if (x > 0.0) own += x * u;                 // its logarithm is known
    }
  }
  __syncwarp();
  // Whether the row names a token twice: the lanes compare theirs; where a lane
  // has several, entries that fall into one place of a table are told apart by
  // the one that stays there, the others try again.
  unsigned open = 0;                             // a bit each of the lane's entries not told apart yet
  bool twice = false;
  if (a.K <= 32) {
    twice = __popc(__match_any_sync(FULL, l.id[0])) > 1 && l.id[0] >= 0;
  } else {
#pragma unroll
    for (int k = 0; k < KL; k++) open |= l.id[k] >= 0 ? 1u << k : 0;
  }
  auto place = [&](int k) { return &to.table[(unsigned)l.id[k] * 2654435769u >> (32 - Entries::BITS)]; };
  while (__any_sync(FULL, open != 0)) {
#pragma unroll
    for (int k = 0; k < KL; k++)
      if (open >> k & 1) *place(k) = (unsigned char)(k * 32 + lane);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < KL; k++)
      if (open >> k & 1) {
        const int j = *place(k);
        const bool mine = j == k * 32 + lane, same = !mine && to.id[j] == l.id[k];
        twice |= same;
        if (mine || same) open ^= 1u << k;
      }
    __syncwarp();
  }
  if (__any_sync(FULL, twice)) {
    unsigned again = 0;                          // a bit each of the lane's entries whose token an earlier one names
#pragma unroll 1
    for (int k = 0; k * 32 < a.K; k++) {
      const int j = k * 32 + lane, id = j < a.K ? to.id[j] : -1;
      if (id < 0) continue;
      double q = to.q[j];
      for (int i = 0; i < a.K; i++)
        if (to.id[i] == id) {
          if (i < j) again |= 1u << k;
          if (i > j) q += to.q[i];
        }
      if (!(again >> k & 1)) to.q[j] = q;        // read by no other lane: it stands first
    }
    __syncwarp();
    own = 0.0;
#pragma unroll 1
    for (int j = lane, k = 0; j < a.K; j += 32, k++) {
      const double x = to.q[j];
      if (again >> k & 1) to.q[j] = -1.0;
      else if (x > 0.0) own += x * log(x);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    mass += __shfl_xor_sync(FULL, mass, o);
    own += __shfl_xor_sync(FULL, own, o);
  }
  double Q = a.tail || mass == 0.0 ? mass : 1.0;
  if (!(mass < (double)INFINITY)) Q = (double)NAN;             // a NaN or +inf among the values
  double qr = a.tail ? 1.0 - Q : 0.0;
  if (qr < (double)TAIL_MIN) qr = 0.0;           // NaN stays
  __syncwarp();
  return Taught{Q, qr, mass, own, 0.0, -FLT_MAX};
}
// The tokens that a row's entries stand for (q not negative) and that lie in a
// piece in shared memory: their logits go to e, and -inf to their
// place in the piece.  By the warp that worked the entries out; m becomes the
// lane's largest logit.
template <typename T> __device__ __forceinline__ void take_out(const DistillArgs &a, const Piece<T> &p, T *st, const Entries &s, float &m) {
  constexpr int EV = Elem<T>::EV;
  for (int j = threadIdx.x & 31; j < a.K; j += 32) {
    const int at = s.id[j] + p.r.mis - p.c0 * EV;              // element of the piece
    if (!(s.q[j] < 0.0) && at >= 0 && at < p.cnt * EV) {
      const float z = Elem<T>::to_f(st[at]);
      s.e[j] = (double)z;
      m = fmaxf(m, z);
      st[at] = Elem<T>::none();
    }
  }
  tc::fence_proxy_async();                       // a later copy into this stage comes after these writes
}
// The student's side of the row's tokens from their logits in e, m the lane's
// largest of them, by that warp; lane 0 writes the result.
__device__ __forceinline__ void look_at_student(const DistillArgs &a, const Entries &s, float m, Taught t, Taught *out) {
  const int lane = threadIdx.x & 31;
  t.m = warp_max(m);
  double sum = 0.0, own = 0.0;
#pragma unroll 1
  for (int j = lane; j < a.K; j += 32) {
    const double q = s.q[j];
    if (q < 0.0) continue;
    const double d = (s.e[j] - (double)t.m) * a.per, e = exp(d);
    s.e[j] = e;
    sum += e;
    if (q > 0.0) own += q * d;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(FULL, sum, o);
    own += __shfl_xor_sync(FULL, own, o);
  }
  t.s = sum;
  t.own -= own;
  if (lane == 0) *out = t;
  __syncwarp();
}

// What the gradient and the loss of a row go by, from the statistics p of the
// tokens not named and its teacher; the same in every thread.
struct RowLoss {
  double fn, n, r, all;                          // n, r: the sums of e of the named and of the others, relative to one logit
  __device__ __forceinline__ RowLoss(const DistillArgs &a, const Part &p, const Taught &t) {
    const float m = fmaxf(p.m, t.m);
    fn = (double)exp2f((t.m - m) * a.c);
    n = t.s * fn;
    r = (double)p.s * (double)exp2f((p.m - m) * a.c);
    all = n + r;
  }
  // The row's loss, by one warp: a difference of terms as large as log V that
  // is small where the student is close to its teacher, so in double throughout.
  __device__ __forceinline__ static void write(const DistillArgs &a, const Part &p, const Taught &t, int n, float w) {
    const int lane = threadIdx.x & 31;
    const double m = fmax((double)p.m, (double)t.m), dn = ((double)t.m - m) * a.per, dr = ((double)p.m - m) * a.per;
    // a lane each for what takes two exponentials and three logarithms
    const double e = exp(lane == 0 ? dn : dr) * (lane == 0 ? t.s : (double)p.s);
    const double all = __shfl_sync(FULL, e, 0) + __shfl_sync(FULL, e, 1);
    const bool shares = !a.tail && t.mass != 0.0;
    const double logs = log(lane == 0 ? all : lane == 1 ? (double)p.s : shares ? t.mass : t.tail);
    const double lall = __shfl_sync(FULL, logs, 0), lrest = __shfl_sync(FULL, logs, 1), lq = __shfl_sync(FULL, logs, 2);
    double L = shares ? t.own / t.mass - lq : t.own;
    if (t.named > 0.0) L -= t.named * (dn - lall);
    if (t.tail > 0.0) L += t.tail * (lq - (lrest + dr - lall));
    const double total = t.named + t.tail;
    if (all == 0.0) L = total > 0.0 ? (double)INFINITY : 0.0;  // a student that allows no token
    if (all != all || total != total) L = (double)NAN;
    L *= (double)w;
    if (lane == 0) {
      if (a.loss) a.loss[n] = (float)L;
      if (a.loss64) a.loss64[n] = L;
    }
  }
  // The factor of e_v of the tokens not named, g times
  //   Q r / (all s) - q_r / s = (q_n r - q_r n) / (all s),
  // the difference in double: near 0 for a student close to its teacher.
  __device__ __forceinline__ float factor(const Part &p, const Taught &t, double g) const {
    if (all == 0.0 || p.s == 0.0f) return 0.0f;
    return (float)g * ((float)(t.named * r - t.tail * n) / (float)(all * (double)p.s));
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
  __device__ __forceinline__ void named(const DistillArgs &a, const Entries &s, const Taught &t, const RowLoss &l, double g,
                                        int c0, int cnt, int tid, int TH) const {
    if (l.all == 0.0 || tid >= a.K) return;
    const double f = (t.named + t.tail) * l.fn / l.all, norm = t.norm(a.tail);
    for (int j = tid; j < a.K; j += TH) {
      const double q = s.q[j] * norm;
      if (q < 0.0) continue;
      const int id = s.id[j], at = (id + r.mis) / EV;
      if (at < c0 || at >= c0 + cnt) continue;
      o.row[id] = Elem<T>::from_f((float)(g * (s.e[j] * f - q)));
    }
  }
};

// Few rows, each split over the blocks of a cluster, a piece a block.
template <typename T, int TH>
__global__ void __launch_bounds__(TH, min_blocks(TH)) distill_cluster_kernel(const DistillArgs a) {
  using TM = Team;
  constexpr int W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  // two of each, for rows in turn: a barrier of the next row lies between a
  // row's last reads and the row after that's writes
  __shared__ Part s_part[2][W], s_from[2][MAX_CLUSTER];
  __shared__ Taught s_teacher[2];
  __shared__ uint64_t s_full;
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = (int)TM::size(), rank = (int)TM::rank();
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x / S, first_row = (int)blockIdx.x / S;
  const Pipe<T> pipe(s_dyn, a.l, 1, &s_abort, a.err);
  auto counts = [&](int n) { return !a.weight || a.weight[n] != 0.0f; };
  int issued = 0;                                // by thread 0
  if (tid == 0) {
    tc::mbar_init(tc::smem_u32(&s_full), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    issued += pipe.issue(t, first_row, rank, 0, &s_full, counts(first_row), l2_normal());
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
      if (tid == 0 && ahead < N) issued += pipe.issue(t, ahead, rank, 0, &s_full, next_counts, l2_normal());
      continue;
    }
    if (warp == 0) {                             // the tokens' logits from memory: another block may hold them
      Loaded l;
      l.load(a, n);
      const Taught of = teach(a, l, s);
      float m = -FLT_MAX;
      for (int j = lane; j < a.K; j += 32)
        if (!(s.q[j] < 0.0)) {
          const float z = Elem<T>::to_f(pc.r.row[s.id[j]]);
          s.e[j] = (double)z;
          m = fmaxf(m, z);
        }
      look_at_student(a, s, m, of, &s_teacher[flip]);
    }
    pipe.wait(&s_full, phase);
    if (t.ragged) pc.mask_ends(pipe.stage(0), [&](int i) { return i % TH == tid; });
    if (warp == 0) {
      for (int j = lane; j < a.K; j += 32) {
        const int at = s.id[j] + pc.r.mis - pc.c0 * Elem<T>::EV;
        if (s.id[j] >= 0 && at >= 0 && at < pc.cnt * Elem<T>::EV) reinterpret_cast<T *>(s_dyn)[at] = Elem<T>::none();
      }
      tc::fence_proxy_async();                   // a later copy into this stage comes after these writes
    }
    __syncthreads();
    Running run;
    add_share<T, TH, false>(run, st, pc.cnt, a.c);
    Part p = run.warp<false>(a.c);
    if (lane == 0) s_part[flip][warp] = p;
    meet<false>(s_part[flip], s_from[flip], 0, a.c);
    p = join_all<false>(s_from[flip], S, a.c);
    const Taught &teacher = s_teacher[flip];
    const RowLoss row(a, p, teacher);
    if (rank == 0 && warp == 0 && (a.loss || a.loss64)) RowLoss::write(a, p, teacher, n, w);
    const double g = (double)w * (double)a.scale * a.per;
    if (a.dz) out.template piece<TH, false>(st, pc.c0, pc.cnt, p, a.c, row.factor(p, teacher, g));
    __syncthreads();
    if (tid == 0 && ahead < N) issued += pipe.issue(t, ahead, rank, 0, &s_full, next_counts, l2_normal());
    if (a.dz) out.named(a, s, teacher, row, g, pc.c0, pc.cnt, tid, TH);
  }
  if (tid == 0) pipe.drain(&s_full, 1, issued);
  TM::sync();                                    // no block leaves while another may write to it
}

// Rows of one block each, in pieces one after another: TH threads compute, one
// more warp keeps the pieces coming and finishes rows (the named tokens'
// gradients, the loss), and one works the teacher's entries out a row ahead and
// takes the named tokens out of the pieces as they arrive.  A row of one piece is
// kept in shared memory between the statistics and the gradient, a longer one
// comes a second time, from L2 if the rows in flight fit there.
template <typename T, int TH>
__global__ void __launch_bounds__(TH + 64, min_blocks(TH + 64)) distill_kernel(const DistillArgs a) {
  constexpr int W = TH / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  __shared__ Part s_part[PLACES][W];
  __shared__ Taught s_teacher[PLACES];
  __shared__ float s_weight[PLACES];
  // s_full, s_ready: of the pieces that come the first time, in a ring of their
  // own (the teacher waits for these alone); s_late: of those that come again
  __shared__ uint64_t s_full[MAX_STAGES], s_ready[MAX_STAGES], s_late[MAX_STAGES], s_free[MAX_STAGES];
  // of a row: its weight is there, its entries are, the others' gradients are
  // written, all of it is
  __shared__ uint64_t s_taught[PLACES], s_seen[PLACES], s_spent[PLACES], s_over[PLACES];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Rows<T> t(a.l);
  const int N = a.l.N, stride = (int)gridDim.x, first_row = (int)blockIdx.x, stages = a.l.stages, pieces = a.l.pieces;
  const int passes = a.dz && pieces > 1 ? 2 : 1;
  void *const entries = s_dyn + (size_t)stages * a.l.chunks * 16;
  const Pipe<T> pipe(s_dyn, a.l, stages, &s_abort, a.err);
  if (tid == 0) {
    for (int i = 0; i < stages; i++) {
      tc::mbar_init(tc::smem_u32(&s_full[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_ready[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_late[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_free[i]), W);
    }
    for (int i = 0; i < PLACES; i++) {
      tc::mbar_init(tc::smem_u32(&s_taught[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_seen[i]), 1);
      tc::mbar_init(tc::smem_u32(&s_spent[i]), W);
      tc::mbar_init(tc::smem_u32(&s_over[i]), 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int rows = (N - first_row + stride - 1) / stride;      // the block's
  if (warp == W) {                               // ---- the pieces, and what is left of rows that are done
    Turn put, early, late, over;                 // over: the place of the row that is finished next
    const uint64_t first = passes == 2 ? l2_again() : l2_normal(), last = l2_once();
    // a row is finished when the copies behind it are under way, as many as there are stages
    const int total = passes * pieces, behind = total == 1 ? stages - 1 : 1, when = min(stages, total) - 1;
    int issued = 0, early_issued = 0, late_issued = 0;
    float w = a.weight ? a.weight[first_row] : 1.0f;
    for (int k = 0; k < rows + behind; k++) {
      const int n = first_row + k * stride;
      const bool read = k < rows && w != 0.0f;
      if (a.weight && k + 1 < rows) w = a.weight[n + stride];
      for (int i = 0; i == 0 || (read && i < total); i++) {
        if (read) {
          if (issued++ >= stages && !pipe.wait_all(&s_free[put.s], put.phase ^ 1)) goto out;
          const bool again = i >= pieces;
          const bool ok = lane != 0 || pipe.issue(t, n, again ? i - pieces : i, put.s,
                                                  again ? &s_late[late.s] : &s_full[early.s], true, again ? last : first);
          if (!__all_sync(FULL, ok)) goto out;
          put.next(stages);
          (again ? late : early).next(stages);
          (again ? late_issued : early_issued)++;
        }
        if (k < behind || i != (read ? when : 0)) continue;
        const int done = n - behind * stride;
        if (!pipe.wait_all(&s_spent[over.s], over.phase)) goto out;
        const float wd = s_weight[over.s];
        if (wd != 0.0f) {
          const Part p = join_all<false>(s_part[over.s], W, a.c);
          const Taught &teacher = s_teacher[over.s];
          if (a.dz) {                            // the others' gradients are written
            const Chunks<T> r = t.row(done);
            Out<T>(a, r, done).named(a, Entries(entries, a.K, over.s), teacher, RowLoss(a, p, teacher),
                                     (double)wd * (double)a.scale * a.per, 0, r.n, lane, 32);
          }
          if (a.loss || a.loss64) RowLoss::write(a, p, teacher, done, wd);
        } else if (lane == 0) {
          if (a.loss) a.loss[done] = 0.0f;
          if (a.loss64) a.loss64[done] = 0.0;
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_over[over.s]));
        over.next(PLACES);
      }
    }
  out:
    if (lane == 0) {
      pipe.drain(s_full, stages, early_issued);
      pipe.drain(s_late, stages, late_issued);
    }
    return;
  }
  if (warp == W + 1) {                           // ---- the teacher
    Turn get, early, at;                         // the stages, the barriers of pieces that come the first time, the places
    Loaded l;                                    // the next row's entries
    Taught of;                                   // the row's teacher, its student's part not yet there
    l.load(a, first_row);
    float w = 0.0f, w_next = a.weight ? a.weight[first_row] : 1.0f;
    for (int k = 0; k <= rows; k++) {            // the block's k-th row
      const int n = first_row + k * stride;
      if (k >= 1) {                              // the row before, as it arrives
        if (w != 0.0f) {
          const Entries s(entries, a.K, at.s);
          float m = -FLT_MAX;
          for (int i = 0; i < pieces; i++) {
            if (!pipe.wait_all(&s_full[early.s], early.phase)) return;
            take_out(a, Piece<T>(t, n - stride, i), reinterpret_cast<T *>(pipe.stage(get.s)), s, m);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_ready[early.s]));
            early.next(stages);
            get.next(stages);
          }
          // the second time the named tokens are written over anyway
          for (int i = pieces; i < passes * pieces; i++) get.next(stages);
          look_at_student(a, s, m, of, &s_teacher[at.s]);
        }
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s_seen[at.s]));
        at.next(PLACES);
      }
      if (k == rows) break;
      // this one's teacher, while the computing warps work on the row before
      if (k >= PLACES && !pipe.wait_all(&s_over[at.s], at.phase ^ 1)) return;
      w = w_next;
      if (w != 0.0f) of = teach(a, l, Entries(entries, a.K, at.s));
      __syncwarp();
      if (lane == 0) {
        s_weight[at.s] = w;
        tc::mbar_arrive(tc::smem_u32(&s_taught[at.s]));
      }
      if (k + 1 < rows) {
        if (a.weight) w_next = a.weight[n + stride];
        l.load(a, n + stride);
      }
    }
    return;
  }
  // ---- the computing warps
  Turn turn, early, late, at;
  auto done = [&](bool ok) {
    __syncwarp();
    if (lane == 0 && ok) tc::mbar_arrive(tc::smem_u32(&s_free[turn.s]));
    turn.next(stages);
  };
  bool ok = true;                                // of each lane; what it leaves undone only its own warp and the barrier see
  for (int k = 0; k < rows; k++) {
    const int n = first_row + k * stride, place = at.s;
    const uint32_t phase = at.phase;
    const Chunks<T> r = t.row(n);
    const Out<T> out(a, r, n);
    ok &= pipe.wait(&s_taught[place], phase);
    at.next(PLACES);
    const float w = __all_sync(FULL, ok) ? s_weight[place] : 0.0f;
    Part p = no_part();
    if (w != 0.0f) {
      Running run;
      for (int i = 0; i < pieces; i++) {
        ok &= pipe.wait(&s_full[early.s], early.phase);
        ok &= pipe.wait(&s_ready[early.s], early.phase);
        early.next(stages);
        if (t.ragged) Piece<T>(t, n, i).mask_ends(pipe.stage(turn.s), [&](int c) { return c % TH == tid; });
        add_share<T, TH, false>(run, tc::smem_u32(pipe.stage(turn.s)), max(0, min(r.n - i * t.per, t.per)), a.c);
        if (pieces > 1 || !a.dz) done(ok);
      }
      p = run.warp<false>(a.c);
      if (lane == 0) s_part[place][warp] = p;
      ok &= pipe.wait(&s_seen[place], phase);
    }
    if (bar_any<TH>(!ok)) return;                // else w is the same in all warps
    if (w == 0.0f) {                             // a row that does not count is not read
      if (a.dz) out.zeros(0, r.n, tid, TH);
    } else if (a.dz) {
      p = join_all<false>(s_part[place], W, a.c);
      const Taught &teacher = s_teacher[place];
      const float coef = RowLoss(a, p, teacher).factor(p, teacher, (double)w * (double)a.scale * a.per);
      if (pieces == 1) {
        out.template piece<TH, false>(tc::smem_u32(pipe.stage(turn.s)), 0, r.n, p, a.c, coef);
        done(true);
      }
      for (int i = 0; pieces > 1 && i < pieces; i++) {
        ok &= pipe.wait(&s_late[late.s], late.phase);
        late.next(stages);
        out.template piece<TH, true>(tc::smem_u32(pipe.stage(turn.s)), i * t.per, max(0, min(r.n - i * t.per, t.per)), p,
                                     a.c, coef);
        done(ok);
      }
    }
    __syncwarp();
    if (lane == 0 && ok) tc::mbar_arrive(tc::smem_u32(&s_spent[place]));
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

template <typename T, int TH> int launch_cluster(DeviceCtx *c, const RowPlan &pl, lg::DistillArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::distill_cluster_kernel<T, TH>, c, pl, 0, lg::Entries::bytes(a.K), &seen[c->device],
                     &a);
}
template <typename T, int TH> int launch_distill(DeviceCtx *c, const RowPlan &pl, lg::DistillArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::distill_kernel<T, TH>, c, pl, 64, lg::Entries::bytes(a.K), &seen[c->device], &a);
}
template <typename T> int distill_typed(DeviceCtx *c, const RowPlan &pl, const lg::DistillArgs &a) {
  if (pl.blocks > 1) {
    if (pl.threads == 128) return launch_cluster<T, 128>(c, pl, a);
    return pl.threads == 256 ? launch_cluster<T, 256>(c, pl, a) : launch_cluster<T, 512>(c, pl, a);
  }
  if (pl.threads == 32) return launch_distill<T, 32>(c, pl, a);
  return pl.threads == 128 ? launch_distill<T, 128>(c, pl, a) : launch_distill<T, 256>(c, pl, a);
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
  const lg::DistillArgs a{pl.l, t_ids, t_vals, K, tail, lg::LOG2E / temperature, 1.0 / (double)temperature, weight, scale,
                          loss, loss64, dlogits, ldd, c->err_flag};
  if (z.dtype == TL_F32) return distill_typed<float>(c, pl, a);
  if (z.dtype == TL_BF16) return distill_typed<__nv_bfloat16>(c, pl, a);
  return distill_typed<__half>(c, pl, a);
}

}  // namespace tl
