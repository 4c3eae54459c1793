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
// threads take CPT chunks each of one row, 256 / TPR rows a block.
constexpr int CPT = 4;
template <typename T, int TPR, bool ENT>
__global__ void __launch_bounds__(256) token_logprobs_bwd_kernel(const GradArgs a, int segs) {
  constexpr int EV = Elem<T>::EV;
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
  float c, inv_t;
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
// The row is read once.  With a tail the named tokens are taken out of it (set
// to -inf in shared memory) before its statistics, so that p_r is summed and
// never 1 - sum p, which loses all its digits for a confident student.  All
// others' gradients are then one factor times e_v; the named tokens' are
// written over them at the end.
template <typename T, bool CL, bool TAIL>
__global__ void __launch_bounds__(MAX_THREADS, 2) distill_kernel(const DistillArgs a) {
  using TM = Team<CL>;
  constexpr int EV = Elem<T>::EV, KL = TL_TOPK_MAX / 32;
  extern __shared__ __align__(128) unsigned char s_dyn[];
  // two of each, for rows in turn: a barrier of the next row lies between a
  // row's last reads and the row after that's writes
  __shared__ Part s_part[2][MAX_WARPS], s_from[2][MAX_CLUSTER];
  __shared__ float s_sum[2][2];                  // sum of q, the tail
  __shared__ uint64_t s_full[MAX_STAGES];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, TH = blockDim.x;
  const int S = (int)TM::size();
  const int rank = (int)TM::rank();
  const Rows<T> t(a.l, rank);
  const int N = a.l.N, V = a.l.V, stride = (int)gridDim.x / S, first_row = (int)blockIdx.x / S;
  Pipe<T> pipe{reinterpret_cast<uint4 *>(s_dyn), a.l.stages, a.l.chunks, s_full, &s_abort, a.err};
  // the row's entries: token (-1: padding), its q and logit, and the mass of
  // the token an entry stands for (-1 if it stands for none)
  float *s_entry = reinterpret_cast<float *>(s_dyn + (size_t)a.l.stages * a.l.chunks * 16);
  auto counts = [&](int n) { return !a.weight || a.weight[n] != 0.0f; };
  if (tid == 0) {
    pipe.init();
    for (int i = 0; i < a.l.stages; i++)
      if (first_row + i * stride < N) pipe.issue(t, first_row + i * stride, i, counts(first_row + i * stride));
  }
  TM::sync();
  for (int n = first_row, flip = 0; n < N; n += stride, flip ^= 1) {
    const Share<T> sh(t, n);
    const Chunks<T> &r = sh.r;
    const Chunks<T> o(static_cast<const T *>(a.dz) + (a.dz ? (size_t)n * a.ldd : 0), V);
    const float w = a.weight ? a.weight[n] : 1.0f;
    const int cnt = sh.cnt, ahead = n + a.l.stages * stride;
    const bool next_counts = tid == 0 && ahead < N && counts(ahead);
    uint4 *st = pipe.stage();
    int *s_id = reinterpret_cast<int *>(s_entry) + flip * 4 * a.K;
    float *s_q = s_entry + flip * 4 * a.K + a.K, *s_z = s_q + a.K, *s_qv = s_z + a.K;
    auto store = [&](int c, const float (&f)[EV]) {
      if (o.mis == r.mis && c >= r.full0 && c < r.full1) {
        o.base[c] = Elem<T>::pack(f);
      } else {
        const int v = r.first(c);
#pragma unroll
        for (int e = 0; e < EV; e++)
          if (v + e >= 0 && v + e < V) o.row[v + e] = Elem<T>::from_f(f[e]);
      }
    };
    if (w == 0.0f) {                             // a row that does not count is not read
      if (a.dz) {
        const float f[EV] = {};
        for (int i = tid; i < cnt; i += TH) store(sh.c0 + i, f);
      }
      if (rank == 0 && tid == 0) {
        if (a.loss) a.loss[n] = 0.0f;
        if (a.loss64) a.loss64[n] = 0.0;
      }
      tc::mbar_wait(tc::smem_u32(&s_full[pipe.at]), pipe.phase, &s_abort, a.err, ERR_COPY);
      TM::sync();
      if (tid == 0 && ahead < N) pipe.issue(t, ahead, pipe.at, next_counts);
      pipe.next();
      continue;
    }
    // ---- the teacher's entries, by the first warp of every block
    if (warp == 0) {
      int id[KL];
      float tv[KL], tm = -FLT_MAX;
#pragma unroll
      for (int k = 0; k < KL; k++) {
        const int j = k * 32 + lane;
        id[k] = -1;
        tv[k] = -INFINITY;
        if (j < a.K) {
          id[k] = a.t_ids[(size_t)n * a.K + j];
          tv[k] = a.t_vals[(size_t)n * a.K + j];
        }
      }
      float zk[KL];
#pragma unroll
      for (int k = 0; k < KL; k++) {
        if ((unsigned)id[k] >= (unsigned)V) {
          if (id[k] != -1) atomicExch(a.err, ERR_TOKEN);
          id[k] = -1;
          tv[k] = -INFINITY;
        }
        zk[k] = id[k] >= 0 ? Elem<T>::to_f(r.row[id[k]]) : -INFINITY;
        tm = fmaxf(tm, tv[k]);
      }
      if (!TAIL) tm = warp_max(tm);
      float q[KL], sum = 0.0f;
#pragma unroll
      for (int k = 0; k < KL; k++) {
        q[k] = id[k] < 0 ? 0.0f : expf(TAIL ? tv[k] : (tv[k] - tm) * a.inv_t);
        sum += q[k];
      }
      sum = warp_sum(sum);
      const float inv = TAIL ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int k = 0; k < KL; k++) {
        const int j = k * 32 + lane;
        if (j < a.K) {
          s_id[j] = id[k];
          s_q[j] = s_qv[j] = q[k] * inv;
          s_z[j] = zk[k];
        }
      }
      __syncwarp();
      // entries naming one token add up; the first of them stands for it
#pragma unroll
      for (int k = 0; k < KL; k++) {
        const int j = k * 32 + lane;
        if (k * 32 < a.K) {
          bool again = false;
          for (int i = 0; i < a.K; i++) again |= s_id[i] == id[k] && i != j;
          if (id[k] < 0) {
            if (j < a.K) s_qv[j] = -1.0f;
          } else if (again) {
            float qv = 0.0f;
            bool first = true;
            for (int i = 0; i < a.K; i++)
              if (s_id[i] == id[k]) {
                qv += s_q[i];
                first = first && i >= j;
              }
            s_qv[j] = first ? qv : -1.0f;
          }
        }
      }
      if (lane == 0) {
        float Q = TAIL || sum == 0.0f ? sum : 1.0f;
        if (!(sum < INFINITY)) Q = NAN;          // a NaN or +inf among the values
        const float qr = TAIL ? 1.0f - Q : 0.0f;
        s_sum[flip][0] = Q;
        s_sum[flip][1] = qr < TAIL_MIN ? 0.0f : qr;            // NaN stays
      }
      if (TAIL) {
        pipe.wait(t, sh);
#pragma unroll
        for (int k = 0; k < KL; k++) {
          const int at = id[k] + r.mis - sh.c0 * EV;           // element of the share
          if (id[k] >= 0 && at >= 0 && at < cnt * EV) reinterpret_cast<T *>(st)[at] = Elem<T>::none();
        }
        tc::fence_proxy_async();                 // a later copy into this stage comes after these writes
      }
    }
    if (!TAIL || warp != 0) pipe.wait(t, sh);
    if (TAIL) __syncthreads();
    // ---- the row's statistics (with a tail: those of the tokens not named)
    Part p = warp_part<T, false>(st, cnt, thread_max<T>(st, cnt), a.c);
    if (lane == 0) s_part[flip][warp] = p;
    if (CL) meet<false>(s_part[flip], s_from[flip], 0, a.c);
    else __syncthreads();
    p = join_all<false>(CL ? s_from[flip] : s_part[flip], CL ? S : TH >> 5, a.c);
    const float Q = s_sum[flip][0], qr = s_sum[flip][1];
    float m = p.m, all = p.s, f = 1.0f;          // e of the row is relative to p.m, times f to m
    if (TAIL) {
      for (int j = lane; j < a.K; j += 32) m = fmaxf(m, s_z[j]);
      m = warp_max(m);
      float named = 0.0f;
      for (int j = lane; j < a.K; j += 32)
        if (!(s_qv[j] < 0.0f)) named += exp2_fast((s_z[j] - m) * a.c);
      f = exp2_fast(bounded((p.m - m) * a.c));
      all = fmaf(p.s, f, warp_sum(named));
    }
    const float total = Q + qr;
    if (rank == 0 && warp == 0 && (a.loss || a.loss64)) {
      const float ls = logf(all);
      float L = 0.0f;
      for (int j = lane; j < a.K; j += 32) {
        const float qv = s_qv[j];
        if (qv > 0.0f) L += qv * (logf(qv) - ((s_z[j] - m) * a.inv_t - ls));
      }
      L = warp_sum(L);
      if (TAIL && qr > 0.0f) L += qr * (logf(qr) - (logf(p.s) + (p.m - m) * a.inv_t - ls));
      if (all == 0.0f) L = total > 0.0f ? INFINITY : 0.0f;     // a student that allows no token
      if (all != all || total != total) L = NAN;
      L *= w;
      if (lane == 0) {
        if (a.loss) a.loss[n] = L;
        if (a.loss64) a.loss64[n] = (double)L;
      }
    }
    const float g = w * a.scale * a.inv_t;
    if (a.dz) {
      const float coef =
          all == 0.0f ? 0.0f : g * (total * f / all - (TAIL && qr > 0.0f && p.s > 0.0f ? qr / p.s : 0.0f));
      const f32x2 nm2 = pack2(-p.m, -p.m), c2 = pack2(a.c, a.c), k2 = pack2(coef, coef);
#pragma unroll 4
      for (int i = tid; i < cnt; i += TH) {
        float v[EV];
        Elem<T>::unpack(st[i], v);
#pragma unroll
        for (int e = 0; e < EV; e += 2) {
          float d0, d1;
          unpack2(mul2(add2(pack2(v[e], v[e + 1]), nm2), c2), d0, d1);
          unpack2(mul2(pack2(exp2_fast(d0), exp2_fast(d1)), k2), v[e], v[e + 1]);
        }
        store(sh.c0 + i, v);
      }
    }
    __syncthreads();
    if (tid == 0 && ahead < N) pipe.issue(t, ahead, pipe.at, next_counts);
    pipe.next();
    if (!a.dz || all == 0.0f) continue;
    for (int j = tid; j < a.K; j += TH) {
      const float q = s_qv[j];
      if (q < 0.0f) continue;
      const int id = s_id[j], at = (id + r.mis) / EV;
      if (at < sh.c0 || at >= sh.c0 + cnt) continue;   // another block's
      const float pv = exp2_fast((s_z[j] - m) * a.c) / all;
      o.row[id] = Elem<T>::from_f(g * (total * pv - q));
    }
  }
  if (CL) TM::sync();                            // no block leaves while another may write to it
}

}  // namespace lg

namespace {

template <typename T, int TPR>
int launch_grad(DeviceCtx *c, int nch, const lg::GradArgs &a) {
  const int segs = (nch + TPR * lg::CPT - 1) / (TPR * lg::CPT);
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
  if (nch <= 32 * lg::CPT) return launch_grad<T, 32>(c, nch, a);
  if (nch <= 128 * lg::CPT) return launch_grad<T, 128>(c, nch, a);
  return launch_grad<T, 256>(c, nch, a);
}

template <typename T, bool CL, bool TAIL> int launch_distill(DeviceCtx *c, const RowPlan &pl, lg::DistillArgs a) {
  static Resident seen[kMaxDevices];
  return launch_rows((const void *)lg::distill_kernel<T, CL, TAIL>, c, pl, 32 * a.K, &seen[c->device], &a);
}
template <typename T> int distill_typed(DeviceCtx *c, const RowPlan &pl, const lg::DistillArgs &a, bool tail) {
  if (pl.blocks > 1) return tail ? launch_distill<T, true, true>(c, pl, a) : launch_distill<T, true, false>(c, pl, a);
  return tail ? launch_distill<T, false, true>(c, pl, a) : launch_distill<T, false, false>(c, pl, a);
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
  const RowPlan pl = plan_rows(c, z, 0);
  const lg::DistillArgs a{pl.l, t_ids, t_vals, K, lg::LOG2E / temperature, 1.0f / temperature, weight, scale, loss,
                          loss64, dlogits, ldd, c->err_flag};
  if (z.dtype == TL_F32) return distill_typed<float>(c, pl, a, tail);
  if (z.dtype == TL_BF16) return distill_typed<__nv_bfloat16>(c, pl, a, tail);
  return distill_typed<__half>(c, pl, a, tail);
}

}  // namespace tl
