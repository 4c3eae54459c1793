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
    if (c0 == 0) atomicExch(a.err, 100);
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
  const void *z;
  long long ld;
  const int *t_ids;
  const float *t_vals;
  int K, V;
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
// The row is loaded once and stays in registers; with a tail the named tokens
// are taken out of it first (a bit for each element of the block's slice), so
// that p_r is summed and never 1 - sum p, which loses all its digits for a
// confident student.  All others' gradients are then one factor times e_v;
// the named tokens' are written over them at the end.
template <typename T, int TH, bool CL, bool TAIL>
__global__ void __launch_bounds__(TH, 1024 / TH) distill_kernel(const DistillArgs a) {
  using TM = Team<CL>;
  constexpr int W = TH / 32, EV = Elem<T>::EV, KL = TL_TOPK_MAX / 32;
  __shared__ Part s_part[W], s_from[MAX_CLUSTER];
  __shared__ int s_id[TL_TOPK_MAX];              // -1: padding
  __shared__ float s_q[TL_TOPK_MAX], s_z[TL_TOPK_MAX];
  __shared__ float s_qv[TL_TOPK_MAX];            // mass of the token an entry stands for, -1 if it stands for none
  __shared__ float s_sum[2];                     // sum of q, the tail
  __shared__ __align__(8) unsigned char s_named[TAIL ? TH * NV : 8];   // a bit an element, a byte a chunk
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = TM::rank(), S = TM::size();
  const size_t n = CL ? blockIdx.x / S : blockIdx.x;
  const Chunks<T> r(static_cast<const T *>(a.z) + n * a.ld, a.V);
  const int per = CL ? (r.n + (int)S - 1) / (int)S : r.n;
  const int c0 = (int)rank * per, c1 = min(r.n, c0 + per), cnt = c1 - c0;
  const Chunks<T> o(static_cast<const T *>(a.dz) + (a.dz ? n * a.ldd : 0), a.V);
  const float w = a.weight ? a.weight[n] : 1.0f;
  const bool same = o.mis == r.mis;
  auto store = [&](int c, const float (&f)[EV]) {
    if (same && c >= r.full0 && c < r.full1) {
      o.base[c] = Elem<T>::pack(f);
    } else {
      const int v = r.first(c);
#pragma unroll
      for (int e = 0; e < EV; e++)
        if (v + e >= 0 && v + e < a.V) o.row[v + e] = Elem<T>::from_f(f[e]);
    }
  };
  if (w == 0.0f) {                               // a row that does not count is not read
    if (a.dz) {
      const float f[EV] = {};
      for (int c = c0 + tid; c < c1; c += TH) store(c, f);
    }
    if (rank == 0 && tid == 0) {
      if (a.loss) a.loss[n] = 0.0f;
      if (a.loss64) a.loss64[n] = 0.0;
    }
    return;
  }
  TM::arrive();
  uint4 x[NV];
  load_slice<T, TH>(r, c0, c1, x);
  if (TAIL) {
    *reinterpret_cast<uint2 *>(&s_named[tid * NV]) = make_uint2(0, 0);
    __syncthreads();
  }
  // ---- the teacher's entries, by the first warp of every block
  if (warp == 0) {
    int id[KL];
    float t[KL], tm = -FLT_MAX;
#pragma unroll
    for (int k = 0; k < KL; k++) {
      const int j = k * 32 + lane;
      id[k] = -1;
      t[k] = -INFINITY;
      if (j < a.K) {
        id[k] = a.t_ids[n * a.K + j];
        t[k] = a.t_vals[n * a.K + j];
      }
    }
    float z[KL];
#pragma unroll
    for (int k = 0; k < KL; k++) {
      const int j = k * 32 + lane;
      if ((unsigned)id[k] >= (unsigned)a.V) {
        if (id[k] != -1) atomicExch(a.err, 100);
        id[k] = -1;
        t[k] = -INFINITY;
      }
      z[k] = -INFINITY;
      if (id[k] >= 0) {
        z[k] = Elem<T>::to_f(r.row[id[k]]);
        if (TAIL) {
          const int at = (id[k] + r.mis) / EV - c0, e = (id[k] + r.mis) % EV;
          if (at >= 0 && at < cnt)
            atomicOr(reinterpret_cast<unsigned *>(s_named) + (at >> 2), 1u << ((at & 3) * 8 + e));
        }
      }
      if (j < a.K) s_id[j] = id[k];
      tm = fmaxf(tm, t[k]);
    }
    if (!TAIL) tm = warp_max(tm);
    float q[KL], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < KL; k++) {
      q[k] = id[k] < 0 ? 0.0f : expf(TAIL ? t[k] : (t[k] - tm) * a.inv_t);
      sum += q[k];
    }
    sum = warp_sum(sum);
    const float inv = TAIL ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < KL; k++) {
      const int j = k * 32 + lane;
      if (j < a.K) {
        s_q[j] = q[k] * inv;
        s_z[j] = z[k];
      }
    }
    if (lane == 0) {
      float Q = TAIL || sum == 0.0f ? sum : 1.0f;
      if (!(sum < INFINITY)) Q = NAN;            // a NaN or +inf among the values
      const float qr = TAIL ? 1.0f - Q : 0.0f;
      s_sum[0] = Q;
      s_sum[1] = qr < TAIL_MIN ? 0.0f : qr;      // NaN stays
    }
  }
  if (TAIL) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const unsigned named = s_named[i * TH + tid];
      if (named) {
        unsigned u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int e = 0; e < EV; e++)
          if (named >> e & 1) {
            if (EV == 4) u[e & 3] = Elem<T>::FILL;
            else u[(e >> 1) & 3] = e & 1 ? (u[(e >> 1) & 3] & 0x0000FFFFu) | (Elem<T>::FILL & 0xFFFF0000u)
                                         : (u[(e >> 1) & 3] & 0xFFFF0000u) | (Elem<T>::FILL & 0x0000FFFFu);
          }
        x[i] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
  // ---- the row's statistics (with a tail: those of the tokens not named)
  Part p = warp_part<T, TH, false>(x, cnt, lane_max_of<T, TH>(x, cnt), a.c);
  if (lane == 0) s_part[warp] = p;
  __syncthreads();
  // entries naming one token add up; the first of them stands for it
  for (int j = tid; j < a.K; j += TH) {
    const int id = s_id[j];
    float qv = 0.0f;
    bool first = id >= 0;
    for (int i = 0; i < a.K; i++)
      if (s_id[i] == id) {
        qv += s_q[i];
        first = first && i >= j;
      }
    s_qv[j] = first ? qv : -1.0f;
  }
  p = join_row<CL, W, false>(s_part, s_from, 0.0f, a.c);
  const float Q = s_sum[0], qr = s_sum[1];
  float m = p.m, all = p.s, f = 1.0f;            // e of the row is relative to p.m, times f to m
  float qv[KL], zj[KL];
#pragma unroll
  for (int k = 0; k < KL; k++) {
    const int j = k * 32 + lane;
    qv[k] = j < a.K ? s_qv[j] : -1.0f;
    zj[k] = j < a.K ? s_z[j] : -INFINITY;
  }
  if (TAIL) {
#pragma unroll
    for (int k = 0; k < KL; k++) m = fmaxf(m, zj[k]);
    m = warp_max(m);
    float named = 0.0f;
#pragma unroll
    for (int k = 0; k < KL; k++)
      if (!(qv[k] < 0.0f)) named += exp2_fast((zj[k] - m) * a.c);
    f = exp2_fast(bounded((p.m - m) * a.c));
    all = fmaf(p.s, f, warp_sum(named));
  }
  const float ls = logf(all);
  const float total = Q + qr;
  if (rank == 0 && warp == 0 && (a.loss || a.loss64)) {
    float L = 0.0f;
#pragma unroll
    for (int k = 0; k < KL; k++)
      if (qv[k] > 0.0f) L += qv[k] * (logf(qv[k]) - ((zj[k] - m) * a.inv_t - ls));
    L = warp_sum(L);
    if (TAIL && qr > 0.0f) L += qr * (logf(qr) - (logf(p.s) + (p.m - m) * a.inv_t - ls));
    if (all == 0.0f) L = total > 0.0f ? INFINITY : 0.0f;       // a student that allows no token
    if (all != all || total != total) L = NAN;
    L *= w;
    if (lane == 0) {
      if (a.loss) a.loss[n] = L;
      if (a.loss64) a.loss64[n] = (double)L;
    }
  }
  if (!a.dz) return;
  const float g = w * a.scale * a.inv_t;
  const float coef = all == 0.0f ? 0.0f : g * (total * f / all - (TAIL && qr > 0.0f && p.s > 0.0f ? qr / p.s : 0.0f));
  const f32x2 nm2 = pack2(-p.m, -p.m), c2 = pack2(a.c, a.c), k2 = pack2(coef, coef);
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = c0 + i * TH + tid;
    if (c >= c1) break;
    float v[EV];
    Elem<T>::unpack(x[i], v);
#pragma unroll
    for (int e = 0; e < EV; e += 2) {
      float d0, d1;
      unpack2(mul2(add2(pack2(v[e], v[e + 1]), nm2), c2), d0, d1);
      unpack2(mul2(pack2(exp2_fast(d0), exp2_fast(d1)), k2), v[e], v[e + 1]);
    }
    store(c, v);
  }
  if (all == 0.0f) return;
  __syncthreads();
  for (int j = tid; j < a.K; j += TH) {
    const float q = s_qv[j];
    if (q < 0.0f) continue;
    const int id = s_id[j], at = (id + r.mis) / EV;
    if (at < c0 || at >= c1) continue;           // another block's
    const float pv = exp2_fast((s_z[j] - m) * a.c) / all;
    o.row[id] = Elem<T>::from_f(g * (total * pv - q));
  }
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

template <typename T, int TH, bool CL, bool TAIL>
int launch_distill(DeviceCtx *c, int N, int S, const lg::DistillArgs &a) {
  if constexpr (!CL) {
    lg::distill_kernel<T, TH, false, TAIL><<<N, TH, 0, c->stream>>>(a);
    TL_TRY_CUDA(cudaGetLastError());
    return TL_OK;
  } else {
    return launch_rows_cluster((const void *)lg::distill_kernel<T, TH, true, TAIL>, c, N, TH, S, const_cast<void *>(static_cast<const void *>(&a)));
  }
}
template <typename T, bool TAIL> int distill_typed(DeviceCtx *c, int N, const RowPlan &pl, const lg::DistillArgs &a) {
  if (pl.blocks > 1)
    return pl.threads == 256 ? launch_distill<T, 256, true, TAIL>(c, N, pl.blocks, a)
                             : launch_distill<T, 512, true, TAIL>(c, N, pl.blocks, a);
  switch (pl.threads) {
    case 32: return launch_distill<T, 32, false, TAIL>(c, N, 1, a);
    case 128: return launch_distill<T, 128, false, TAIL>(c, N, 1, a);
    case 256: return launch_distill<T, 256, false, TAIL>(c, N, 1, a);
    default: return launch_distill<T, 512, false, TAIL>(c, N, 1, a);
  }
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
  const lg::DistillArgs a{z.p, z.ld, t_ids, t_vals, K, z.V, lg::LOG2E / temperature, 1.0f / temperature, weight,
                          scale, loss, loss64, dlogits, ldd, c->err_flag};
  if (z.dtype == TL_F32) return tail ? distill_typed<float, true>(c, z.N, pl, a) : distill_typed<float, false>(c, z.N, pl, a);
  if (z.dtype == TL_BF16)
    return tail ? distill_typed<__nv_bfloat16, true>(c, z.N, pl, a) : distill_typed<__nv_bfloat16, false>(c, z.N, pl, a);
  return tail ? distill_typed<__half, true>(c, z.N, pl, a) : distill_typed<__half, false>(c, z.N, pl, a);
}

}  // namespace tl
