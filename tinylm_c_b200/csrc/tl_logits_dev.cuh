// tl_logits_dev.cuh -- device pieces shared by the vocabulary-row kernels: a
// row's slice held in registers, the softmax statistics, the exchange between
// the blocks of a row.
//
// A row is held as 16-byte chunks of memory, counted from the aligned address
// at or below its start, so a row of any element alignment is loaded and
// stored 16 bytes at a time; only the (at most two) chunks that reach past
// the row's ends go element by element.  A row is owned by one block, or by
// the blocks of one cluster, each with a contiguous range of chunks; thread t
// of TH holds chunks t, t + TH, ... of its block's range, NV of them.
#pragma once
#include <cfloat>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tl_logits.cuh"

namespace tl {
namespace lg {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int MAX_CLUSTER = 16;
// Chunks held by one thread.
constexpr int NV = 8;

// ------------------------------------------------------------- arithmetic
// Two fp32 operations in one instruction (sm_100's packed pairs), each
// rounded as the single one is.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// 2^x, relative error 2^-22; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// max(x, -1e30), NaN kept: an exponent whose power is 0 anyway, made finite so
// that power times exponent is 0 and not NaN.
__device__ __forceinline__ float bounded(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-1e30f));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// ------------------------------------------------------------ element types
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int EV = 4;                       // elements of a chunk
  static constexpr unsigned FILL = 0xFF800000u;      // -inf in every element
  static __device__ __forceinline__ float to_f(float x) { return x; }
  static __device__ __forceinline__ float from_f(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4 &c, float (&f)[EV]) {
    f[0] = __uint_as_float(c.x); f[1] = __uint_as_float(c.y);
    f[2] = __uint_as_float(c.z); f[3] = __uint_as_float(c.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[EV]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  // NaN counts as the smallest, in every type: it shows in the sums.
  static __device__ __forceinline__ float max_of(const uint4 &c) {
    float f[EV];
    unpack(c, f);
    return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  }
  static __device__ __forceinline__ unsigned bits(float x) { return __float_as_uint(x); }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr int EV = 8;
  static constexpr unsigned FILL = 0xFF80FF80u;
  static __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4 &c, float (&f)[EV]) {
    const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[EV]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned *>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float max_of(const uint4 &c) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&c);
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ unsigned bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
};
template <> struct Elem<__half> {
  static constexpr int EV = 8;
  static constexpr unsigned FILL = 0xFC00FC00u;
  static __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4 &c, float (&f)[EV]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&c);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 p = __half22float2(h[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[EV]) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned *>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float max_of(const uint4 &c) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&c);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ unsigned bits(__half x) { return __half_as_ushort(x); }
};

// ------------------------------------------------------------------- rows
// One row's chunks.  Chunk c holds elements c*EV - mis ... of the row; chunks
// [full0, full1) lie inside it, the others reach past an end.
template <typename T> struct Chunks {
  static constexpr int EV = Elem<T>::EV;
  T *row;
  uint4 *base;
  int mis, n, full0, full1, V;
  __device__ __forceinline__ Chunks(const T *p, int V_) : row(const_cast<T *>(p)), V(V_) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    mis = (int)(a & 15) / (int)sizeof(T);
    base = reinterpret_cast<uint4 *>(a & ~(uintptr_t)15);
    n = (V + mis + EV - 1) / EV;
    full0 = mis ? 1 : 0;
    full1 = (V + mis) / EV;
  }
  __device__ __forceinline__ int first(int c) const { return c * EV - mis; }
  // A chunk that reaches past an end: the elements inside, -inf elsewhere.
  __device__ __forceinline__ uint4 load_edge(int c) const {
    const int v = first(c);
    unsigned w[4] = {Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL};
#pragma unroll
    for (int e = 0; e < EV; e++)
      if (v + e >= 0 && v + e < V) {
        const unsigned b = Elem<T>::bits(row[v + e]);
        if (EV == 4) w[e & 3] = b;
        else w[(e >> 1) & 3] = e & 1 ? (w[(e >> 1) & 3] & 0x0000FFFFu) | (b << 16) : (w[(e >> 1) & 3] & 0xFFFF0000u) | b;
      }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void store_each(int c, const float (&f)[EV]) const {
    const int v = first(c);
#pragma unroll
    for (int e = 0; e < EV; e++)
      if (v + e >= 0 && v + e < V) row[v + e] = Elem<T>::from_f(f[e]);
  }
};

// This thread's chunks of [c0, c1): all loads in flight together.
template <typename T, int TH>
__device__ __forceinline__ void load_slice(const Chunks<T> &r, int c0, int c1, uint4 (&x)[NV]) {
  const int lo = max(c0, r.full0), hi = min(c1, r.full1), t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < NV; i++) {
    const int c = c0 + i * TH + t;
    x[i] = make_uint4(Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL);
    if (c >= lo && c < hi) x[i] = __ldcg(r.base + c);
  }
  // the row's first and last chunk, where they reach past it
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int c = k ? r.n - 1 : 0;
    const bool reaches = k ? r.full1 < r.n && (r.n > 1 || r.full0 == 0) : r.full0 == 1;
    if (reaches && c >= c0 && c < c1 && (c - c0) % TH == t) {
      const uint4 v = r.load_edge(c);
      const int at = (c - c0) / TH;
#pragma unroll
      for (int i = 0; i < NV; i++)
        if (i == at) x[i] = v;
    }
  }
}

// ------------------------------------------------- statistics and exchange
// Of a part of a row: m its largest logit (at least -FLT_MAX), s the sum of
// e = 2^((z - m) c) and t that of e (z - m) c, c = log2(e) / temperature; w is
// free for the caller.
struct Part {
  float m, s, t, w;
};
__device__ __forceinline__ Part no_part(float w) { return Part{-FLT_MAX, 0.0f, 0.0f, w}; }
// The parts of lanes 0..15 as one; every lane of both halves gets the same
// bits (each step adds the same two values on both sides).
template <bool ENT> __device__ __forceinline__ Part join_lanes(Part p, float c) {
  float m = p.m;
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    p.w = fminf(p.w, __shfl_xor_sync(FULL, p.w, o));
  }
  const float d = bounded((p.m - m) * c), f = exp2_fast(d);
  if (ENT) p.t = f * (p.t + p.s * d);
  p.s *= f;
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    p.s += __shfl_xor_sync(FULL, p.s, o);
    if (ENT) p.t += __shfl_xor_sync(FULL, p.t, o);
  }
  p.m = m;
  return p;
}

// A warp's part of the row from its lanes' chunks; `lane_max` is this lane's
// largest logit (-inf if it has none).  cnt: chunks of the block's range.
template <typename T, int TH, bool ENT>
__device__ __forceinline__ Part warp_part(const uint4 (&x)[NV], int cnt, float lane_max, float c) {
  constexpr int EV = Elem<T>::EV;
  const float m = fmaxf(warp_max(lane_max), -FLT_MAX);
  const f32x2 nm = pack2(-m, -m), cc = pack2(c, c);
  f32x2 s2 = pack2(0.0f, 0.0f), t2 = s2;
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (i * TH < cnt) {
      float f[EV];
      Elem<T>::unpack(x[i], f);
#pragma unroll
      for (int e = 0; e < EV; e += 2) {
        f32x2 d = mul2(add2(pack2(f[e], f[e + 1]), nm), cc);
        float d0, d1;
        unpack2(d, d0, d1);
        const f32x2 ex = pack2(exp2_fast(d0), exp2_fast(d1));
        s2 = add2(s2, ex);
        if (ENT) t2 = fma2(ex, pack2(bounded(d0), bounded(d1)), t2);
      }
    }
  float a, b;
  unpack2(s2, a, b);
  Part p;
  p.m = m;
  p.s = warp_sum(a + b);
  unpack2(t2, a, b);
  p.t = ENT ? warp_sum(a + b) : 0.0f;
  p.w = 0.0f;
  return p;
}
template <typename T, int TH>
__device__ __forceinline__ float lane_max_of(const uint4 (&x)[NV], int cnt) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; i++)
    if (i * TH < cnt) m = fmaxf(m, Elem<T>::max_of(x[i]));
  return m;
}

// The blocks of a row.  One block: barriers are the block's and no memory is
// mapped.  A cluster: `arrive` then `wait` is a barrier of all its threads.
template <bool CL> struct Team;
template <> struct Team<false> {
  static __device__ __forceinline__ unsigned rank() { return 0; }
  static __device__ __forceinline__ unsigned size() { return 1; }
  static __device__ __forceinline__ void arrive() {}
  static __device__ __forceinline__ void wait() {}
  static __device__ __forceinline__ void sync() { __syncthreads(); }
  template <typename P> static __device__ __forceinline__ P *at(P *p, unsigned) { return p; }
};
template <> struct Team<true> {
  static __device__ __forceinline__ unsigned rank() { return cg::this_cluster().block_rank(); }
  static __device__ __forceinline__ unsigned size() { return cg::this_cluster().num_blocks(); }
  static __device__ __forceinline__ void arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
  static __device__ __forceinline__ void wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
  static __device__ __forceinline__ void sync() { arrive(); wait(); }
  template <typename P> static __device__ __forceinline__ P *at(P *p, unsigned r) {
    return cg::this_cluster().map_shared_rank(p, r);
  }
};

// Every warp's part (in part[], written by its lane 0) joined over the row's
// blocks; every thread gets the same result.  `none` is w where there is no
// part.  The cluster's blocks have arrived at its first barrier before
// (Team::arrive), which is waited for here: memory of a block that has not
// started is not written.
template <bool CL, int W, bool ENT>
__device__ __forceinline__ Part join_row(const Part *part, Part *from, float none, float c) {
  using TM = Team<CL>;
  const int lane = threadIdx.x & 15;
  __syncthreads();
  if (!CL) return W == 1 ? part[0] : join_lanes<ENT>(lane < W ? part[lane] : no_part(none), c);
  TM::wait();
  if (threadIdx.x < 32) {
    const Part p = join_lanes<ENT>(lane < W ? part[lane] : no_part(none), c);
    if (threadIdx.x < TM::size()) *TM::at(&from[TM::rank()], threadIdx.x) = p;
  }
  TM::sync();
  return join_lanes<ENT>(lane < (int)TM::size() ? from[lane] : no_part(none), c);
}

}  // namespace lg

// ------------------------------------------------------------ launch plan
// How a row is laid over the GPU: `threads` a block, `blocks` a row (more than
// one: a cluster).
struct RowPlan {
  int threads, blocks;
};
RowPlan plan_rows(const DeviceCtx *c, const LogitRows &z, int K);
// Launches N clusters of `blocks` blocks; `args` is the kernel's one argument.
int launch_rows_cluster(const void *kernel, DeviceCtx *c, int N, int threads, int blocks, void *args);

}  // namespace tl
