// tl_logits_dev.cuh -- device pieces shared by the vocabulary-row kernels: a
// row's share in shared memory, the softmax statistics, the exchange between
// the blocks of a row.
//
// A row is handled as 16-byte chunks of memory, counted from the aligned
// address at or below its start, so a row of any element alignment is moved 16
// bytes at a time; elements of a neighbouring row in its first and last chunk
// are set to -inf once they are in shared memory, and only chunks that reach
// past the whole tensor go element by element.  A row is owned by one block,
// or by the blocks of one cluster, each with a contiguous share of its chunks.
// The blocks stay on the GPU and take rows in turn; while one row is worked on
// the share of the next is on its way by a bulk copy into another stage of
// shared memory, so the memory system is busy throughout.  A row is read from
// memory once, however often a kernel goes over it, but for distilled rows of
// several pieces (distill_kernel).
#pragma once
#include <cfloat>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tl_logits.cuh"
#include "tl_tc_ptx.cuh"

namespace tl {
namespace lg {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int MAX_CLUSTER = 16;
constexpr int MAX_WARPS = 16, MAX_STAGES = 4;
// Blocks of TH threads an SM holds at least: 64 registers a thread.
constexpr int min_blocks(int TH) { return 1024 / TH; }
constexpr int ERR_COPY = 90;                       // error word: a bulk copy did not arrive in time
constexpr int ERR_TOKEN = 100;                     // a token id outside [0, V)
// The error word keeps an expired wait, whose results are lost: a token that is
// taken as none does not replace it.
__device__ __forceinline__ void report_token(int *err) { atomicCAS(err, 0, ERR_TOKEN); }

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
// max(x, LEAST), NaN kept: an exponent whose power is 0 anyway, made finite so
// that power times exponent is 0 and not NaN.  -1e30 is below every difference
// of logits that counts; where the exponent meets a factor of the caller's
// first, -256 leaves that room (fp32 powers end at 2^-126).
template <int LEAST = 0> __device__ __forceinline__ float bounded(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(LEAST ? (float)LEAST : -1e30f));
  return r;
}
// The warp's largest value (NaN only if all are).
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// What L2 should do with the lines of a copy: let them go first, keep them, or
// nothing special.
__device__ __forceinline__ uint64_t l2_once() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_again() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_normal() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// 16 bytes of shared memory at a 32-bit address.
__device__ __forceinline__ uint4 lds(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

// A barrier of the TH computing threads of a block that has other warps too.
template <int TH> __device__ __forceinline__ void bar_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(TH) : "memory");
}
// The same, and whether any of the threads says so.
template <int TH> __device__ __forceinline__ bool bar_any(bool x) {
  uint32_t r;
  asm volatile(
      "{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 1, %2, p; selp.u32 %0, 1, 0, q; }"
      : "=r"(r)
      : "r"((uint32_t)x), "n"(TH)
      : "memory");
  return r != 0;
}

// ------------------------------------------------------------ element types
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int EV = 4;                       // elements of a chunk
  static constexpr unsigned FILL = 0xFF800000u;      // -inf in every element
  static __device__ __forceinline__ float none() { return __uint_as_float(FILL); }
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
  static __device__ __forceinline__ __nv_bfloat16 none() { return __ushort_as_bfloat16(0xFF80); }
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
  static __device__ __forceinline__ __half none() { return __ushort_as_half(0xFC00); }
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
};

// The tensor's rows and how they are cut up, as the host lays it out: into
// pieces of `per` chunks, one for each block of a row's cluster or, one after
// another, for the one block that has the row (`pieces` of them, the last with
// what is left); each block has `stages` buffers of `chunks` >= per chunks.
// `ragged`: some row's ends do not fill their chunks.
struct Layout {
  const void *z;
  long long ld;
  int N, V, per, pieces, stages, chunks, ragged;
  unsigned wait_ns;                    // how long a wait lasts at most
};
template <typename T> struct Rows {
  const T *z;
  long long ld;
  int V, per;
  uintptr_t end;                       // one past the last row
  bool ragged;
  __device__ __forceinline__ explicit Rows(const Layout &l)
      : z(static_cast<const T *>(l.z)), ld(l.ld), V(l.V), per(l.per),
        end(reinterpret_cast<uintptr_t>(z + ((long long)(l.N - 1) * ld + V))), ragged(l.ragged) {}
  __device__ __forceinline__ Chunks<T> row(int n) const { return Chunks<T>(z + (size_t)n * ld, V); }
  // Whether a chunk lies inside the tensor as a whole, so that it may be copied.
  __device__ __forceinline__ bool inside(const uint4 *p) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return a >= reinterpret_cast<uintptr_t>(z) && a + 16 <= end;
  }
};
// A piece of a row: chunks [c0, c0 + cnt), in shared memory from 0.
template <typename T> struct Piece {
  Chunks<T> r;
  int c0, cnt;
  __device__ __forceinline__ Piece(const Rows<T> &t, int n, int i) : r(t.row(n)), c0(i * t.per) {
    cnt = max(0, min(r.n - c0, t.per));
  }
  // The copied elements of other rows in the row's first and last chunk set
  // to -inf, by the thread for whom `mine(chunk of the piece)`.
  template <typename F> __device__ __forceinline__ void mask_ends(uint4 *st, F &&mine) const {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int c = k ? r.n - 1 : 0;
      const bool partial = k ? r.full1 < r.n && (r.n > 1 || r.full0 == 0) : r.full0 == 1;
      if (partial && c >= c0 && c < c0 + cnt && mine(c - c0)) {
        T *e = reinterpret_cast<T *>(st + (c - c0));
        const int v = r.first(c);
        for (int i = 0; i < Elem<T>::EV; i++)
          if (v + i < 0 || v + i >= r.V) e[i] = Elem<T>::none();
        tc::fence_proxy_async();       // a later copy into this stage comes after these writes
      }
    }
  }
};

// The stages of a block and their barriers.
//
// Every wait ends: after `wait_ns` it sets the block's abort flag and the error
// word, and from then on all waits that are not met at once fail and nothing is
// copied any more.  A warp whose wait failed goes by nothing that the wait was
// to protect: in the one-block kernels it leaves its loop without arriving
// anywhere, so that the others' order holds until their own waits fail, and
// the computing warps, which have a barrier without a time limit in common,
// carry the failure to that barrier and leave together.  A cluster's blocks
// meet whatever happened and run over the rows left, which are addressed by
// what does not come from a copy.  Whoever issues copies drains them before it
// leaves: shared memory that a copy is still to write is given up by no block.
template <typename T> struct Pipe {
  uint4 *buf;                          // stage 0
  int stages, stage_chunks;
  unsigned wait_ns;
  int *abort_flag;                     // a wait ran out: nothing is waited for or copied any more
  int *err;
  __device__ __forceinline__ Pipe(void *buf_, const Layout &l, int stages_, int *abort_flag_, int *err_)
      : buf(static_cast<uint4 *>(buf_)), stages(stages_), stage_chunks(l.chunks), wait_ns(l.wait_ns),
        abort_flag(abort_flag_), err(err_) {}
  __device__ __forceinline__ uint4 *stage(int s) const { return buf + (size_t)s * stage_chunks; }
  // Piece p into stage s (`read` false: nothing is copied, the stage is full
  // at once), by one thread; barrier `arrived` completes a phase when it is
  // there.  The stage's earlier readers are done.  The tensor's first and last
  // chunk, where it does not fill them, are written by the calling thread.
  // False after an expired wait.
  __device__ __forceinline__ bool issue(const Rows<T> &t, int n, int piece, int s, uint64_t *arrived, bool read,
                                        uint64_t policy) const {
    const uint32_t bar = tc::smem_u32(arrived);
    if (*(volatile int *)abort_flag) return false;
    int lo = 0, hi = 0;
    const uint4 *from = nullptr;
    uint4 *st = stage(s);
    // what other threads read and wrote of the stage comes before the copy
    tc::fence_proxy_async();
    if (read) {
      const Piece<T> p(t, n, piece);
      from = p.r.base + p.c0;
      hi = p.cnt;
      if (lo < hi && !t.inside(from)) {
        st[0] = p.r.load_edge(p.c0);
        lo++;
      }
      if (lo < hi && !t.inside(from + hi - 1)) {
        hi--;
        st[hi] = p.r.load_edge(p.c0 + hi);
      }
    }
    const uint32_t bytes = (uint32_t)(hi - lo) * 16u;
    tc::mbar_arrive_expect_tx(bar, bytes);
    if (bytes)
      asm volatile(
          "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
              tc::smem_u32(st + lo)),
          "l"(__cvta_generic_to_global(from + lo)), "r"(bytes), "r"(bar), "l"(policy)
          : "memory");
    return true;
  }
  // Waits for a phase of a barrier; false where that did not come.
  __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) const {
    const uint32_t at = tc::smem_u32(bar), suspend = min(wait_ns, tc::SUSPEND_NS);
    const long long t0 = clock64();
    while (!tc::mbar_try_wait(at, parity, suspend)) {
      if (*(volatile int *)abort_flag) return false;
      if (clock64() - t0 >= 2ll * wait_ns) {     // of a clock that ends below 2 GHz
        *(volatile int *)abort_flag = 1;
        atomicExch(err, ERR_COPY);
        return false;
      }
    }
    return true;
  }
  // The same for a whole warp, which goes on together.
  __device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity) const {
    return __all_sync(FULL, wait(bar, parity));
  }
  // Waits until the copies of the latest uses of a ring of barriers are there,
  // `issued` uses in all, each for two seconds at most.
  __device__ __forceinline__ void drain(uint64_t *ring, int size, int issued) const {
    for (int u = max(0, issued - size); u < issued; u++) {
      const long long t0 = clock64();
      while (!tc::mbar_try_wait(tc::smem_u32(&ring[u % size]), (u / size) & 1))
        if (clock64() - t0 > tc::WAIT_LIMIT_CYCLES) {
          atomicExch(err, ERR_COPY);
          break;
        }
    }
  }
};
// Place and phase of the k-th use of a ring (stages, barriers).
struct Turn {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) { s = 0; phase ^= 1; }
  }
};

// ------------------------------------------------- statistics and exchange
// Of a part of a row: m its largest logit (at least -FLT_MAX), s the sum of
// e = 2^((z - m) c) and t that of e (z - m) c, c = log2(e) / temperature; w a
// value of which the part's elements hold at least some known number of larger
// ones (-inf: none known).
struct Part {
  float m, s, t, w;
};
__device__ __forceinline__ Part no_part() { return Part{-FLT_MAX, 0.0f, 0.0f, -INFINITY}; }
// The parts of lanes 0..15 as one; every lane of both halves gets the same
// bits (each step adds the same two values on both sides).
template <bool ENT> __device__ __forceinline__ Part join_lanes(Part p, float c) {
  float m = p.m;
#pragma unroll
  for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
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

// The j-th largest of the values of N neighbouring lanes, 1 <= j <= N: a
// bitonic sort in descending order.
template <int N> __device__ __forceinline__ float nth_largest(float v, int j) {
  const int lane = threadIdx.x & (N - 1);
#pragma unroll
  for (int k = 2; k <= N; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o; o >>= 1) {
      const float u = __shfl_xor_sync(FULL, v, o);
      v = ((lane & o) == 0) == ((lane & k) == 0) ? fmaxf(v, u) : fminf(v, u);
    }
  return __shfl_sync(FULL, v, j - 1);
}

// f4(chunks, index of the first) for four of a thread's chunks tid, tid + TH,
// ... of a piece in shared memory at a time while the whole warp has four left,
// then f1 for one at a time; a lane without a chunk gets one of -inf.  The
// warp's lanes stay together.
template <typename T, int TH, typename F4, typename F1>
__device__ __forceinline__ void for_chunks(uint32_t st, int cnt, F4 &&f4, F1 &&f1) {
  const int lane = threadIdx.x & 31;
  int i = threadIdx.x - lane;                      // of the warp's first lane
  uint32_t at = st + 16u * threadIdx.x;
  for (; i + 3 * TH + 31 < cnt; i += 4 * TH, at += 64u * TH) {
    const uint4 x[4] = {lds(at), lds(at + 16 * TH), lds(at + 32 * TH), lds(at + 48 * TH)};
    f4(x, i + lane);
  }
  for (; i < cnt; i += TH, at += 16 * TH) {
    uint4 x[1] = {make_uint4(Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL, Elem<T>::FILL)};
    if (i + lane < cnt) x[0] = lds(at);
    f1(x, i + lane);
  }
}
template <typename T, int TH, typename F> __device__ __forceinline__ void for_chunks(uint32_t st, int cnt, F &&f) {
  for_chunks<T, TH>(st, cnt, [&](const uint4 (&x)[4], int i) {
#pragma unroll
    for (int k = 0; k < 4; k++) f(x[k], i + k * TH);
  }, [&](const uint4 (&x)[1], int i) { f(x[0], i); });
}

// This thread's running statistics of a row: m the largest logit so far, s and
// t relative to it, of the piece at hand (s2, t2) and of those before (s, t).
// A piece adds at most 64 values to a sum one after another, so a long row's
// rounding stays that of 64 and its pieces' additions (one sum for the whole
// row: 1024 at 262144 logits).
struct Running {
  float m = -FLT_MAX, top = -INFINITY, s = 0.0f, t = 0.0f;
  f32x2 s2 = 0, t2 = 0;
  // Adds C chunks; the largest of their logits.
  template <typename T, bool ENT, int C> __device__ __forceinline__ float add(const uint4 (&x)[C], float c) {
    constexpr int EV = Elem<T>::EV;
    float b = Elem<T>::max_of(x[0]);
#pragma unroll
    for (int k = 1; k < C; k++) b = fmaxf(b, Elem<T>::max_of(x[k]));
    top = fmaxf(top, b);
    if (b > m) {                       // the sums move to the new reference
      const float d = bounded((m - b) * c), f = exp2_fast(d);
      const f32x2 f2 = pack2(f, f);
      if (ENT) {
        t2 = mul2(f2, fma2(s2, pack2(d, d), t2));
        t = f * fmaf(s, d, t);
      }
      s2 = mul2(s2, f2);
      s *= f;
      m = b;
    }
    const f32x2 nm = pack2(-m, -m), cc = pack2(c, c);
#pragma unroll
    for (int k = 0; k < C; k++) {
      float f[EV];
      Elem<T>::unpack(x[k], f);
#pragma unroll
      for (int e = 0; e < EV; e += 2) {
        float d0, d1;
        unpack2(mul2(add2(pack2(f[e], f[e + 1]), nm), cc), d0, d1);
        const f32x2 ex = pack2(exp2_fast(d0), exp2_fast(d1));
        s2 = add2(s2, ex);
        if (ENT) t2 = fma2(ex, pack2(bounded(d0), bounded(d1)), t2);
      }
    }
    return b;
  }
  // A piece ends.
  template <bool ENT> __device__ __forceinline__ void fold() {
    float a, b;
    unpack2(s2, a, b);
    s += a + b;
    s2 = 0;
    if (ENT) {
      unpack2(t2, a, b);
      t += a + b;
      t2 = 0;
    }
  }
  // The warp's part, all pieces folded.
  template <bool ENT> __device__ __forceinline__ Part warp(float c) const {
    Part p = no_part();
    p.m = warp_max(m);
    const float d = bounded((m - p.m) * c), f = exp2_fast(d);
    p.s = warp_sum(s * f);
    if (ENT) p.t = warp_sum(f * fmaf(s, d, t));
    return p;
  }
};
template <typename T, int TH, bool ENT>
__device__ __forceinline__ void add_share(Running &run, uint32_t st, int cnt, float c) {
  for_chunks<T, TH>(st, cnt, [&](const uint4 (&x)[4], int) { run.add<T, ENT>(x, c); },
                 [&](const uint4 (&x)[1], int) { run.add<T, ENT>(x, c); });
  run.fold<ENT>();
}

// The blocks of a row: `sync` is a barrier of all their threads.
struct Team {
  static __device__ __forceinline__ unsigned rank() { return cg::this_cluster().block_rank(); }
  static __device__ __forceinline__ unsigned size() { return cg::this_cluster().num_blocks(); }
  static __device__ __forceinline__ void sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  }
  template <typename P> static __device__ __forceinline__ P *at(P *p, unsigned r) {
    return cg::this_cluster().map_shared_rank(p, r);
  }
};

// The parts of a row's warps (one block) or blocks (cluster) as one; for every
// lane of the calling warp.
template <bool ENT> __device__ __forceinline__ Part join_all(const Part *part, int count, float c) {
  const int lane = threadIdx.x & 15;
  Part p = no_part();
  if (lane < count) p = part[lane];
  return join_lanes<ENT>(p, c);
}
// Hands the block's part to the row's blocks (from[], by rank) and waits for
// theirs; the block's warps have written part[] before.  w becomes the g-th
// largest of the warps', +inf where g is 0.  The caller takes part[] and
// from[] in turn from two buffers: a barrier lies between a row's reads of one
// and the next write of it.
template <bool ENT>
__device__ __forceinline__ void meet(const Part *part, Part *from, int g, float c) {
  using TM = Team;
  __syncthreads();
  if (threadIdx.x < 32) {
    Part p = join_all<ENT>(part, blockDim.x >> 5, c);
    p.w = INFINITY;
    if (g) p.w = nth_largest<16>((threadIdx.x & 15) < (blockDim.x >> 5) ? part[threadIdx.x & 15].w : -INFINITY, g);
    if (threadIdx.x < TM::size()) *TM::at(&from[TM::rank()], threadIdx.x) = p;
  }
  TM::sync();
}

}  // namespace lg

// ------------------------------------------------------------ launch plan
// How rows are laid over the GPU: `threads` a block, `blocks` a row (more than
// one: a cluster).
struct RowPlan {
  int threads, blocks;
  lg::Layout l;
};
RowPlan plan_rows(const DeviceCtx *c, const LogitRows &z, int K, bool twice);
// Launches a kernel over N rows: as many blocks (clusters of `blocks`) as the
// GPU holds at once, each taking rows in turn.  `more_threads` beside the
// plan's in a block, `more_smem` bytes of dynamic shared memory after the stages, `args` is the kernel's one argument, `seen`
// belongs to the kernel and the device: how many fit, for its latest shapes.
struct Resident {
  static constexpr int N = 16;
  struct Shape {
    int threads, blocks, smem, fit;
  };
  int ready, next;
  Shape of[N];
};
int launch_rows(const void *kernel, DeviceCtx *c, const RowPlan &p, int more_threads, int more_smem, Resident *seen, void *args);

}  // namespace tl
