// Scoring kernels over [B, V] logits (fp32, bf16, fp16): log-probabilities of
// given tokens with the row's entropy and top alternatives, their gradient,
// and distillation from a teacher's top values.
//
// With z = x / T, m = max z, s = sum exp(z - m):
//   logprob(y) = z_y - m - log s
//   H          = log s - (1/s) sum exp(z - m) (z - m)
// so one pass over the row with a running maximum (m, s and the sum of
// exp(z - m)(z - m), rescaled when the maximum moves) gives everything but the
// alternatives.  Each thread keeps its own running maximum and fp32 sums (of a
// step's terms, then of the steps); warps are joined in fp64.
//
// A row is one thread-block cluster's: its CTAs take equal slices and exchange
// their sums (a few numbers) through distributed shared memory, so a call needs
// no scratch in global memory and one launch, whether it holds one row or
// thousands.  The grid holds as many clusters as the GPU runs at once, each
// working through its rows; every thread keeps a ring of asynchronous copies of
// its own vectors in flight (shared memory that no other thread touches, so no
// barrier guards it), which runs ahead into the next row while a row is
// finished.  The reads of HBM bound the large calls, latency the small ones.
//
// A row's special cases follow from the same sums: a NaN or +Inf logit makes s
// NaN (Inf - Inf), a row of -Inf alone leaves s = 0.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <mutex>
#include <type_traits>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_scores.cuh"

namespace cg = cooperative_groups;

namespace ms {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
// 16-byte vectors of a thread's step.  2 instead, with twice the steps in flight
// (same bytes): 2048 x 151936 bf16 102 -> 115 us, 512 x 262144 top 64 130 -> 142,
// distillation of 4096 x 151936 540 -> 551.
constexpr int kBatch = 4;
constexpr int kMaxCluster = 16;
constexpr int kBuf = 2048;      // keys the selection holds (runs of 32)
constexpr int kScan = 512;      // of them, those that the tiled selection uses: top_n and a tile of kRowThreads

// ---------------------------------------------------------------- row access
// A row is read in 16-byte vectors on 16-byte boundaries, whatever its start:
// vector v holds elements [v * VEC - mis, v * VEC - mis + VEC), those inside
// [0, V) being the row's.  Only the row's own elements are touched.
template <typename T>
struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  const T* p;  // the row's first element
  int V, mis, nvec;
  __device__ Row(const void* x, int64_t r, int64_t ld, int V_) : p((const T*)x + r * ld), V(V_) {
    mis = (int)(((uintptr_t)p & 15) / sizeof(T));
    nvec = (mis + V + VEC - 1) / VEC;
  }
  __device__ __forceinline__ bool whole(int v) const { return v * VEC >= mis && (v + 1) * VEC - mis <= V; }
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ void unpack(uint4 u, float (&f)[4], float) {
  f[0] = __uint_as_float(u.x);
  f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z);
  f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(uint4 u, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(uint4 u, float (&f)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Vector v as floats; elements outside the row are -Inf.  Plain loads: a
// gradient may be written over the logits it was read from.
template <typename T>
__device__ __forceinline__ void load_vec(const Row<T>& R, int v, float (&f)[Row<T>::VEC]) {
  const int i0 = v * Row<T>::VEC - R.mis;
  if (R.whole(v)) {
    unpack(*reinterpret_cast<const uint4*>(R.p + i0), f, T());
  } else {
#pragma unroll
    for (int j = 0; j < Row<T>::VEC; j++) {
      const int i = i0 + j;
      f[j] = (i >= 0 && i < R.V) ? to_f(R.p[i]) : -INFINITY;
    }
  }
}

// Vector v of a row's gradient, in the vectors of the logits' row; `same` when
// the gradient's row starts at the same offset from a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_vec(const Row<T>& R, T* d, bool same, int v, const float (&f)[Row<T>::VEC]) {
  const int i0 = v * Row<T>::VEC - R.mis;
  if (same && R.whole(v)) {
    *reinterpret_cast<uint4*>(d + i0) = pack(f, T());
  } else {
#pragma unroll
    for (int j = 0; j < Row<T>::VEC; j++) {
      const int i = i0 + j;
      if (i >= 0 && i < R.V) d[i] = from_f<T>(f[j]);
    }
  }
}

// ---------------------------------------------------------------- running sums
// Sums over some of a thread's elements: their maximum m (-Inf while there is
// none), z = fp32(m a), and with y = x a - z, one rounding each,
// s = sum 2^y and q = sum 2^y y, in two halves (the lanes of the paired fp32
// instructions).  What z's rounding leaves, z - m a, is in every term, and is put
// right in fp64 when the threads' sums are joined.  It is at most 2^-25 |z|: half
// a unit below kFar, but beyond fp32's exponents for a mask of -1e10 or a type's
// lowest value.  Where z is that large (or an Inf) the reference is m a itself,
// y = (x - m) a, an instruction more an element.
typedef unsigned long long f32x2;
struct Sums {
  float m = -INFINITY, z = 0.f;
  f32x2 s = 0, q = 0;
  bool odd = false;  // masked elements (0 times their y of -Inf): each term with care from here on
};
constexpr float kFar = 16777216.f;  // 2^24
__device__ __forceinline__ bool far(float z) { return !(fabsf(z) < kFar); }

// the larger of two, NaN when one of them is
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// y, bounded below so that a term of 0 times it is 0 (a NaN stays one)
__device__ __forceinline__ float bounded(float d) { return max_or_nan(d, -1e30f); }
__device__ __forceinline__ float below(float x, float m) { return bounded(__fsub_rn(x, m)); }
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float warp_max_f(float v) {
  float d;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}

// The step from a reference (m, z) to (M, Z), M >= m, in units of y.
__device__ __forceinline__ float step_of(float m, float z, float M, float Z, float a) {
  if (m == -INFINITY) return 0.f;  // sums of nothing (0), or of NaN alone: both stay
  if (!far(z) && !far(Z)) return bounded(__fsub_rn(z, Z));
  float d = __fsub_rn(m, M) * a;
  if (!far(z)) d += fmaf(-m, a, z);
  if (!far(Z)) d += fmaf(M, a, -Z);
  return bounded(d);
}

// A word of a vector as two fp32 elements (of 4-byte types: two words).
__device__ __forceinline__ f32x2 pair_of(uint32_t a, uint32_t, __nv_bfloat16) {
  return f2_pack(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
}
__device__ __forceinline__ f32x2 pair_of(uint32_t a, uint32_t, __half) {
  const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&a));
  return f2_pack(t.x, t.y);
}
__device__ __forceinline__ f32x2 pair_of(uint32_t a, uint32_t b, float) {
  return f2_pack(__uint_as_float(a), __uint_as_float(b));
}
// The largest element of N words (a NaN is in no maximum).
template <int N>
__device__ __forceinline__ float largest(const uint32_t (&w)[N], __nv_bfloat16) {
  __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
  for (int i = 1; i < N; i++) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
  return fmaxf(__low2float(m), __high2float(m));
}
template <int N>
__device__ __forceinline__ float largest(const uint32_t (&w)[N], __half) {
  __half2 m = *reinterpret_cast<const __half2*>(&w[0]);
#pragma unroll
  for (int i = 1; i < N; i++) m = __hmax2(m, *reinterpret_cast<const __half2*>(&w[i]));
  return fmaxf(__low2float(m), __high2float(m));
}
template <int N>
__device__ __forceinline__ float largest(const uint32_t (&w)[N], float) {
  float m = __uint_as_float(w[0]);
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) m = fmax3(m, __uint_as_float(w[i]), __uint_as_float(w[i + 1]));
  return fmaxf(m, __uint_as_float(w[N - 1]));
}

// A larger maximum: the sums carried over to it.
template <bool ENT>
__device__ __forceinline__ void raise_to(Sums& t, float hi, float a) {
  const float z = hi * a, d = step_of(t.m, t.z, hi, z, a), c = ex2_approx(d);
  const f32x2 c2 = f2_pack(c, c);
  if constexpr (ENT) t.q = f2_mul(c2, f2_fma(t.s, f2_pack(d, d), t.q));
  t.s = f2_mul(t.s, c2);
  t.m = hi;
  t.z = z;
}

// The terms of N words (N even); returns their largest element.
template <typename T, int N, bool ENT>
__device__ __forceinline__ float add_words(Sums& t, const uint32_t (&w)[N], float a) {
  constexpr int PER = sizeof(T) == 4 ? 2 : 1;  // words a pair
  const float hi = largest(w, T());
  if (hi > t.m) raise_to<ENT>(t, hi, a);
  // The words' own sum first, then onto the thread's: its roundings grow with
  // the thread's steps and not with its elements.
  if (!t.odd && !far(t.z)) {
    const f32x2 z2 = f2_pack(-t.z, -t.z), a2 = f2_pack(a, a);
    f32x2 s = 0, q = 0;
#pragma unroll
    for (int i = 0; i < N; i += PER) {
      const f32x2 y2 = f2_fma(pair_of(w[i], w[i + PER - 1], T()), a2, z2);
      const float2 y = f2_unpack(y2);
      const f32x2 e = f2_pack(ex2_approx(y.x), ex2_approx(y.y));
      s = i == 0 ? e : f2_add(s, e);
      if constexpr (ENT) q = i == 0 ? f2_mul(e, y2) : f2_fma(e, y2, q);
    }
    if constexpr (ENT) {
      const float2 h = f2_unpack(q);
      t.odd = isnan(h.x + h.y);
    }
    if (!t.odd) {
      t.s = f2_add(t.s, s);
      if constexpr (ENT) t.q = f2_add(t.q, q);
      return hi;
    }
  }
  const float m = t.m == -INFINITY ? 0.f : t.m;
  const bool from_m = far(t.z);
  f32x2 s = 0, q = 0;
#pragma unroll
  for (int i = 0; i < N; i += PER) {
    const float2 x = f2_unpack(pair_of(w[i], w[i + PER - 1], T()));
    const float y0 = bounded(from_m ? __fsub_rn(x.x, m) * a : fmaf(x.x, a, -t.z));
    const float y1 = bounded(from_m ? __fsub_rn(x.y, m) * a : fmaf(x.y, a, -t.z));
    const f32x2 e = f2_pack(ex2_approx(y0), ex2_approx(y1));
    s = i == 0 ? e : f2_add(s, e);
    if constexpr (ENT) q = i == 0 ? f2_mul(e, f2_pack(y0, y1)) : f2_fma(e, f2_pack(y0, y1), q);
  }
  t.s = f2_add(t.s, s);
  if constexpr (ENT) t.q = f2_add(t.q, q);
  return hi;
}

template <bool ENT>
__device__ __forceinline__ void add_term(Sums& t, float x, float a) {
  const uint32_t w[2] = {__float_as_uint(x), 0xff800000u};
  add_words<float, 2, ENT>(t, w, a);
}

// A warp's sums: {m, z, s, q} in every lane.
template <bool ENT>
__device__ __forceinline__ float4 warp_sums(const Sums& t, float a) {
  const float m = warp_max_f(t.m), z = m == -INFINITY ? 0.f : m * a;
  const float d = step_of(t.m, t.z, m, z, a), c = ex2_approx(d);
  const float2 s2 = f2_unpack(t.s), q2 = f2_unpack(t.q);
  float s = s2.x + s2.y, q = q2.x + q2.y;
  q = c * fmaf(s, d, q);
  s *= c;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    if constexpr (ENT) q += __shfl_xor_sync(0xffffffffu, q, o);
  }
  return make_float4(m, z, s, q);
}

// Sums of a CTA's or a row's elements in fp64: s = sum exp((x - m) / T) and
// q = sum exp((x - m) / T) (x - m) / T for their maximum m.
struct RowSums {
  float m;
  double s, q;
};

// exp(d), |d| next to 0 as a rule
__device__ __forceinline__ double exp_small(double d) {
  return fabs(d) < 1e-3 ? 1.0 + d * (1.0 + d * (0.5 + d * (1.0 / 6))) : exp(d);
}

// A warp's sums, relative to m itself.
__device__ __forceinline__ RowSums exact_sums(float4 w, float a) {
  const double ln2 = 0.693147180559945309417;
  RowSums r = {w.x, (double)w.z, (double)w.w * ln2};
  if (w.x != -INFINITY && !far(w.y)) {
    const double d = ((double)w.y - (double)w.x * (double)a) * ln2;  // |d| <= |z| 2^-24
    const double c = exp_small(d);
    r.q = (r.q + r.s * d) * c;
    r.s *= c;
  }
  return r;
}

// The sums of the lanes' parts (m = -Inf, s = q = 0 for none) in every lane.
template <bool ENT>
__device__ __forceinline__ RowSums lane_sums(const RowSums& p, float a) {
  RowSums r;
  r.m = warp_max_f(p.m);
  const float d = p.m == -INFINITY ? 0.f : below(p.m, r.m) * a;
  const double c = (double)ex2_approx(d);
  r.q = (p.q + p.s * (double)d * 0.693147180559945309417) * c;
  r.s = p.s * c;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    if constexpr (ENT) r.q += __shfl_xor_sync(0xffffffffu, r.q, o);
  }
  return r;
}

// The sums of n warps, warp(i) being the i-th's.
template <bool ENT, typename Warp>
__device__ __forceinline__ RowSums join_warps(int n, float a, Warp warp) {
  const int lane = threadIdx.x & 31;
  RowSums r = {-INFINITY, 0.0, 0.0};
  if (lane < n) r = exact_sums(warp(lane), a);
  r = lane_sums<ENT>(r, a);
#pragma unroll 1
  for (int i = 32; i < n; i += 32) {
    RowSums p = {-INFINITY, 0.0, 0.0};
    if (i + lane < n) p = exact_sums(warp(i + lane), a);
    p = lane_sums<ENT>(p, a);
    r = lane_sums<ENT>(lane == 0 ? r : lane == 1 ? p : RowSums{-INFINITY, 0.0, 0.0}, a);
  }
  return r;
}

// Named barriers: the warps that only tell others something do not wait.
__device__ __forceinline__ void bar_arrive(int id) { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "n"(kRowThreads) : "memory"); }
__device__ __forceinline__ void bar_sync(int id) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(kRowThreads) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The CTA's slice of a row: whole vectors [w0, w1), thread t's being w0 + t,
// w0 + t + kRowThreads, ..., kBatch of them a step; and the elements of a vector
// that reaches over the row's first or last element, one a thread (`edge`, -1
// for most threads).
template <typename T>
struct Slice {
  static constexpr int VEC = Row<T>::VEC;
  int w0, w1, edge;
  __device__ __forceinline__ Slice(const Row<T>& R, int rank, int ranks) {
    const int per = (R.nvec + ranks - 1) / ranks;
    const int v0 = min(R.nvec, rank * per), v1 = min(R.nvec, v0 + per);
    w0 = v0 + (v0 < v1 && !R.whole(v0));
    w1 = v1 - (v1 > w0 && !R.whole(v1 - 1));
    const int t = threadIdx.x;
    edge = -1;
    if (t < VEC && v0 < w0) edge = v0 * VEC - R.mis + t;
    if (t >= VEC && t < 2 * VEC && w1 < v1) edge = w1 * VEC - R.mis + t - VEC;
    if (edge >= R.V) edge = -1;
  }
  __device__ __forceinline__ int steps() const { return (w1 - w0 + kBatch * kRowThreads - 1) / (kBatch * kRowThreads); }
  // how many of them the thread has in full, and its vectors in the one after those (none: 0)
  __device__ __forceinline__ int whole_steps(int* rest) const {
    const int n = max(0, (w1 - w0 - (int)threadIdx.x + kRowThreads - 1) / kRowThreads);  // its vectors
    *rest = n % kBatch;
    return n / kBatch;
  }
  // the thread that holds element i, or -1 when it is not the slice's
  __device__ __forceinline__ int owner(const Row<T>& R, int i, int rank, int ranks) const {
    const int v = (i + R.mis) / VEC, l = (i + R.mis) % VEC;
    if (v >= w0 && v < w1) return (v - w0) % kRowThreads;
    const int per = (R.nvec + ranks - 1) / ranks;
    if (v < rank * per || v >= min(R.nvec, (rank + 1) * per)) return -1;
    return v < w0 ? l : VEC + l;
  }
};

// ---------------------------------------------------------------- the ring
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most n of the thread's latest groups are in flight.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// The rows first, first + step, ... that a cluster works on, and which of them
// are read at all: those with an id inside [0, V) in their list of n (every row
// when n = 0), and, where `weight` is given, a weight other than 0.  The row
// after the one in question is looked up early (lane l holds entry l).
struct RowList {
  const int32_t* ids;
  const float* weight;
  int n, V;
  int64_t B, step;
  int pre;
  float pre_w;
  __device__ __forceinline__ void fetch(int64_t row) {
    const int lane = threadIdx.x & 31;
    pre = -1;
    pre_w = 1.f;
    if (row < B) {
      if (lane < n) pre = ids[row * n + lane];
      if (weight) pre_w = weight[row];
    }
  }
  // for the row that was fetched last; the same in every thread of the cluster
  __device__ __forceinline__ bool read(int64_t row) const {
    if (n == 0) return true;
    bool any = __any_sync(0xffffffffu, (uint32_t)pre < (uint32_t)V);
    for (int j = 32 + (threadIdx.x & 31); !any && j - (int)(threadIdx.x & 31) < n; j += 32)
      any = __any_sync(0xffffffffu, j < n && (uint32_t)ids[row * n + min(j, n - 1)] < (uint32_t)V);
    return any && pre_w != 0.f;
  }
};

// The ring's places go round: the step that was just worked on frees the place
// that the feed fills next.
template <int DEPTH>
struct Place {
  uint32_t at, begin;  // the thread's first vector of the step, in shared memory
  __device__ __forceinline__ explicit Place(uint32_t first) : at(first), begin(first) {}
  __device__ __forceinline__ void next() {
    at += kBatch * kRowThreads * 16;
    if (at == begin + DEPTH * kBatch * kRowThreads * 16) at = begin;
  }
};

// The copies of a thread's vectors, in the order of the rows and of their
// steps, one group a step (an empty one when the rows are through).  TWICE:
// each row a second time, from its last step to its first, so that what was
// read last, which L2 still holds, comes first.
template <typename T, int DEPTH, bool TWICE = false>
struct Feed {
  RowList rows;
  const void* x;
  int64_t ld, row;
  int rank, ranks;
  int run, left;           // the pass's whole steps to come, and steps (0 or 1) after the whole ones
  int whole, part, rest;   // the row's whole steps, steps after them and vectors in that
  bool again;         // in the row's second pass
  const uint4* src;   // the thread's next vector
  // from the row that rows has fetched
  __device__ __forceinline__ void start(int64_t first, Place<DEPTH> place) {
    row = first;
    run = left = 0;
    settle();
#pragma unroll 1
    for (int i = 0; i < DEPTH; i++) {
      next(place.at);
      place.next();
    }
  }
  // the next row, from `row` on, that is read and has vectors here
  __device__ __forceinline__ void settle() {
    while (row < rows.B) {
      const bool yes = rows.read(row);
      rows.fetch(row + rows.step);
      if (yes) {
        const Row<T> R(x, row, ld, rows.V);
        const Slice<T> S(R, rank, ranks);
        src = reinterpret_cast<const uint4*>(R.p - R.mis) + S.w0 + threadIdx.x;
        run = whole = S.whole_steps(&rest);
        left = part = S.steps() - whole;
        again = false;
        if (run + left > 0) return;
      }
      row += rows.step;
    }
  }
  __device__ __forceinline__ void next(uint32_t dst) {
    bool end = false;  // of the pass: at the same call in every thread, however its last steps are made up
    if (run > 0) {
#pragma unroll
      for (int i = 0; i < kBatch; i++) copy16(dst + i * (kRowThreads * 16), src + i * kRowThreads);
      src += TWICE && again ? -kBatch * kRowThreads : kBatch * kRowThreads;
      end = --run == 0 && left == 0;
    } else if (left > 0) {  // the step that the thread has in part, or not at all
#pragma unroll
      for (int i = 0; i + 1 < kBatch; i++)
        if (i < rest) copy16(dst + i * (kRowThreads * 16), src + i * kRowThreads);
      left = 0;
      end = true;
      if (TWICE && again && whole > 0) {
        run = whole;
        src -= kBatch * kRowThreads;
        end = false;
      }
    }
    copies_end_group();
    if (end) turn();
  }
  // the end of a pass
  __device__ __forceinline__ void turn() {
    if (TWICE && !again) {
      again = true;
      // the second pass begins with the step that comes after the whole ones,
      // where src is; without one, with the last of those
      left = part;
      if (left == 0) {
        run = whole;
        src -= kBatch * kRowThreads;
      }
      return;
    }
    row += rows.step;
    settle();
  }
};

// One vector out of the ring.
__device__ __forceinline__ uint4 ring_vec(uint32_t at) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
  return u;
}
// A whole step's words.
__device__ __forceinline__ void ring_step(uint32_t at, uint32_t (&w)[4 * kBatch]) {
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    const uint4 u = ring_vec(at + i * (kRowThreads * 16));
    w[4 * i] = u.x;
    w[4 * i + 1] = u.y;
    w[4 * i + 2] = u.z;
    w[4 * i + 3] = u.w;
  }
}

// Element l of a thread's step (its vectors lie kRowThreads vectors apart, l
// counting elements of memory from the first one) set to -Inf.
template <typename T, int N>
__device__ __forceinline__ void mask_element(uint32_t (&w)[N], int l) {
  constexpr int VEC = Row<T>::VEC, PER = VEC / 4;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int at = (i / 4) * (kRowThreads * VEC) + (i % 4) * PER;  // the word's first element
    if constexpr (PER == 1) {
      if (l == at) w[i] = 0xff800000u;
    } else {
      const uint32_t inf = std::is_same_v<T, __half> ? 0xfc00u : 0xff80u;
      if (l == at) w[i] = (w[i] & 0xffff0000u) | inf;
      if (l == at + 1) w[i] = (w[i] & 0xffffu) | (inf << 16);
    }
  }
}

// ---------------------------------------------------------------- top alternatives
// A logit's key: its order, then the lowest id first (no two keys are alike; 0 is none).
__device__ __forceinline__ unsigned long long top_key(float x, int i) {
  return ((unsigned long long)fkey(x + 0.f) << 32) | (uint32_t)~i;
}

// Bitonic sort of n (a power of two) keys in shared memory, largest first.
__device__ __forceinline__ void sort_desc(unsigned long long* k, int n) {
  for (int size = 2; size <= n; size <<= 1) {
    for (int st = size >> 1; st > 0; st >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += blockDim.x) {
        const int lo = 2 * i - (i & (st - 1)), hi = lo + st;
        const unsigned long long x = k[lo], y = k[hi];
        if (((lo & size) == 0) == (x < y)) {
          k[lo] = y;
          k[hi] = x;
        }
      }
    }
  }
  __syncthreads();
}

struct TopSmem {
  unsigned long long key[kBuf];
  int n;
};

// Up to this many (CTAs a row) * (bounds) a CTA goes by its own bound; beyond,
// the CTAs meet first to find the row's.  Meeting costs about 1 us of a row and
// leaves fewer keys: one row of 50257, top 5, 7 CTAs (7): 10.0 us alone, 10.5 met;
// 16 CTAs (16): 12.3 alone, 11.3 met; 64 x 128256 top 20, 4 CTAs (12): 18.4 alone,
// 17.5 met; 512 x 262144 top 64, 2 CTAs (16): 130 alone, 128 met.
constexpr int kAlone = 10;
constexpr int kRounds = kScoreMax / kRowWarps;  // bounds that a CTA gives for the largest top_n

// A warp's share of the bounds for the alternatives: its j-th largest thread
// maximum into red[j], j < rounds (-Inf where it has fewer).  The least of them
// over the warps is reached by (j + 1) * kRowWarps of the CTA's elements at
// least.  tm: the thread's largest element.
__device__ __forceinline__ void top_maxima(float tm, int rounds, float (*red)[kRowWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t key = fkey(tm);
  for (int j = 0; j < rounds; j++) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == best);
    if (lane == __ffs(who) - 1) key = 0;  // one at a time: equal maxima count each
    if (lane == 0) red[j][warp] = best <= fkey(-INFINITY) ? -INFINITY : fkey_inv(best);
  }
}

// The row's bound from its CTAs' (each a list of `told`, largest first, in
// `lists` one after the other): every bound at or above the rounds-th largest
// of all of them stands for kRowWarps more elements.
__device__ __forceinline__ float row_bound(const float* lists, int ranks, int told, int rounds) {
  const int lane = threadIdx.x & 31;
  int at = 0;
  uint32_t best = 0;
  for (int j = 0; j < rounds; j++) {
    const uint32_t key = lane < ranks && at < told ? fkey(lists[lane * told + at]) : 0;
    best = __reduce_max_sync(0xffffffffu, key);
    if (lane == __ffs(__ballot_sync(0xffffffffu, key == best)) - 1) at++;
  }
  return best <= fkey(-INFINITY) ? -INFINITY : fkey_inv(best);
}

// A warp's keys, one a lane, sorted largest first.
__device__ __forceinline__ unsigned long long warp_sort_desc(unsigned long long k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int st = size >> 1; st > 0; st >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, st);
      const bool first = (lane & st) == 0, down = (lane & size) == 0;
      k = (first == down) == (k > o) ? k : o;
    }
  }
  return k;
}

// n keys (n <= kBuf) in runs of 32, each sorted by a warp.
__device__ __forceinline__ void sort_runs(TopSmem& sh, int n) {
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i - lane < n; i += kRowThreads)
    sh.key[i] = warp_sort_desc(i < n ? sh.key[i] : 0ull);
  __syncthreads();
}

// put(place, key) for each of the first top_n of n keys in sorted runs: a key's
// place is its place in its run and the number of larger keys in each of the
// others.  The places beyond the keys get 0.
template <typename Put>
__device__ __forceinline__ void place_keys(const TopSmem& sh, int n, int top_n, Put put) {
  const int runs = (n + 31) / 32;
  for (int i = threadIdx.x; i < n; i += kRowThreads) {
    const unsigned long long k = sh.key[i];
    int place = i & 31;
#pragma unroll 4
    for (int q = 0; q < runs; q++) {
      const unsigned long long* run = sh.key + q * 32;
      int at = 0;
#pragma unroll
      for (int st = 16; st > 0; st >>= 1) at += run[at + st - 1] > k ? st : 0;
      at += run[at] > k;
      if (q != i / 32) place += at;
    }
    if (place < top_n) put(place, k);
  }
  for (int i = n + threadIdx.x; i < top_n; i += kRowThreads) put(i, 0ull);
}

// Where a thread's largest elements lie: the two steps with the largest maxima,
// m1 >= m2, and the largest maximum m3 of the others.
struct TopSteps {
  float m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
  uint32_t at = 0;  // the first's step, and the second's in the upper half
  __device__ __forceinline__ void add(float hi, int step) {
    if (hi > m3) {
      if (hi > m1) {
        m3 = m2;
        m2 = m1;
        m1 = hi;
        at = at << 16 | (uint32_t)step;
      } else if (hi > m2) {
        m3 = m2;
        m2 = hi;
        at = (at & 0xffffu) | (uint32_t)step << 16;
      } else {
        m3 = hi;
      }
    }
  }
};
constexpr int kMostSteps = 0xffff;  // a thread's, for `at`

// Who holds a CTA's elements that reach the bound: threads' steps (thread and
// step << 8), and threads of which every step has to be read.
struct TopOwners {
  uint32_t step[2 * kRowThreads];
  uint8_t thread[kRowThreads];
  int n_steps, n_threads;
};

// The CTA's elements >= bound, as keys into the buffer `to` (a peer's).  Only
// steps whose maximum reaches the bound hold any; a thread knows its two
// largest, and only where a third reaches the bound too are all of its steps
// read.  All threads read those vectors together, out of L2 or HBM (every step
// of those threads instead: 512 x 262144 top 64 142 us, against 129).  A
// thread that finds the buffer full leaves the count above kBuf and takes no
// more keys.  xe: the thread's edge element.
template <typename T>
__device__ __forceinline__ void top_gather(const Row<T>& R, const Slice<T>& S, const TopSteps& t, float xe, float bound,
                                           TopOwners& own, TopSmem* to) {
  constexpr int VEC = Row<T>::VEC, AHEAD = 4;
  const uint4* base = reinterpret_cast<const uint4*>(R.p - R.mis);
  bool room = true;  // as far as this thread has seen
  auto take = [&](float x, int i) {
    if (room && x >= bound && x > -INFINITY) {
      const int n = atomicAdd(&to->n, 1);
      room = n < kBuf;
      if (room) to->key[n] = top_key(x, i);
    }
  };
  auto take_vec = [&](int v, const uint4& u) {
    float f[VEC];
    unpack(u, f, T());
#pragma unroll
    for (int j = 0; j < VEC; j++) take(f[j], v * VEC - R.mis + j);
  };
  if (t.m3 >= bound && t.m3 > -INFINITY) {
    own.thread[atomicAdd(&own.n_threads, 1)] = (uint8_t)threadIdx.x;
  } else {
    if (t.m1 >= bound && t.m1 > -INFINITY)
      own.step[atomicAdd(&own.n_steps, 1)] = threadIdx.x | (t.at & 0xffffu) << 8;
    if (t.m2 >= bound && t.m2 > -INFINITY)
      own.step[atomicAdd(&own.n_steps, 1)] = threadIdx.x | (t.at >> 16) << 8;
  }
  if (S.edge >= 0) take(xe, S.edge);
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; room && i < own.n_steps * kBatch; i += kRowThreads) {
    const uint32_t o = own.step[i / kBatch];
    const int v = S.w0 + (int)(o & 0xffu) + ((int)(o >> 8) * kBatch + i % kBatch) * kRowThreads;
    if (v < S.w1) take_vec(v, base[v]);
  }
  const int n = own.n_threads, each = (S.w1 - S.w0 + kRowThreads - 1) / kRowThreads;
#pragma unroll 1
  for (int i = threadIdx.x; room && i < n * each; i += AHEAD * kRowThreads) {
    uint4 u[AHEAD];
    int v[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      const int it = i + a * kRowThreads, k = it / n;
      v[a] = it < n * each ? S.w0 + own.thread[it - k * n] + k * kRowThreads : INT_MAX;
      if (v[a] < S.w1) u[a] = base[v[a]];
    }
#pragma unroll
    for (int a = 0; a < AHEAD; a++)
      if (v[a] < S.w1) take_vec(v[a], u[a]);
  }
}

// The row's top_n keys, largest first, at the front of sh.key (0 beyond the
// row's finite elements).  One element a thread at a time goes in when it
// beats the n-th best of those sorted so far; the buffer is sorted and cut
// back to top_n whenever the next tile might not fit.  Right for every row.
// Tiles come in order of their ids, so an element that only equals the n-th
// best of earlier tiles loses to it: tiles without a larger one are passed
// over, which is most of a row that ties by the thousand (10 finite logits
// among the type's lowest value, top 20, 64 x 128256 fp32: 73 us; each
// tile element by element 156).
template <typename T>
__device__ void top_scan(const Row<T>& R, int top_n, TopSmem& sh) {
  constexpr int VEC = Row<T>::VEC, AHEAD = 4;
  unsigned long long thr = 0;
  float least = -INFINITY;  // thr's logit
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  const int tiles = (R.nvec + kRowThreads - 1) / kRowThreads;
#pragma unroll 1
  for (int t0 = 0; t0 < tiles; t0 += AHEAD) {
    float hi[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      const int v = (t0 + a) * kRowThreads + threadIdx.x;
      hi[a] = -INFINITY;
      if (v >= R.nvec) continue;
      float f[VEC];
      load_vec(R, v, f);
#pragma unroll
      for (int j = 0; j < VEC; j++) hi[a] = fmaxf(hi[a], f[j]);
    }
    float any = hi[0];
#pragma unroll
    for (int a = 1; a < AHEAD; a++) any = fmaxf(any, hi[a]);
    if (!__syncthreads_or(any > least)) continue;
#pragma unroll
    for (int a = 0; a < AHEAD; a++) {
      if (!__syncthreads_or(hi[a] > least)) continue;
      const int v = (t0 + a) * kRowThreads + threadIdx.x;
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) f[j] = -INFINITY;
      if (v < R.nvec) load_vec(R, v, f);
#pragma unroll 1
      for (int j = 0; j < VEC; j++) {
        float x = f[0];
#pragma unroll
        for (int l = 1; l < VEC; l++) x = l == j ? f[l] : x;
        const unsigned long long k = x > -INFINITY ? top_key(x, v * VEC - R.mis + j) : 0ull;
        if (k > thr) sh.key[atomicAdd(&sh.n, 1)] = k;
        __syncthreads();
        const int n = sh.n;
        __syncthreads();
        if (n + kRowThreads > kScan) {
          for (int i = n + threadIdx.x; i < kScan; i += kRowThreads) sh.key[i] = 0;
          sort_desc(sh.key, kScan);
          thr = sh.key[top_n - 1];
          least = fkey_inv((uint32_t)(thr >> 32));
          __syncthreads();
          if (threadIdx.x == 0) sh.n = top_n;
          __syncthreads();
        }
      }
    }
  }
  const int n = sh.n;
  for (int i = n + threadIdx.x; i < kScan; i += kRowThreads) sh.key[i] = 0;
  sort_desc(sh.key, kScan);
}

// ---------------------------------------------------------------- forward
// CTAs an SM and steps of their rings: 96 KiB in flight an SM.  Every other load
// (tokens, the alternatives' second read) waits behind what the rings have asked
// for.  us of 2048 x 151936 bf16, 512 x 262144 top 64, 333 x 50257 top 3:
// 102, 130, 16 (now 103, 123, 16); with 3 steps 102, 128, 17; with 4 (and so 2 CTAs where there are
// alternatives) 102, 120, 23; 4 CTAs, at 64 registers, 121, 130, 17; 2 CTAs with
// 6 steps 112, 125, 21.
constexpr int kScoreCtas = 3, kScoreDepth = 2;
constexpr int kScoreRing = kScoreDepth * kBatch * kRowThreads * 16;

// A row's sums while they are joined: the warps', and the CTAs' (in the CTA
// that finishes the row) for a row and the next.
struct ScoreJoin {
  float4 warp[kRowWarps][kRowWarps];  // a place for each warp whose turn it is, in a cluster two that alternate
  RowSums cta[2][kMaxCluster];
};
// With alternatives: every warp's sums go to rank 0 as they are.
struct TopJoin {
  float red[kRounds][kRowWarps];   // then in red[.][0] the bounds that the CTA tells the others
  float lists[4 * kRounds];        // what they all told
  TopOwners own;
  float m;                         // the row's maximum and log of its sum
  double s, log_s;
  float warps[kMaxCluster * kRowWarps][3];  // every warp's {m, s, q}
  TopSmem sel;                     // rank 0's is the row's
};

// A padded row's outputs, by one warp.
__device__ __forceinline__ void write_padding(const ScoreArgs& A, int64_t r) {
  const ms_scores& O = A.out;
  const int lane = threadIdx.x & 31;
  for (int t = lane; t < A.n_tok; t += 32)
    if (O.logprobs) O.logprobs[r * A.n_tok + t] = 0.f;
  for (int i = lane; i < A.top_n; i += 32) {
    if (O.top_ids) O.top_ids[r * A.top_n + i] = -1;
    if (O.top_logprobs) O.top_logprobs[r * A.top_n + i] = -INFINITY;
  }
  if (lane == 0) {
    if (O.entropy) O.entropy[r] = 0.f;
    if (O.row_max) O.row_max[r] = 0.0;
    if (O.row_sum) O.row_sum[r] = 0.0;
  }
}

// log s for s >= 1, in fp32's precision near 1 too
__device__ __forceinline__ double log_sum(double s) {
  if (s < 1.0) s = 1.0;  // the largest term is 1 but for its rounding
  return s < 2.0 ? (double)log1pf((float)(s - 1.0)) : (double)logf((float)s);
}

// A row's numbers and its tokens' log-probabilities from its sums, by one warp.
// log s is -Inf for a row of -Inf alone, NaN for a NaN row.
// y, x: lane t's token and its logit, t < 32.
template <typename T, bool ENT>
__device__ __forceinline__ void write_row(const ScoreArgs& A, int64_t r, const Row<T>& R, const RowSums& sum, int y,
                                          float x) {
  const ms_scores& O = A.out;
  const int lane = threadIdx.x & 31;
  const double log_s = sum.s == 0.0 ? -INFINITY : log_sum(sum.s);
  const bool empty = sum.s == 0.0;
  if (O.logprobs)
    for (int t = lane; t < A.n_tok; t += 32) {
      if (t >= 32) {
        y = A.tokens[r * A.n_tok + t];
        x = (uint32_t)y < (uint32_t)A.V ? to_f(R.p[y]) : 0.f;
      }
      float lp = 0.f;
      if ((uint32_t)y < (uint32_t)A.V)
        lp = empty ? -INFINITY : (float)(((double)x - (double)sum.m) * A.rT - log_s);
      O.logprobs[r * A.n_tok + t] = lp;
    }
  if (lane == 0) {
    if (ENT) {
      const double h = empty ? 0.0 : log_s - sum.q / sum.s;
      O.entropy[r] = h < 0.0 ? 0.f : (float)h;  // one id left: 0 but for rounding
    }
    if (O.row_max) O.row_max[r] = (double)sum.m / A.T;
    if (O.row_sum) O.row_sum[r] = sum.s;
  }
}

// A cluster's rows, one after the other.  Every warp sums its share of the
// slice.  Without alternatives only the warp whose turn it is waits for the
// others: it joins the CTA's sums and hands them to the CTA whose turn it is,
// which writes the row; both turns go round, and everyone else is at the next
// row meanwhile.  A place of the join is free again when it is written next: by
// itself, a CTA's warp has had its own turn since, for which the place's warp
// had to arrive; in a cluster, it has passed the barrier of the row before.
//
// With alternatives, every CTA also finds bounds that top_n of its elements
// reach, from the thread maxima that the sums need anyway.  The best bound of
// all the CTAs' is reached by top_n elements of the row, so the alternatives
// are among the elements that reach it: about top_n and a few more, held by
// about top_n threads, whose vectors (and no others) are read once more, out
// of L2.  Rank 0 gathers and orders them.
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(kRowThreads, kScoreCtas) logprobs_kernel(ScoreArgs A) {
  extern __shared__ uint4 ring[];
  __shared__ std::conditional_t<TOP, TopJoin, ScoreJoin> joins;
  TopJoin& tp = reinterpret_cast<TopJoin&>(joins);
  ScoreJoin& join = reinterpret_cast<ScoreJoin&>(joins);
  TopSmem* const top = &tp.sel;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ranks = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // bounds that the alternatives need, and those that each CTA tells: twice its share and two more
  const int rounds = (A.top_n + kRowWarps - 1) / kRowWarps;
  const int share = min(rounds, (2 * rounds + ranks - 1) / ranks + 2);
  // with few CTAs or alternatives each CTA's own bound leaves few enough elements
  const bool alone = ranks == 1 || ranks * rounds <= kAlone;
  const int64_t first = blockIdx.x / ranks, step = gridDim.x / ranks;
  const ms_scores& O = A.out;
  Feed<T, kScoreDepth> feed;
  feed.rows = {A.tokens, nullptr, A.n_tok, A.V, A.B, step, -1, 1.f};
  feed.rows.fetch(first);
  RowList rows = feed.rows;  // the rows as they are worked on
  feed.x = A.x;
  feed.ld = A.ld;
  feed.rank = rank;
  feed.ranks = ranks;
  Place<kScoreDepth> place(smem_addr(ring + tid));
  feed.start(first, place);
  int which = 0, turn_rank = 0, turn_warp = 0;
  // for the cluster's barrier of the row before (at first: for its CTAs to have started)
  bool waiting = !TOP && ranks > 1;
  if (waiting) cluster_arrive();
  for (int64_t r = first; r < A.B; r += step) {
    const bool live = rows.read(r);  // the same in every CTA of the cluster
    rows.fetch(r + step);
    if (!live) {
      if (rank == 0 && warp == 0) write_padding(A, r);
      continue;
    }
    const Row<T> R(A.x, r, A.ld, A.V);
    const Slice<T> S(R, rank, ranks);
    const float xe = S.edge >= 0 ? to_f(R.p[S.edge]) : -INFINITY;
    if constexpr (TOP) {
      if (tid == 0) top->n = tp.own.n_steps = tp.own.n_threads = 0;
      if (ranks > 1) cluster_arrive();
    }
    // the warp that writes the row's numbers
    const bool writes = TOP ? rank == 0 && warp == kRowWarps - 1 : rank == turn_rank && warp == turn_warp;
    int y = -1;
    if (writes && lane < A.n_tok) y = A.tokens[r * A.n_tok + lane];
    const float xy = (uint32_t)y < (uint32_t)A.V ? to_f(R.p[y]) : 0.f;

    Sums t;
    TopSteps steps;
    int rest;
    const int whole = S.whole_steps(&rest);
    if (TOP && whole > kMostSteps) steps.m3 = INFINITY;  // a step has no number: all of them are read
#pragma unroll 1
    for (int k = 0; k < whole; k++) {
      copies_wait<kScoreDepth - 1>();
      uint32_t w[4 * kBatch];
      ring_step(place.at, w);
      const float hi = add_words<T, 4 * kBatch, ENT>(t, w, A.a);
      if constexpr (TOP) steps.add(hi, k);
      feed.next(place.at);
      place.next();
    }
    if (whole < S.steps()) {
      copies_wait<kScoreDepth - 1>();
      float hi = -INFINITY;
#pragma unroll 1
      for (int i = 0; i < rest; i++) {
        const uint4 u = ring_vec(place.at + i * (kRowThreads * 16));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        hi = fmaxf(hi, add_words<T, 4, ENT>(t, w, A.a));
      }
      if constexpr (TOP) steps.add(hi, whole);
      feed.next(place.at);
      place.next();
    }
    if (S.edge >= 0) add_term<ENT>(t, xe, A.a);
    const float4 ws = warp_sums<ENT>(t, A.a);
    if constexpr (!TOP) {
      const int place = ranks == 1 ? turn_warp : which;
      if (lane == 0) join.warp[place][warp] = ws;
      __syncwarp();
      RowSums mine = {-INFINITY, 0.0, 0.0};
      if (warp == turn_warp) {
        bar_sync(1 + place);
        mine = join_warps<ENT>(kRowWarps, A.a, [&](int i) { return join.warp[place][i]; });
        if (ranks == 1) write_row<T, ENT>(A, r, R, mine, y, xy);
      } else {
        bar_arrive(1 + place);
      }
      if (ranks > 1) {
        if (waiting) cluster_wait();
        if (warp == turn_warp && lane == 0) *cl.map_shared_rank(&join.cta[which][rank], turn_rank) = mine;
        __syncwarp();
        cluster_arrive();
        waiting = true;
        if (writes) {
          cluster_wait();
          waiting = false;
          const RowSums sum = lane_sums<ENT>(lane < ranks ? join.cta[which][lane] : RowSums{-INFINITY, 0.0, 0.0}, A.a);
          write_row<T, ENT>(A, r, R, sum, y, xy);
        }
        which ^= 1;
      }
      if (++turn_rank == ranks) {
        turn_rank = 0;
        turn_warp = turn_warp + 1 == kRowWarps ? 0 : turn_warp + 1;
      }
    } else {
      // Its own bound: from the warps all of whose threads hold vectors (in a
      // short slice not all do), each with its share of top_n; none where a
      // warp's 32 threads are too few for that.
      const int full = min(kRowWarps, (S.w1 - S.w0) / 32), own = full > 0 ? (A.top_n + full - 1) / full : 33;
      const int told = alone ? (own <= 32 ? own : 0) : share;
      top_maxima(t.m, told, tp.red);
      __syncthreads();
      if (ranks > 1) cluster_wait();  // rank 0 is at this row
      float bound = -INFINITY;
      if (alone) {
        if (told > 0) {
          bound = INFINITY;
          for (int w = 0; w < full; w++) bound = fminf(bound, tp.red[told - 1][w]);
        }
      } else {
        if (tid < told) {
          float b = tp.red[tid][0];
#pragma unroll
          for (int w = 1; w < kRowWarps; w++) b = fminf(b, tp.red[tid][w]);
          tp.red[tid][0] = b;
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (tid < ranks * told) tp.lists[tid] = cl.map_shared_rank(&tp, tid / told)->red[tid % told][0];
        __syncthreads();
        bound = row_bound(tp.lists, ranks, told, rounds);
      }
      if (lane < 3) cl.map_shared_rank(&tp, 0)->warps[rank * kRowWarps + warp][lane] = lane == 0 ? ws.x : lane == 1 ? ws.z : ws.w;
      top_gather(R, S, steps, xe, bound, tp.own, cl.map_shared_rank(top, 0));
      if (ranks > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
      if (rank != 0) continue;  // the gathered keys are rank 0's
      if (writes) {
        const RowSums sum = join_warps<ENT>(ranks * kRowWarps, A.a, [&](int i) {
          const float m = tp.warps[i][0];
          return make_float4(m, m == -INFINITY ? 0.f : m * A.a, tp.warps[i][1], tp.warps[i][2]);
        });
        if (lane == 0) {
          tp.m = sum.m;
          tp.s = sum.s;
          tp.log_s = log_sum(sum.s);
        }
        write_row<T, ENT>(A, r, R, sum, y, xy);
      }
      const int n = top->n;
      bool bad = false;  // known once the warp above is done
      auto put = [&](int i, unsigned long long k) {
        if (O.top_ids) O.top_ids[r * A.top_n + i] = k ? (int32_t)~(uint32_t)k : -1;
        if (O.top_logprobs) {
          const double x = (double)fkey_inv((uint32_t)(k >> 32));
          O.top_logprobs[r * A.top_n + i] =
              k ? (float)((x - (double)tp.m) * A.rT - tp.log_s) : (bad ? (float)tp.s : -INFINITY);
        }
      };
      if (n > kBuf) {  // rows whose largest elements crowd into few threads, or tie by the hundred
        __syncthreads();  // every thread has read n
        top_scan(R, A.top_n, *top);
      } else {
        sort_runs(*top, n);
      }
      bad = !(tp.s >= 0.0);
      if (bad) {
        for (int i = tid; i < A.top_n; i += kRowThreads) put(i, 0);
      } else if (n > kBuf) {
        for (int i = tid; i < A.top_n; i += kRowThreads) put(i, top->key[i]);
      } else {
        place_keys(*top, n, A.top_n, put);
      }
      __syncthreads();  // before the next row's keys
    }
  }
  copies_wait<0>();
  if (waiting) cluster_wait();
  if (ranks > 1) {  // no CTA ends while a peer may write to it or read from it
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
}

// ---------------------------------------------------------------- backward
// dx_i = (1/T) [ sum_t g_t [i = y_t] - p_i (G + g_H (log p_i + H)) ], G = sum of
// the g_t of the row's tokens.  With e = 2^((x - m) a) this is e (c0 + c1 (x - m))
// for every element but the tokens', which are written after the others.
// Reads and writes a row once, in chunks that a CTA's start (the row's numbers,
// its tokens) is spread over.  2048 x 151936 bf16, a fifth padding: 174 us, 0.985
// of the copy rate; with one batch a thread 193 us, four 175, 256 threads 176.
// 61 x 50257: 6.1, 5.8, 8.3 and 6.6 us.
constexpr int kGradThreads = 128;
constexpr int kGradVecs = 8;     // vectors that a thread has in flight
constexpr int kGradBatches = 2;  // times that, a thread's share
constexpr int kGradChunk = kGradThreads * kGradVecs * kGradBatches;

template <typename T>
__global__ void __launch_bounds__(kGradThreads) logprobs_backward_kernel(ScoreArgs A, int chunks) {
  constexpr int VEC = Row<T>::VEC;
  __shared__ int s_y[kScoreMax];
  __shared__ float s_g[kScoreMax], s_x[kScoreMax];
  const int64_t r = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x % chunks);
  const Row<T> R(A.x, r, A.ld, A.V);
  T* d = (T*)A.dx + r * A.dld;
  const bool same = (((uintptr_t)d ^ (uintptr_t)R.p) & 15) == 0;
  const int v0 = chunk * kGradChunk, v1 = min(R.nvec, v0 + kGradChunk);
  const int e0 = max(0, v0 * VEC - R.mis), e1 = min(R.V, v1 * VEC - R.mis);  // this CTA's elements
  int any = 0;
  for (int t = threadIdx.x; t < A.n_tok; t += kGradThreads) {
    const int y = A.tokens[r * A.n_tok + t];
    const bool ok = (uint32_t)y < (uint32_t)A.V;
    s_y[t] = ok ? y : -1;
    s_g[t] = ok && A.g_lp ? A.g_lp[r * A.n_tok + t] : 0.f;
    if (y >= e0 && y < e1) s_x[t] = to_f(R.p[y]);  // before anything is written
    any |= ok;
  }
  const bool live = __syncthreads_or(any) != 0 || A.n_tok == 0;
  const uint4* src = reinterpret_cast<const uint4*>(R.p - R.mis);
  uint4 u[kGradVecs];
  auto fetch = [&](int v) {
#pragma unroll
    for (int i = 0; i < kGradVecs; i++) {
      const int w = v + i * kGradThreads;
      if (w < v1 && R.whole(w)) u[i] = src[w];
    }
  };
  int v = v0 + threadIdx.x;
  if (live) fetch(v);  // on their way while the row's numbers are read
  const double S = live ? A.row_sum[r] : 0.0;
  double G = 0.0;
  const double gH = A.g_ent ? (double)A.g_ent[r] : 0.0;
  bool some = gH != 0.0;  // not G: gradients that cancel in it are the tokens' own, and NaN in a NaN row
  for (int t = 0; t < A.n_tok; t++) {
    G += (double)s_g[t];
    some |= s_g[t] != 0.f;
  }
  const bool zero = S == 0.0 || !some;  // padded, all -Inf, or nothing to pass on
  const float m = (float)(A.row_max[r] * A.T);  // the row's largest logit, exact
  const double log_s = log(S), H = gH != 0.0 ? (double)A.entropy[r] : 0.0;
  const double k = -A.rT / S;
  const float c0 = (float)(k * (G + gH * (H - log_s)));
  const float c1 = (float)(k * gH * A.rT);
  // e (c0 + c1 (x - m)), x - m bounded below where e is 0 already (-256 ln 2 T): masks lie so far
  // off that c1 times their distance is beyond fp32 (T 0.001, g_H 655), and 0 times that NaN.
  // As -256 / a, a division in every thread, a call of 2048 x 151936 bf16 takes 189 us for 183.
  const float lowest = (float)(-177.4 * A.T);
  auto term = [&](float x) {
    const float dd = max_or_nan(__fsub_rn(x, m), lowest);
    return ex2_approx(dd * A.a) * fmaf(c1, dd, c0);
  };
  auto put = [&](int v, float(&f)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = term(f[j]);
    store_vec(R, d, same, v, f);
  };
  if (zero) {
    const float f[VEC] = {};
    for (; v < v1; v += kGradThreads) store_vec(R, d, same, v, f);
  }
  while (v < v1) {  // the same number of times in every thread but for the last
#pragma unroll
    for (int i = 0; i < kGradVecs; i++) {
      const int w = v + i * kGradThreads;
      if (w >= v1) break;
      float f[VEC];
      if (R.whole(w)) unpack(u[i], f, T());
      else load_vec(R, w, f);
      put(w, f);
    }
    v += kGradThreads * kGradVecs;
    fetch(v);
  }
  if (zero) return;
  __syncthreads();
  for (int t = threadIdx.x; t < A.n_tok; t += kGradThreads) {
    const int y = s_y[t];
    if (y < e0 || y >= e1) continue;
    double g = 0.0;
    bool first = true;
    for (int u = 0; u < A.n_tok; u++)
      if (s_y[u] == y) {
        if (u < t) first = false;
        g += (double)s_g[u];
      }
    if (!first) continue;  // the same token twice: its first place writes the sum
    d[y] = from_f<T>((float)(g * A.rT + (double)term(s_x[t])));
  }
}

// ---------------------------------------------------------------- distillation
// What is joined of a row: the sums of the ids not listed and of the listed
// ones, the warps' and the CTA's (which the others of the cluster read).
struct DistillJoin {
  float4 warp[kRowWarps];
  RowSums warp_listed[kRowWarps];
  RowSums others, listed;
};

// exp((x - m) / T) in fp64, m being a maximum that x is part of.
__device__ __forceinline__ double exact_term(float x, float m, double rT) {
  return x == -INFINITY ? 0.0 : exp(((double)x - (m == -INFINITY ? 0.0 : (double)m)) * rT);
}
// lane_sums for the listed ids' masses, whose terms are few and exact.
__device__ __forceinline__ RowSums lane_list(const RowSums& p, double rT) {
  RowSums r = {warp_max_f(p.m), 0.0, 0.0};
  r.s = warp_sum(p.m == -INFINITY ? p.s : p.s * exact_term(p.m, r.m, rT));
  return r;
}
// The teacher's list of a row, and what its warps add up of it: the masses,
// relative to exp(m / T) for a list of logits, and the terms of the loss.
struct DistillList {
  int id[kScoreMax];       // the listed ids, -1 where absent
  double q[kScoreMax];     // the teacher's masses
  int head[kRowThreads];   // the listed ids that a thread's vectors hold, as a chain of places in the list
  int link[kScoreMax];
  float m[kRowWarps];
  double mass[kRowWarps], loss[kRowWarps];
};

template <typename T>
__device__ __forceinline__ void zero_slice(const Row<T>& R, const Slice<T>& S, T* d, bool same) {
  const float f[Row<T>::VEC] = {};
  for (int v = S.w0 + threadIdx.x; v < S.w1; v += kRowThreads) store_vec(R, d, same, v, f);
  if (S.edge >= 0) d[S.edge] = from_f<T>(0.f);
}

// CTAs an SM, and steps of their rings.  The gradient's second loop takes the
// registers of a third CTA: 4096 x 151936 bf16 with gradient 540 us, with three
// CTAs that spill 570; the loss alone, 1024 x 151936 with 256 listed ids, 104 us
// with three, 123 with two.  With rings of 2 steps 571 us, of 4 and of 6 560.
template <bool GRAD>
struct DistillShape {
  static constexpr int kCtas = GRAD ? 2 : 3, kDepth = GRAD ? 3 : 2, kRing = kDepth * kBatch * kRowThreads * 16;
};

// A cluster's rows, one after the other.  The teacher's list (thread j holds
// entry j) is every CTA's; the sums are over the ids that are not listed, so
// that the mass outside the list is a sum of its own and no difference of two
// near 1; the listed ids come out of the vectors as they are read, each thread
// following the chain of those that its vectors hold.  The gradient (GRAD) is
// a second pass over the slice, out of L2 and through the same rings, whose
// copies start before the sums are joined.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kRowThreads, DistillShape<GRAD>::kCtas) distill_kernel(DistillArgs A) {
  static_assert(kScoreMax <= kRowThreads, "one list entry a thread");
  extern __shared__ uint4 ring[];
  __shared__ DistillList list[2];  // a row's and the next's
  __shared__ DistillJoin join[2];
  constexpr int VEC = Row<T>::VEC, STEP = kBatch * kRowThreads, kDepth = DistillShape<GRAD>::kDepth;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ranks = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = A.K;
  const bool logits = A.kind == MS_TEACHER_LOGITS;
  const int64_t begin = blockIdx.x / ranks, stride = gridDim.x / ranks;
  Feed<T, kDepth, GRAD> feed;
  feed.rows = {A.ids, A.loss ? nullptr : A.weight, K, A.V, A.B, stride, -1, 1.f};
  feed.x = A.x;
  feed.ld = A.ld;
  feed.rank = rank;
  feed.ranks = ranks;
  Place<kDepth> place(smem_addr(ring + tid));
  feed.rows.fetch(begin);
  feed.start(begin, place);
  int which = 0, joined = 0, turn = 0;
  int id_in = -1;  // thread j's entry of the row after the next prepared one, and its weight
  float val_in = -INFINITY, w_in = 1.f;
  auto fetch = [&](int64_t r) {
    if (r >= A.B) return;
    if (tid < K) {
      id_in = A.ids[r * K + tid];
      val_in = A.values[r * K + tid];
    }
    if (A.weight) w_in = A.weight[r];
  };
  // The list of the row that was fetched, into L: the ids and their masses, by warp.
  int id_next = -1;
  float val_next = -INFINITY, w_next = 1.f;
  auto prepare = [&](DistillList& L, int64_t after) {
    id_next = (uint32_t)id_in < (uint32_t)A.V ? id_in : -1;  // absent outside the vocabulary
    val_next = val_in;
    w_next = w_in;
    fetch(after);
    L.head[tid] = -1;
    if (warp * 32 >= K) {
      id_next = -1;
      if (lane == 0) L.m[warp] = -INFINITY, L.mass[warp] = 0.0;
      return;
    }
    const int id = logits && val_next == -INFINITY ? -1 : id_next;  // a logit of -Inf is absent too
    const float vm = logits ? warp_max_f(id >= 0 ? val_next : -INFINITY) : 0.f;
    const double q = id < 0 ? 0.0 : exp(logits ? ((double)val_next - (double)vm) * A.rT : (double)val_next);
    L.id[tid] = id;
    L.q[tid] = q;
    const double mass = warp_sum(q);
    if (lane == 0) L.m[warp] = vm, L.mass[warp] = mass;
  };
  fetch(begin);
  prepare(list[0], begin + stride);
  for (int64_t r = begin; r < A.B; r += stride, which ^= 1) {
    const Row<T> R(A.x, r, A.ld, A.V);
    const Slice<T> S(R, rank, ranks);
    T* d = (T*)A.dx + r * A.dld;
    const bool same = (((uintptr_t)d ^ (uintptr_t)R.p) & 15) == 0;
    int rest_vecs;  // of the step after the thread's whole ones
    const int whole = S.whole_steps(&rest_vecs);
    const bool part = whole < S.steps();
    DistillList& L = list[which];
    DistillJoin& J = join[joined];
    const float w = w_next, val = val_next;
    const bool read = __syncthreads_or(id_next >= 0) != 0 && (A.loss || w != 0.f);  // as the feed has it
    const bool grad = A.dx != nullptr && w != 0.f;
    if (!read) {  // in every CTA of the cluster
      if (tid == 0 && rank == 0 && A.loss) A.loss[r] = 0.f;
      if (A.dx) zero_slice(R, S, d, same);
      prepare(list[which ^ 1], r + 2 * stride);
      continue;
    }
    joined ^= 1;  // with the cluster's barriers, which rows that are not read do not reach

    // ---- the list
    const int id = warp * 32 < K ? L.id[tid] : -1;
    const bool mine = rank == turn;  // this CTA writes the row's loss
    if (++turn == ranks) turn = 0;
    const int own = id >= 0 ? S.owner(R, id, rank, ranks) : -1;
    const bool inside = own >= 0;
    float xl = -INFINITY;
    if (inside || (mine && id >= 0)) xl = to_f(R.p[id]);
    if (inside) L.link[tid] = atomicExch(&L.head[own], tid);
    const float xe = S.edge >= 0 ? to_f(R.p[S.edge]) : -INFINITY;
    __syncthreads();

    // ---- the sums over the ids that are not listed
    Sums t;
    const int head = L.head[tid];
    // the thread's first vector at or after v that holds a listed id
    auto next_from = [&](int v) {
      int next = INT_MAX;
      for (int j = head; j >= 0; j = L.link[j]) {
        const int vj = (L.id[j] + R.mis) / VEC;
        if (vj >= v && vj < S.w1) next = min(next, vj);
      }
      return next;
    };
    int next = next_from(S.w0);
    int v = S.w0 + tid;
#pragma unroll 1
    for (int k = 0; k < whole; k++, v += STEP) {
      copies_wait<kDepth - 1>();
      uint32_t x[4 * kBatch];
      ring_step(place.at, x);
      if (next < v + STEP) {
        for (int j = head; j >= 0; j = L.link[j]) mask_element<T>(x, L.id[j] + R.mis - v * VEC);
        next = next_from(v + STEP);
      }
      add_words<T, 4 * kBatch, false>(t, x, A.a);
      feed.next(place.at);
      place.next();
    }
    if (part) {
      copies_wait<kDepth - 1>();
#pragma unroll 1
      for (int i = 0; i < rest_vecs; i++) {
        const uint4 u = ring_vec(place.at + i * (kRowThreads * 16));
        uint32_t x[4] = {u.x, u.y, u.z, u.w};
        if (next < INT_MAX)
          for (int j = head; j >= 0; j = L.link[j]) mask_element<T>(x, L.id[j] + R.mis - (v + i * kRowThreads) * VEC);
        add_words<T, 4, false>(t, x, A.a);
      }
      feed.next(place.at);
      place.next();
    }
    if (S.edge >= 0) {
      bool listed = false;
      for (int j = head; j >= 0; j = L.link[j]) listed |= L.id[j] == S.edge;
      if (!listed) add_term<false>(t, xe, A.a);
    }
    const float4 ws = warp_sums<false>(t, A.a);
    RowSums wl = {-INFINITY, 0.0, 0.0};
    bool first = inside, twice = false;  // an id's first place in the list stands for it
    if (warp * 32 < K) {
      if (inside)
        for (int j = L.head[own]; j >= 0; j = L.link[j])
          if (j != tid && L.id[j] == id) {
            twice = true;
            first &= tid < j;
          }
      // in fp64: p - q of a listed id is what is left of two close numbers
      wl.m = warp_max_f(first ? xl : -INFINITY);  // a NaN is in no maximum, and in the sum
      wl.s = warp_sum(first ? exact_term(xl, wl.m, A.rT) : 0.0);
    }
    if (lane == 0) {
      J.warp[warp] = ws;
      J.warp_listed[warp] = wl;
    }
    __syncthreads();

    // ---- the row's sums
    auto others = [&](int i) { return J.warp[i]; };
    auto listed = [&] {
      return lane_list(lane < kRowWarps ? J.warp_listed[lane] : RowSums{-INFINITY, 0.0, 0.0}, A.rT);
    };
    RowSums O, l;
    // a CTA by itself: every warp joins the sums (without the gradient the third
    // CTA an SM leaves no registers for that: 1024 x 151936 111 us against 102)
    const bool each = GRAD && ranks == 1;
    if (each) {
      O = join_warps<false>(kRowWarps, A.a, others);
      l = listed();
    } else {
      if (warp == 0) {
        const RowSums o = join_warps<false>(kRowWarps, A.a, others);
        const RowSums p = listed();
        if (lane == 0) {
          J.others = o;
          J.listed = p;
        }
        __syncwarp();
      }
      if (ranks > 1) cluster_arrive();
    }
    prepare(list[which ^ 1], r + 2 * stride);  // in a cluster, meanwhile
    double Q = 0.0, log_top = 0.0;  // the teacher's mass; for logits, its log relative to the largest
    float top = 0.f;
    bool live = true;               // some entry is present
    const double mass_in = lane < kRowWarps ? L.mass[lane] : 0.0;
    if (logits) {
      const float m_in = lane < kRowWarps ? L.m[lane] : -INFINITY;
      top = warp_max_f(m_in);
      Q = mass_in == 0.0 ? 0.0 : mass_in * exp(((double)m_in - (double)top) * A.rT);
    } else {
      Q = mass_in;
    }
#pragma unroll
    for (int o = kRowWarps / 2; o > 0; o >>= 1) Q += __shfl_xor_sync(0xffffffffu, Q, o);
    Q = __shfl_sync(0xffffffffu, Q, 0);
    if (logits) {
      live = Q != 0.0;
      log_top = log(Q);
      Q = Q == Q ? 1.0 : Q;
    }
    double rest = logits ? 0.0 : 1.0 - Q;
    if (rest < kNoTail) rest = 0.0;
    const double wt = (double)w * A.rT, all = Q + rest;
    // an entry's log mass, and its mass
    auto log_q = [&] { return logits ? ((double)val - (double)top) * A.rT - log_top : (double)val; };
    auto mass = [&] { return id < 0 ? 0.0 : logits ? exp(log_q()) : L.q[tid]; };
    if (!each) {
      if (ranks > 1) cluster_wait();
      else __syncthreads();
      O = l = {-INFINITY, 0.0, 0.0};
      if (lane < ranks) {
        const DistillJoin* p = cl.map_shared_rank(&J, lane);
        O = p->others;
        l = p->listed;
      }
      O = lane_sums<false>(O, A.a);
      l = lane_list(l, A.rT);
    }
    const float m = fmaxf(O.m, l.m);
    // from the other ids' and the listed ones' maximum to the row's
    const double scale = O.m == -INFINITY ? 1.0 : exact_term(O.m, m, A.rT);
    const double scale_l = l.m == -INFINITY ? 1.0 : exact_term(l.m, m, A.rT);
    const double s = O.s * scale + l.s * scale_l;
    const bool empty = s == 0.0;
    if (A.loss && mine) {
      const double log_s = log(s);
      double loss = 0.0;
      if (warp * 32 < K) {
        const double q = mass();
        if (q != 0.0) loss = q * (log_q() - (((double)xl - (double)m) * A.rT - log_s));
        loss = warp_sum(loss);
      }
      if (lane == 0) L.loss[warp] = loss;
      __syncwarp();
      if (warp < kRowWarps - 1) {  // the others are at the gradient while the last one adds up
        bar_arrive(1);
      } else {
        bar_sync(1);
        loss = 0.0;
        for (int i = 0; i < kRowWarps; i++) loss += L.loss[i];
        if (rest != 0.0) {
          const double gap = O.m == -INFINITY ? 0.0 : ((double)O.m - (double)m) * A.rT;
          loss += rest * (log(rest) - (log(O.s) + gap - log_s));
        }
        if (empty) loss = INFINITY;
        if (lane == 0) A.loss[r] = live ? (float)loss : 0.f;
      }
    }

    // ---- the gradient: p_i (Q + rest - rest / R) outside the list, p_i (Q + rest) - q_i in it
    const bool pass = grad && live && !empty;
    if (A.dx && !pass) zero_slice(R, S, d, same);
    // Relative to the other ids' own maximum, so that a share of the rest stays
    // finite however little the student gives them.  What this writes for the
    // listed ids is overwritten below.
    const float mo = O.m == -INFINITY ? 0.f : O.m, zo = mo * A.a;
    // Nothing but -Inf outside the list: 0, or NaN in a row whose listed ids make it so.
    double cd = O.s == 0.0 ? 0.0 * s : wt * (all * (scale / s) - rest / O.s);
    if (!far(zo)) cd *= exp_small(((double)zo - (double)mo * (double)A.a) * 0.693147180559945309417);
    const float c = (float)cd;
    auto term = [&](float x) { return c * ex2_approx(far(zo) ? __fsub_rn(x, mo) * A.a : fmaf(x, A.a, -zo)); };
    const bool plain = same && !far(zo);
    const f32x2 a2 = f2_pack(A.a, A.a), z2 = f2_pack(-zo, -zo), c2 = f2_pack(c, c);
    // n of the step's vectors, the first being the row's v
    auto put = [&](int v, uint32_t at, int n) {
#pragma unroll 1
      for (int i = 0; i < n; i++) {
        float f[VEC];
        unpack(ring_vec(at + i * (kRowThreads * 16)), f, T());
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = term(f[j]);
        store_vec(R, d, same, v + i * kRowThreads, f);
      }
    };
    if (GRAD) {  // from the last step to the first
      if (part) {
        copies_wait<kDepth - 1>();
        if (pass) put(v, place.at, rest_vecs);
        feed.next(place.at);
        place.next();
      }
      uint4* to = reinterpret_cast<uint4*>(d - R.mis) + v;  // a 16-byte boundary where `same`
#pragma unroll 1
      for (int k = 0; k < whole; k++) {
        v -= STEP;
        to -= STEP;
        copies_wait<kDepth - 1>();
        if (pass && plain) {
#pragma unroll
          for (int i = 0; i < kBatch; i++) {
            constexpr int PER = VEC / 4, WORDS = 2 / PER;  // elements a word, words a pair
            const uint4 u = ring_vec(place.at + i * (kRowThreads * 16));
            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
            float f[VEC];
#pragma unroll
            for (int j = 0; j < 4; j += WORDS) {
              const float2 y = f2_unpack(f2_fma(pair_of(x[j], x[j + WORDS - 1], T()), a2, z2));
              const float2 e = f2_unpack(f2_mul(f2_pack(ex2_approx(y.x), ex2_approx(y.y)), c2));
              f[j * PER] = e.x;
              f[j * PER + 1] = e.y;
            }
            to[i * kRowThreads] = pack(f, T());
          }
        } else if (pass) {
          put(v, place.at, kBatch);
        }
        feed.next(place.at);
        place.next();
      }
    }
    if (pass) {
      if (S.edge >= 0) d[S.edge] = from_f<T>(term(xe));
      __syncthreads();
      if (first) {
        double qs = mass();
        if (twice) {  // in the list's order, whatever the chain's
          qs = 0.0;
          for (int j = 0; j < K; j++)
            if (L.id[j] == id)
              qs += logits ? L.q[j] * exp(((double)L.m[j >> 5] - (double)top) * A.rT - log_top) : L.q[j];
        }
        d[id] = from_f<T>((float)(wt * (all * (exact_term(xl, m, A.rT) / s) - qs)));
      }
    }
  }
  copies_wait<0>();
  if (ranks > 1) {  // no CTA ends while a peer may read from it
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  switch (dtype) {
    case MS_F32: return f(float());
    case MS_BF16: return f(__nv_bfloat16());
    case MS_F16: return f(__half());
    default: return cudaErrorInvalidValue;
  }
}

cudaLaunchConfig_t row_config(int ranks, int64_t ctas, int ring, cudaStream_t stream, cudaLaunchAttribute* at) {
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = (unsigned)ranks;
  at->val.clusterDim.y = at->val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = (size_t)ring;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cfg;
}

// A row kernel's clusters: how many of each size the current device runs at
// once (0: none), asked of the driver once.  A grid of that many clusters has
// no second wave, which would cost as much as the first.
struct RowClusters {
  const void* kernel;
  int device, n[kMaxCluster + 1];
};
template <typename Args>
cudaError_t row_clusters(void (*kernel)(Args), int ring, const RowClusters** found) {
  constexpr int kKnown = 512;  // kernels times devices
  static std::mutex mu;
  static RowClusters known[kKnown];
  static int n_known = 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < n_known; i++)
    if (known[i].kernel == (const void*)kernel && known[i].device == device) {
      *found = &known[i];
      return cudaSuccess;
    }
  if (n_known == kKnown) return cudaErrorMemoryAllocation;
  RowClusters& k = known[n_known];
  k = {(const void*)kernel, device, {}};
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring);
  // clusters beyond the portable size
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int c = 1; c <= kMaxCluster && e == cudaSuccess; c++) {
    cudaLaunchAttribute at;
    const cudaLaunchConfig_t cfg = row_config(c, c, ring, nullptr, &at);
    e = cudaOccupancyMaxActiveClusters(&k.n[c], kernel, &cfg);
    if (e != cudaSuccess && c > 8) {  // a size that this device does not run
      cudaGetLastError();
      k.n[c] = 0;
      e = cudaSuccess;
    }
  }
  if (e != cudaSuccess) return e;
  n_known++;
  *found = &k;
  return cudaSuccess;
}

// The best CTAs a row, `fit` or more, from a kernel's clusters.  The rows go over
// the clusters in rounds, so the time is about rounds * (slice + what a row
// costs its CTAs beside the copies), in bytes at a CTA's share of the
// bandwidth: `one` for a CTA by itself, `joined` where CTAs meet, and 2 KiB for
// each of them.  The figures are fitted to timings of every size; what a wrong
// choice costs, in us: 2048 x 151936 bf16 1 CTA 102, 2 121; one row of 50257 1 CTA
// 12.8, 2 10.5, 6 9.5, 16 11.3; 512 x 262144 top 64 1 CTA 134, 3 126, 4 130, 7 167;
// distillation of 1024 x 128256 1 CTA 132, 2 154, and of 8 x 262144 54, 31, 14 (16).
int best_ranks(const RowClusters& k, int64_t B, int64_t row_bytes, int fit, int64_t one, int64_t joined) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int c = fit; c <= kMaxCluster; c++) {
    const int n = k.n[c];
    if (n < 1) continue;
    const int64_t cost = (B + n - 1) / n * (row_bytes / c + (c == 1 ? one : joined + 2048 * c));
    if (cost < least) {
      least = cost;
      best = c;
    }
  }
  return best;
}

template <typename Args>
cudaError_t launch_rows(void (*kernel)(Args), const Args& A, const RowClusters& k, int ranks, int ring,
                        cudaStream_t stream) {
  if (ranks < 1 || k.n[ranks] < 1) return cudaErrorInvalidConfiguration;
  cudaLaunchAttribute at;
  const cudaLaunchConfig_t cfg = row_config(ranks, std::min<int64_t>(A.B, k.n[ranks]) * ranks, ring, stream, &at);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A);
  if (e != cudaSuccess) cudaGetLastError();  // it is returned here, not left for a later call
  return e;
}

}  // namespace

cudaError_t launch_logprobs(const ScoreArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const bool ent = A.out.entropy != nullptr, top = A.top_n > 0;
    auto k = ent ? (top ? logprobs_kernel<T, true, true> : logprobs_kernel<T, true, false>)
                 : (top ? logprobs_kernel<T, false, true> : logprobs_kernel<T, false, false>);
    // the bounds want twice as many threads a row as alternatives
    const int fit = A.top_n > kRowThreads / 2 ? 2 : 1;
    const RowClusters* rc = nullptr;
    const cudaError_t e = row_clusters(k, kScoreRing, &rc);
    if (e != cudaSuccess) return e;
    const int ranks = best_ranks(*rc, A.B, (int64_t)A.V * sizeof(T), fit, 16384, top ? 98304 : 24576);
    return launch_rows(k, A, *rc, ranks, kScoreRing, stream);
  });
}

// CTAs a row of the backward grid: one vector more than V / VEC, as a row may
// start anywhere in its first.
static int64_t grad_chunks(int32_t V, int vec) {
  const int64_t vecs = ((int64_t)V + 2 * vec - 2) / vec;
  return (vecs + kGradChunk - 1) / kGradChunk;
}
int64_t logprobs_backward_blocks(int64_t B, int32_t V, int dtype) { return B * grad_chunks(V, dtype == MS_F32 ? 4 : 8); }

cudaError_t launch_logprobs_backward(const ScoreArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int chunks = (int)grad_chunks(A.V, Row<T>::VEC);
    logprobs_backward_kernel<T><<<(unsigned)(A.B * chunks), kGradThreads, 0, stream>>>(A, chunks);
    return cudaGetLastError();
  });
}

cudaError_t launch_distill(const DistillArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    // the same CTAs a row with and without the gradient: the loss is the same to the bit
    const RowClusters* rc = nullptr;
    cudaError_t e = row_clusters(distill_kernel<T, true>, DistillShape<true>::kRing, &rc);
    if (e != cudaSuccess) return e;
    const int ranks = best_ranks(*rc, A.B, (int64_t)A.V * sizeof(T) * 2, 1, 65536, 131072);
    if (A.dx) return launch_rows(distill_kernel<T, true>, A, *rc, ranks, DistillShape<true>::kRing, stream);
    e = row_clusters(distill_kernel<T, false>, DistillShape<false>::kRing, &rc);
    if (e != cudaSuccess) return e;
    return launch_rows(distill_kernel<T, false>, A, *rc, ranks, DistillShape<false>::kRing, stream);
  });
}

}  // namespace ms
