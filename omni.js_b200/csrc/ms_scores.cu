// Scoring kernels over [B, V] logits (fp32, bf16, fp16): log-probabilities of
// given tokens with the row's entropy and top alternatives, their gradient,
// and distillation from a teacher's top values.
//
// With z = x / T, m = max z, s = sum exp(z - m):
//   logprob(y) = z_y - m - log s
//   H          = log s - (1/s) sum exp(z - m) (z - m)
// so one pass over the row with a running maximum (m, s and the sum of
// exp(z - m)(z - m), rescaled when the maximum moves) gives everything but the
// alternatives.  Each thread keeps its own running maximum and fp32 sums of at
// most a few hundred terms; threads are combined in fp64.
//
// A row's special cases follow from the same sums: a NaN or +Inf logit makes s
// NaN (Inf - Inf), a row of -Inf alone leaves s = 0.
#include <cfloat>
#include <climits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ms_scores.cuh"

namespace ms {
namespace {

constexpr int kRowThreads = 512;
constexpr int kBuf = 1024;  // keys the selection holds: top_n (<= 256) and at least one tile of kRowThreads

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
// Sums over some of a row's elements, relative to their maximum m (-Inf and
// s = 0 while there is none): s = sum 2^((x - m) a), q = sum 2^((x - m) a) (x - m).
struct Sums {
  float m = -INFINITY, s = 0.f, q = 0.f;
};

// x - m, bounded below so that a term of 0 times it is 0 (a NaN stays one)
__device__ __forceinline__ float below(float x, float m) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(__fsub_rn(x, m)), "f"(-1e30f));
  return d;
}

template <int N, bool ENT>
__device__ __forceinline__ void add_terms(Sums& t, const float (&f)[N], float a) {
  float bm = f[0];
#pragma unroll
  for (int i = 1; i < N; i++) bm = fmaxf(bm, f[i]);
  if (bm > t.m) {
    const float d = below(t.m, bm);  // -1e30 for the first terms: the factor is 0
    const float c = ex2_approx(d * a);
    if constexpr (ENT) t.q = c * fmaf(t.s, d, t.q);
    t.s *= c;
    t.m = bm;
  }
  // while every element so far is -Inf any finite reference gives terms of 0
  const float m = t.m == -INFINITY ? 0.f : t.m;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float d = below(f[i], m);
    const float e = ex2_approx(d * a);
    t.s += e;
    if constexpr (ENT) t.q = fmaf(e, d, t.q);
  }
}

// The sums of a whole row, in fp64: relative to the row's maximum m.
struct RowSums {
  float m;
  double s, q;
};

struct BlockScratch {
  float m[32];
  double s[32], q[32];
};

__device__ __forceinline__ RowSums block_sums(const Sums& t, float a, BlockScratch& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const float wm = warp_max(t.m);
  if (lane == 0) sh.m[warp] = wm;
  __syncthreads();
  RowSums r;
  r.m = sh.m[0];
  for (int w = 1; w < nw; w++) r.m = fmaxf(r.m, sh.m[w]);
  // a thread without a finite or infinite element has s = 0 or NaN: both stay
  const float d = t.m == -INFINITY ? 0.f : below(t.m, r.m);
  const float c = ex2_approx(d * a);
  double s = (double)t.s * c;
  double q = ((double)t.q + (double)t.s * d) * c;
  s = warp_sum(s);
  q = warp_sum(q);
  if (lane == 0) {
    sh.s[warp] = s;
    sh.q[warp] = q;
  }
  __syncthreads();
  r.s = 0.0;
  r.q = 0.0;
  for (int w = 0; w < nw; w++) {
    r.s += sh.s[w];
    r.q += sh.q[w];
  }
  return r;
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

// The row's top_n keys, largest first, at the front of sh.key (0 beyond the
// row's finite elements).  One element a thread at a time goes in when it
// beats the n-th best of those sorted so far; the buffer is sorted and cut
// back to top_n whenever the next tile might not fit.  Right for every row.
template <typename T>
__device__ void top_scan(const Row<T>& R, int top_n, TopSmem& sh) {
  constexpr int VEC = Row<T>::VEC;
  unsigned long long thr = 0;
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  const int tiles = (R.nvec + (int)blockDim.x - 1) / (int)blockDim.x;
  for (int t = 0; t < tiles; t++) {
    const int v = t * blockDim.x + threadIdx.x;
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
      if (n + (int)blockDim.x > kBuf) {
        for (int i = n + threadIdx.x; i < kBuf; i += blockDim.x) sh.key[i] = 0;
        sort_desc(sh.key, kBuf);
        thr = sh.key[top_n - 1];
        __syncthreads();
        if (threadIdx.x == 0) sh.n = top_n;
        __syncthreads();
      }
    }
  }
  const int n = sh.n;
  for (int i = n + threadIdx.x; i < kBuf; i += blockDim.x) sh.key[i] = 0;
  sort_desc(sh.key, kBuf);
}

// ---------------------------------------------------------------- forward
// Whether a row counts: no tokens asked for, or one of its ids inside [0, V).
__device__ __forceinline__ bool row_live(const ScoreArgs& A, int64_t r) {
  if (A.n_tok == 0) return true;
  int any = 0;
  for (int t = threadIdx.x; t < A.n_tok; t += blockDim.x) any |= (uint32_t)A.tokens[r * A.n_tok + t] < (uint32_t)A.V;
  return __syncthreads_or(any) != 0;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprobs_kernel(ScoreArgs A) {
  __shared__ BlockScratch bs;
  __shared__ TopSmem top;
  constexpr int VEC = Row<T>::VEC;
  const int64_t r = blockIdx.x;
  const Row<T> R(A.x, r, A.ld, A.V);
  const int32_t* tok = A.tokens + r * A.n_tok;
  const ms_scores& O = A.out;
  if (!row_live(A, r)) {
    for (int t = threadIdx.x; t < A.n_tok; t += blockDim.x)
      if (O.logprobs) O.logprobs[r * A.n_tok + t] = 0.f;
    for (int i = threadIdx.x; i < A.top_n; i += blockDim.x) {
      if (O.top_ids) O.top_ids[r * A.top_n + i] = -1;
      if (O.top_logprobs) O.top_logprobs[r * A.top_n + i] = -INFINITY;
    }
    if (threadIdx.x == 0) {
      if (O.entropy) O.entropy[r] = 0.f;
      if (O.row_max) O.row_max[r] = 0.0;
      if (O.row_sum) O.row_sum[r] = 0.0;
    }
    return;
  }
  Sums t;
  for (int v = threadIdx.x; v < R.nvec; v += blockDim.x) {
    float f[VEC];
    load_vec(R, v, f);
    add_terms<VEC, true>(t, f, A.a);
  }
  const RowSums S = block_sums(t, A.a, bs);
  const double log_s = log(S.s);  // -Inf for a row of -Inf alone, NaN for a NaN row
  const bool empty = S.s == 0.0;
  auto logprob = [&](float x) { return empty ? -INFINITY : (float)(((double)x - (double)S.m) / A.T - log_s); };
  if (threadIdx.x == 0) {
    if (O.entropy) O.entropy[r] = empty ? 0.f : (float)(log_s - S.q / S.s / A.T);
    if (O.row_max) O.row_max[r] = (double)S.m / A.T;
    if (O.row_sum) O.row_sum[r] = S.s;
  }
  if (O.logprobs)
    for (int i = threadIdx.x; i < A.n_tok; i += blockDim.x) {
      const int y = tok[i];
      O.logprobs[r * A.n_tok + i] = (uint32_t)y < (uint32_t)A.V ? logprob(to_f(R.p[y])) : 0.f;
    }
  if (A.top_n == 0) return;
  const bool bad = !(S.s >= 0.0);
  if (!bad) top_scan(R, A.top_n, top);
  for (int i = threadIdx.x; i < A.top_n; i += blockDim.x) {
    const unsigned long long k = bad ? 0ull : top.key[i];
    if (O.top_ids) O.top_ids[r * A.top_n + i] = k ? (int32_t)~(uint32_t)k : -1;
    if (O.top_logprobs)
      O.top_logprobs[r * A.top_n + i] = k ? logprob(fkey_inv((uint32_t)(k >> 32))) : (bad ? (float)S.s : -INFINITY);
  }
}

// ---------------------------------------------------------------- backward
// dx_i = (1/T) [ sum_t g_t [i = y_t] - p_i (G + g_H (log p_i + H)) ], G = sum of
// the g_t of the row's tokens.  With e = 2^((x - m) a) this is e (c0 + c1 (x - m))
// for every element but the tokens', which are written after the others.
constexpr int kGradThreads = 256;
constexpr int kGradVecs = 8;  // vectors a thread

template <typename T>
__global__ void __launch_bounds__(kGradThreads) logprobs_backward_kernel(ScoreArgs A, int chunks) {
  constexpr int VEC = Row<T>::VEC;
  __shared__ int s_y[kScoreMax];
  __shared__ float s_g[kScoreMax];
  const int64_t r = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x % chunks);
  const Row<T> R(A.x, r, A.ld, A.V);
  T* d = (T*)A.dx + r * A.dld;
  const bool same = (((uintptr_t)d ^ (uintptr_t)R.p) & 15) == 0;
  const int v0 = chunk * kGradThreads * kGradVecs, v1 = min(R.nvec, v0 + kGradThreads * kGradVecs);
  const int e0 = max(0, v0 * VEC - R.mis), e1 = min(R.V, v1 * VEC - R.mis);  // this CTA's elements
  int any = 0;
  float x_y = 0.f;  // thread t's token's logit, read before anything is written
  for (int t = threadIdx.x; t < A.n_tok; t += kGradThreads) {
    const int y = A.tokens[r * A.n_tok + t];
    const bool ok = (uint32_t)y < (uint32_t)A.V;
    s_y[t] = ok ? y : -1;
    s_g[t] = ok && A.g_lp ? A.g_lp[r * A.n_tok + t] : 0.f;
    if (y >= e0 && y < e1) x_y = to_f(R.p[y]);
    any |= ok;
  }
  const bool live = __syncthreads_or(any) != 0 || A.n_tok == 0;
  const double S = live ? A.row_sum[r] : 0.0;
  double G = 0.0;
  for (int t = 0; t < A.n_tok; t++) G += (double)s_g[t];
  const double gH = A.g_ent ? (double)A.g_ent[r] : 0.0;
  const bool zero = S == 0.0 || (G == 0.0 && gH == 0.0);  // padded, all -Inf, or nothing to pass on
  bool tokens_too = !zero;
  if (zero && S != 0.0)
    for (int t = 0; t < A.n_tok; t++) tokens_too |= s_g[t] != 0.f;  // gradients that cancel in G
  const float m = (float)(A.row_max[r] * A.T);  // the row's largest logit, exact
  const double log_s = log(S), H = gH != 0.0 ? (double)A.entropy[r] : 0.0;
  const double k = -A.rT / S;
  const float c0 = (float)(k * (G + gH * (H - log_s)));
  const float c1 = (float)(k * gH * A.rT);
  for (int v = v0 + threadIdx.x; v < v1; v += kGradThreads) {
    float f[VEC];
    if (zero) {
#pragma unroll
      for (int j = 0; j < VEC; j++) f[j] = 0.f;
    } else {
      load_vec(R, v, f);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float dd = below(f[j], m);
        f[j] = ex2_approx(dd * A.a) * fmaf(c1, dd, c0);
      }
    }
    store_vec(R, d, same, v, f);
  }
  if (!tokens_too) return;
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
    const float dd = below(x_y, m);
    d[y] = from_f<T>((float)(g * A.rT + (double)(ex2_approx(dd * A.a) * fmaf(c1, dd, c0))));
  }
}

// ---------------------------------------------------------------- distillation
struct DistillSmem {
  int id[kScoreMax];       // the listed ids, -1 where absent
  float x[kScoreMax];      // their logits
  double q[kScoreMax];     // the teacher's masses
  double red[32];
  int first[kScoreMax];    // 1: the id's first place in the list
  int next[kRowThreads];   // the first vector step of a thread that holds a listed id
};

// Sum of one value a thread, the same in every thread, in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) t += red[w];
  return t;
}
__device__ __forceinline__ float block_max(float v, double* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = (double)v;
  __syncthreads();
  float t = -INFINITY;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) t = fmaxf(t, (float)red[w]);
  return t;
}

// One row: the teacher's list (thread j holds entry j), then the row's sums
// without the listed ids, so that the mass outside the list is a sum of its own
// and no difference of two near 1, then the gradient over the row again.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_kernel(DistillArgs A) {
  __shared__ DistillSmem sh;
  __shared__ BlockScratch bs;
  constexpr int VEC = Row<T>::VEC;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, K = A.K;
  const Row<T> R(A.x, r, A.ld, A.V);
  T* d = (T*)A.dx + r * A.dld;
  const bool same = (((uintptr_t)d ^ (uintptr_t)R.p) & 15) == 0;

  // ---- the teacher
  int id = -1;
  float val = -INFINITY;
  if (tid < K) {
    id = A.ids[r * K + tid];
    val = A.values[r * K + tid];
    // an id outside the vocabulary is absent, and so is a logit of -Inf
    if ((uint32_t)id >= (uint32_t)A.V || (A.kind == MS_TEACHER_LOGITS && val == -INFINITY)) id = -1;
    sh.id[tid] = id;
  }
  sh.next[tid] = INT_MAX;
  const bool live = __syncthreads_or(id >= 0) != 0;
  const float w = A.weight ? A.weight[r] : 1.f;
  const bool grad = A.dx != nullptr && live && w != 0.f;
  if (!live || (!grad && !A.loss)) {
    if (tid == 0 && A.loss) A.loss[r] = 0.f;
    if (A.dx) {
      const float f[VEC] = {};
      for (int v = tid; v < R.nvec; v += blockDim.x) store_vec(R, d, same, v, f);
    }
    return;
  }
  double log_q = (double)val;
  if (A.kind == MS_TEACHER_LOGITS) {
    const float top = block_max(id >= 0 ? val : -INFINITY, sh.red);
    const double dv = ((double)val - (double)top) / A.T;
    log_q = dv - log(block_sum(id >= 0 ? exp(dv) : 0.0, sh.red));
  }
  const double q = id >= 0 ? exp(log_q) : 0.0;
  const double Q = block_sum(q, sh.red);
  double rest = A.kind == MS_TEACHER_LOGITS ? 0.0 : 1.0 - Q;
  if (rest < kNoTail) rest = 0.0;
  float xl = -INFINITY;
  bool first = false;
  if (id >= 0) {
    xl = to_f(R.p[id]);
    first = true;
    for (int j = 0; j < tid; j++) first &= sh.id[j] != id;
    const int v = (id + R.mis) / VEC;
    atomicMin(&sh.next[v % kRowThreads], v / kRowThreads);
  }
  if (tid < K) {
    sh.q[tid] = q;
    sh.first[tid] = first;
  }
  __syncthreads();

  // ---- the row's sums over the ids that are not listed
  Sums t;
  int next = sh.next[tid];
  for (int v = tid, step = 0; v < R.nvec; v += kRowThreads, step++) {
    float f[VEC];
    load_vec(R, v, f);
    if (step == next) {  // this vector holds a listed id: take them out, and find the thread's next
      next = INT_MAX;
      const int i0 = v * VEC - R.mis;
      for (int j = 0; j < K; j++) {
        const int i = sh.id[j];
        if (i < 0) continue;
        const int vj = (i + R.mis) / VEC;
        if (vj == v) {
#pragma unroll
          for (int l = 0; l < VEC; l++)
            if (i0 + l == i) f[l] = -INFINITY;
        } else if (vj % kRowThreads == tid && vj > v) {
          next = min(next, vj / kRowThreads);
        }
      }
    }
    add_terms<VEC, false>(t, f, A.a);
  }
  const float ml = block_max(first ? xl : -INFINITY, sh.red);
  RowSums S = block_sums(t, A.a, bs);
  const float m = fmaxf(S.m, ml);
  // a listed NaN is in no maximum; its term below makes the row NaN
  const double gap = S.m == -INFINITY ? 0.0 : ((double)S.m - (double)m) / A.T;
  const double scale = exp(gap);  // from the other ids' maximum to the row's
  const double tail = S.s * scale;
  const bool none = m == -INFINITY;
  const double e = first ? (xl == -INFINITY ? 0.0 : exp(((double)xl - (none ? 0.0 : (double)m)) / A.T)) : 0.0;
  const double s = tail + block_sum(e, sh.red);
  const bool empty = s == 0.0;
  const double log_s = log(s);
  if (A.loss) {
    double term = 0.0;
    if (id >= 0 && q != 0.0) term = q * (log_q - (((double)xl - (double)m) / A.T - log_s));
    double loss = block_sum(term, sh.red);
    if (rest != 0.0) loss += rest * (log(rest) - (log(S.s) + gap - log_s));
    if (empty) loss = INFINITY;
    if (tid == 0) A.loss[r] = (float)loss;
  }
  if (!A.dx) return;

  // ---- the gradient: p_i (Q + rest - rest / R) outside the list, p_i (Q + rest) - q_i in it
  if (!grad || empty) {
    const float f[VEC] = {};
    for (int v = tid; v < R.nvec; v += blockDim.x) store_vec(R, d, same, v, f);
    return;
  }
  // Relative to the other ids' own maximum, so that a share of the rest stays
  // finite however little the student gives them.  What this writes for the
  // listed ids is overwritten below.
  const double wt = (double)w / A.T, all = Q + rest;
  const float c = S.s == 0.0 ? 0.f : (float)(wt * (all * (scale / s) - rest / S.s));
  const float mo = S.m == -INFINITY ? 0.f : S.m;
  for (int v = tid; v < R.nvec; v += kRowThreads) {
    float f[VEC];
    load_vec(R, v, f);
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = c * ex2_approx(__fsub_rn(f[j], mo) * A.a);
    store_vec(R, d, same, v, f);
  }
  __syncthreads();
  if (first) {
    double qs = 0.0;
    for (int j = 0; j < K; j++)
      if (sh.id[j] == id) qs += sh.q[j];
    d[id] = from_f<T>((float)(wt * (all * (e / s) - qs)));
  }
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  switch (dtype) {
    case MS_F32: f(float()); break;
    case MS_BF16: f(__nv_bfloat16()); break;
    case MS_F16: f(__half()); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_logprobs(const ScoreArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) { logprobs_kernel<decltype(t)><<<(unsigned)A.B, kRowThreads, 0, stream>>>(A); });
}

// CTAs a row of the backward grid: one vector more than V / VEC, as a row may
// start anywhere in its first.
static int64_t grad_chunks(int32_t V, int vec) {
  const int64_t vecs = ((int64_t)V + 2 * vec - 2) / vec;
  return (vecs + kGradThreads * kGradVecs - 1) / (kGradThreads * kGradVecs);
}
int64_t logprobs_backward_blocks(int64_t B, int32_t V, int dtype) { return B * grad_chunks(V, dtype == MS_F32 ? 4 : 8); }

cudaError_t launch_logprobs_backward(const ScoreArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int chunks = (int)grad_chunks(A.V, Row<T>::VEC);
    logprobs_backward_kernel<T><<<(unsigned)(A.B * chunks), kGradThreads, 0, stream>>>(A, chunks);
  });
}

cudaError_t launch_distill(const DistillArgs& A, int dtype, cudaStream_t stream) {
  return by_type(dtype, [&](auto t) { distill_kernel<decltype(t)><<<(unsigned)A.B, kRowThreads, 0, stream>>>(A); });
}

}  // namespace ms
