// Log-probability of given tokens, entropy and the best alternatives of each row of logits, in one pass; the gradient in another.
//
// Forward. A thread keeps a reference m, sum e^(x - m) and sum e^(x - m) (x - m); they join into log sum exp and the entropy
// H = log s - t / s. The reference is raised only when a value passes it by more than kLag, so the loop has no dependent maximum.
// Bound by memory (one read of the logits) in fp32, 4095 x 32000 in 83 us, 6.3 TB/s; in 16 bits by the exponentials (16 a clock and SM: their
// unit is busy for 79 % of the time) and the issue slots (73 %), 51.5 us, 5.1 TB/s. Twenty alternatives add 30 us there (the threads' own
// largest value 17, the second look 13). The gradient reads and writes once: 88 us, 5.9 TB/s.
// A row belongs to one CTA; few rows are split over the CTAs of a cluster, which push their sums into the first one's shared memory.
//
// Alternatives. Nothing is sorted while the row streams by: every thread only remembers its largest value and the vector that it came from,
// as a key (value, lowest index first; keys are unique). The K-th largest of 64 groups' largest keys is a bound that K elements reach,
// and only threads whose own key reaches it, about K of them, can hold an element that does. Their vectors (K of 256 shares of the row)
// are read once more, most of them from L2, one a thread, and what reaches the bound is put down in shared memory in any order: its place is the
// number of better ones. If more reach the bound than there is room for (equal or sorted values), the K-th of those that were put down
// is a better bound. The result does not depend on any order of execution.
//
// Values that are masked with -inf or with the type's lowest value take no part in the sums (0 * inf is not computed); a row with a NaN or
// with +inf, or with nothing but -inf, has a NaN log-probability as log_softmax has.
#include "token_logprobs.h"

#include "gemm.h"
#include "ptx.cuh"

#include <algorithm>
#include <cfloat>
#include <cstring>

namespace ccl {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLag = 8.f;
constexpr float kFar = 131072.f;  // rows whose maximum is larger go value by value: natural() is exact enough below
constexpr int kMaxCluster = 16;
constexpr int kClusterVecs = 1024;  // 16-byte vectors of a row for each CTA of its cluster, at least
constexpr uint32_t kAbsent = 0xffffffffu;  // bits of "the target is in another shard"

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// ---- keys: larger is better; a NaN above everything, equal values by the lower index; 0: nothing --------------------------------------
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) { return ((unsigned long long)ordered(x) << 32) | (uint32_t)~index; }
__device__ __forceinline__ float value_of(unsigned long long key) { return unordered((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint32_t index_of(unsigned long long key) { return ~(uint32_t)key; }

// How many of keys[0 .. n) are better than k.
__device__ __forceinline__ int rank_of(const unsigned long long* keys, int n, unsigned long long k) {
  int better = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) better += keys[i] > k;
  return better;
}

// ---- sums -------------------------------------------------------------------------------------------------------------------------------
struct Sums {
  float m, s, t;  // t: of e^(x - m) (x - m) log2 e
};
__device__ __forceinline__ Sums nothing() { return {-FLT_MAX, 0.f, 0.f}; }
__device__ __forceinline__ void rebase(Sums& a, float m) {
  const float delta = (a.m - m) * kLog2e, f = ex2(delta);
  a.t = f == 0.f ? 0.f : f * (a.t + delta * a.s);
  a.s = f == 0.f ? 0.f : f * a.s;
  if (m != m) a.s = m;
  a.m = m;
}
__device__ __forceinline__ void add(Sums& a, float x) {
  const float d = (x - a.m) * kLog2e, e = ex2(d);
  a.s += e;
  a.t += e * fmaxf(d, -150.f);
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = max_nan(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  a.s += b.s;
  a.t += b.t;
  return a;
}

// The same in the loop over a row, where m is a whole number of powers of two: x log2 e - m is one multiply-add without an error in m, and sums
// join exactly. A value that is masked (-inf, or the type's lowest) is raised to where its exponential beside any other is still zero but 0 * d
// is not NaN.
// Rows that this does not hold for (nothing but masked values, infinities, NaN) are found by their sums and done again with Sums.
struct FastSums {
  float m, s, t;
};
__device__ __forceinline__ FastSums fast_nothing() { return {-FLT_MAX, 0.f, 0.f}; }
__device__ __forceinline__ void rebase(FastSums& a, float m) {
  const float delta = a.m - m, f = ex2(delta);
  a.t = f * (a.t + delta * a.s);
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void raise_to(FastSums& a, float most) {
  // The product rounded up: the nearest number may lie further below a masked value's product than e^x takes, and an infinite sum would send
  // the whole row through value by value (4095 x 32000 fp32, the first half masked: 199 instead of 82 us).
  if (fmaf(most, kLog2e, -a.m) > kLag) rebase(a, rintf(__fmul_ru(most, kLog2e)));
}
__device__ __forceinline__ void add(FastSums& a, float x) {
  const float d = fmaf(x, kLog2e, -a.m), e = ex2(d);
  a.s += e;
  a.t = fmaf(e, d, a.t);
}
__device__ __forceinline__ FastSums join(FastSums a, FastSums b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  a.s += b.s;
  a.t += b.t;
  return a;
}
// m to natural units, over the same rounded log2 e that the logits were multiplied with (at 2^20, ln 2 in its place is 2^-6 off); what its
// rounding leaves goes into the sums.
__device__ __forceinline__ Sums natural(const FastSums& a) {
  constexpr float kHigh = 0.693145752f;                                    // the upper 16 bits of 1 / kLog2e
  constexpr float kLow = (float)(1.0 / (double)kLog2e - (double)kHigh);    // and the rest
  const float high = a.m * kHigh, low = a.m * kLow;
  const float m = high + low, left = (fmaf(a.m, kHigh, -high) + (high - m)) + low;
  const float f = 1.f + left + 0.5f * left * left;
  return {m, a.s * f, fmaf(left * kLog2e, a.s, a.t) * f};
}

template <typename P>
__device__ __forceinline__ P halves(uint32_t a) {
  P p;
  memcpy(&p, &a, 4);
  return p;
}
template <typename P>
__device__ __forceinline__ uint32_t bits(const P& p) {
  uint32_t a;
  memcpy(&a, &p, 4);
  return a;
}

// ---- vectors of 16 bytes ------------------------------------------------------------------------------------------------------------------
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr float kMasked = -1e37f, kLow = -1e30f;  // what masked values are raised to; below kLow a row's maximum makes it a special one
  static __device__ __forceinline__ uint4 raised(const uint4& w) {
    return make_uint4(__float_as_uint(max_nan(__uint_as_float(w.x), kMasked)), __float_as_uint(max_nan(__uint_as_float(w.y), kMasked)),
                      __float_as_uint(max_nan(__uint_as_float(w.z), kMasked)), __float_as_uint(max_nan(__uint_as_float(w.w), kMasked)));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    float x[N];
    unpack(w, x);
    return most(w, x);
  }
  static __device__ __forceinline__ float most(const uint4&, const float (&x)[4]) { return max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3])); }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ float to(float x) { return x; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr float kMasked = -9.96921e36f, kLow = -1e30f;
  static __device__ __forceinline__ uint4 raised(const uint4& w) {
    const __nv_bfloat162 low = __float2bfloat162_rn(kMasked);
    auto up = [&](uint32_t a) { return bits(__hmax2_nan(halves<__nv_bfloat162>(a), low)); };
    return make_uint4(up(w.x), up(w.y), up(w.z), up(w.w));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(a[i] << 16), x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const float unused[8] = {};
    return most(w, unused);
  }
  static __device__ __forceinline__ float most(const uint4& w, const float (&)[8]) {
    using P = __nv_bfloat162;
    const P m = __hmax2_nan(__hmax2_nan(halves<P>(w.x), halves<P>(w.y)), __hmax2_nan(halves<P>(w.z), halves<P>(w.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    return make_uint4(bits(__floats2bfloat162_rn(x[0], x[1])), bits(__floats2bfloat162_rn(x[2], x[3])), bits(__floats2bfloat162_rn(x[4], x[5])),
                      bits(__floats2bfloat162_rn(x[6], x[7])));
  }
  static __device__ __forceinline__ __nv_bfloat16 to(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr float kMasked = -65504.f, kLow = -3e4f;
  static __device__ __forceinline__ uint4 raised(const uint4& w) {
    const __half2 low = __float2half2_rn(kMasked);
    auto up = [&](uint32_t a) { return bits(__hmax2_nan(halves<__half2>(a), low)); };
    return make_uint4(up(w.x), up(w.y), up(w.z), up(w.w));
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(halves<__half2>(a[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const float unused[8] = {};
    return most(w, unused);
  }
  static __device__ __forceinline__ float most(const uint4& w, const float (&)[8]) {
    using P = __half2;
    const P m = __hmax2_nan(__hmax2_nan(halves<P>(w.x), halves<P>(w.y)), __hmax2_nan(halves<P>(w.z), halves<P>(w.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    return make_uint4(bits(__floats2half2_rn(x[0], x[1])), bits(__floats2half2_rn(x[2], x[3])), bits(__floats2half2_rn(x[4], x[5])), bits(__floats2half2_rn(x[6], x[7])));
  }
  static __device__ __forceinline__ __half to(float x) { return __float2half_rn(x); }
};

// A row as [head scalars | vectors | tail scalars]: the vectors start at a 16-byte boundary.
struct Shape {
  int head, vecs, tail;
};
template <typename T>
__device__ __forceinline__ Shape shape_of(const T* row, int vocab) {
  Shape s;
  s.head = min(vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  s.vecs = (vocab - s.head) / Vec<T>::N;
  s.tail = vocab - s.head - s.vecs * Vec<T>::N;
  return s;
}

// What one thread writes when the sums of a row are known.
struct RowResult {
  float m, log_s, logprob, entropy;  // log sum e^x = m + log_s: their sum in one number would lose 2^-24 of m
};
__device__ __forceinline__ RowResult finish(const Sums& a, long long target, long long total, float x_target) {
  RowResult r;
  const float log_s = logf(a.s);
  r.m = a.m;
  r.log_s = log_s;
  r.entropy = log_s - kLn2 * a.t / a.s;
  r.logprob = target < 0 ? 0.f : (target >= total ? __int_as_float(0x7fc00000) : (x_target - a.m) - log_s);
  return r;
}

constexpr int kGroups = 64, kRoom = 512;
template <int WARPS>
struct FwdSmem {
  FastSums fast[WARPS];
  Sums warp[WARPS];
  Sums rank[kMaxCluster];                          // in the cluster's first CTA
  unsigned long long group[kGroups];               // the largest key of each group of threads
  unsigned long long found[kRoom];                 // candidates
  unsigned long long best[kMaxCluster][kMaxTopLogprobs];  // in the cluster's first CTA: the best of each CTA, in order
  unsigned long long bound;
  int n_threads, n_found;
  uint16_t threads[WARPS * 32];                    // those that may hold a candidate
  float m, log_s;
  bool special;
};

template <typename T, int WARPS, bool TOP>
__global__ void __launch_bounds__(WARPS * 32, 48 / WARPS) token_logprobs_kernel(const LogprobParams p, int cluster) {
  constexpr int N = Vec<T>::N, kThreads = WARPS * 32, U = 4;
  __shared__ FwdSmem<WARPS> sm;
  if (cluster > 1) ptx::cluster_arrive();  // the first CTA's shared memory is written to only after it has started
  ptx::griddep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = (int)(blockIdx.x / cluster), rank = (int)(blockIdx.x - (unsigned)r * cluster);
  const T* row = static_cast<const T*>(p.logits) + (size_t)r * p.stride;
  const Shape sh = shape_of(row, p.vocab);
  const int v0 = (int)((long long)sh.vecs * rank / cluster), v1 = (int)((long long)sh.vecs * (rank + 1) / cluster);
  const T* vec0 = row + sh.head;

  FastSums a = fast_nothing();
  float top = 0.f;     // the thread's largest and the vector that it is in
  int top_vec = -1;
  auto take = [&](const uint4& w, int v) {
    float x[N];
    const uint4 y = Vec<T>::raised(w);
    Vec<T>::unpack(y, x);
    const float most = Vec<T>::most(y, x);
    if constexpr (TOP) {
      // (equal to or below kMasked: the vector's own largest)
      const float m = most <= Vec<T>::kMasked ? Vec<T>::largest(w) : most;
      if (top_vec < 0 || m > top || (m != m && top == top)) top = m, top_vec = v;
    }
    raise_to(a, most);
#pragma unroll
    for (int i = 0; i < N; ++i) add(a, x[i]);
  };
  int v = v0 + tid;
  for (; v + (U - 1) * kThreads < v1; v += U * kThreads) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = ptx::ld_nc_v4(vec0 + (size_t)(v + u * kThreads) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) take(w[u], v + u * kThreads);
  }
  for (; v < v1; v += kThreads) take(ptx::ld_nc_v4(vec0 + (size_t)v * N), v);
  // the scalars at both ends of the row: one each for the first threads of two warps of the first CTA
  int extra = -1;
  if (rank == 0) {
    if (tid < sh.head) extra = tid;
    if (tid >= 32 && tid - 32 < sh.tail) extra = sh.head + sh.vecs * N + tid - 32;
  }
  float x_extra = 0.f;
  if (extra >= 0) {
    x_extra = Vec<T>::one(row + extra);
    const float x = max_nan(x_extra, Vec<T>::kMasked);
    raise_to(a, x);
    add(a, x);
  }

  // ---- alternatives of this CTA's share -----------------------------------------------------------------------------------------------------
  if constexpr (TOP) {
    const int K = p.top;
    // a thread's key has the last element of the vector that its largest value is in, so that all of that vector's equal ones reach it
    const unsigned long long mine = top_vec >= 0 ? key_of(top, (uint32_t)(sh.head + top_vec * N + N - 1)) : 0;
    unsigned long long g = mine;
#pragma unroll
    for (int x = kThreads / kGroups / 2; x; x >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, g, x);
      g = other > g ? other : g;
    }
    if (tid % (kThreads / kGroups) == 0) sm.group[tid / (kThreads / kGroups)] = g;
    if (tid == 0) sm.n_threads = sm.n_found = 0, sm.bound = 0;
    if (tid < kMaxTopLogprobs) sm.best[rank][tid] = 0;
    __syncthreads();
    if (tid < kGroups) {
      const unsigned long long k = sm.group[tid];
      if (k != 0 && rank_of(sm.group, kGroups, k) == K - 1) sm.bound = k;  // (0, with fewer than K groups that have anything)
    }
    __syncthreads();
    unsigned long long bound = sm.bound;
    if (mine != 0 && mine >= bound) sm.threads[atomicAdd(&sm.n_threads, 1)] = (uint16_t)tid;
    __syncthreads();
    const int each = (v1 - v0 + kThreads - 1) / kThreads, items = sm.n_threads * each;  // vectors of a thread, and of all these
    int n;
    while (true) {
      auto put = [&](unsigned long long k) {
        if (k >= bound) {
          const int at = atomicAdd(&sm.n_found, 1);
          if (at < kRoom) sm.found[at] = k;
        }
      };
      if (extra >= 0) put(key_of(x_extra, (uint32_t)extra));
      for (int i0 = tid; i0 < items; i0 += U * kThreads) {
        int at[U];
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * kThreads;
          at[u] = i < items ? v0 + sm.threads[i / each] + i % each * kThreads : v1;
          if (at[u] < v1) w[u] = ptx::ld_nc_v4(vec0 + (size_t)at[u] * N);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (at[u] >= v1 || ordered(Vec<T>::largest(w[u])) < (uint32_t)(bound >> 32)) continue;
          float x[N];
          Vec<T>::unpack(w[u], x);
#pragma unroll
          for (int e = 0; e < N; ++e) put(key_of(x[e], (uint32_t)(sh.head + at[u] * N + e)));
        }
      }
      __syncthreads();
      n = sm.n_found;
      if (n <= kRoom) break;
      // more than there is room for: the K-th best of those that found room, and again
      for (int i = tid; i < kRoom; i += kThreads)
        if (rank_of(sm.found, kRoom, sm.found[i]) == K - 1) sm.bound = sm.found[i];
      __syncthreads();
      bound = sm.bound;
      if (tid == 0) sm.n_found = 0;
      __syncthreads();
    }
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long k = sm.found[i];
      const int place = rank_of(sm.found, n, k);
      if (place < K) sm.best[rank][place] = k;
    }
    __syncthreads();
  }

  // ---- sums of the CTA, then of the cluster ----------------------------------------------------------------------------------------------------
  auto over_warp = [&](auto a) {
#pragma unroll
    for (int x = 16; x; x >>= 1) {
      auto b = a;
      b.m = __shfl_xor_sync(0xffffffffu, a.m, x);
      b.s = __shfl_xor_sync(0xffffffffu, a.s, x);
      b.t = __shfl_xor_sync(0xffffffffu, a.t, x);
      a = join(a, b);
    }
    return a;
  };
  a = over_warp(a);
  if (lane == 0) sm.fast[warp] = a;
  __syncthreads();
  if (warp == 0) {  // WARPS numbers, over the lanes again
    a = over_warp(lane < WARPS ? sm.fast[lane] : fast_nothing());
    if (lane == 0) sm.warp[0] = natural(a);
  }
  if (cluster > 1) {
    ptx::cluster_wait();
    if (tid == 0) {
      const Sums mine = sm.warp[0];
      const uint32_t dst = ptx::mapa(ptx::smem_u32(&sm.rank[rank]), 0);
      ptx::st_cluster_f32(dst, mine.m);
      ptx::st_cluster_f32(dst + 4, mine.s);
      ptx::st_cluster_f32(dst + 8, mine.t);
    }
    if (TOP && rank > 0 && tid < kMaxTopLogprobs) {
      const unsigned long long k = sm.best[rank][tid];
      const uint32_t dst = ptx::mapa(ptx::smem_u32(&sm.best[rank][tid]), 0);
      ptx::st_cluster_f32(dst, __uint_as_float((uint32_t)k));
      ptx::st_cluster_f32(dst + 4, __uint_as_float((uint32_t)(k >> 32)));
    }
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (rank != 0) return;
  }
  Sums sum = nothing();
  if (tid == 0) {
    sum = cluster > 1 ? sm.rank[0] : sm.warp[0];
    for (int w = 1; w < cluster; ++w) sum = join(sum, sm.rank[w]);
    sm.special = !(sum.s > 0.f && sum.s < INFINITY && fabsf(sum.t) < INFINITY && sum.m > Vec<T>::kLow && sum.m < kFar && sum.m > -kFar);
  }
  __syncthreads();
  if (sm.special) {  // the whole row once more, value by value
    sum = nothing();
    for (unsigned i = tid; i < (unsigned)p.vocab; i += kThreads) {  // (i + kThreads may pass 2^31)
      const float x = Vec<T>::one(row + i);
      if (!(x - sum.m <= kLag)) rebase(sum, x);
      add(sum, x);
    }
    sum = over_warp(sum);
    if (lane == 0) sm.warp[warp] = sum;
    __syncthreads();
    if (tid == 0)
      for (int w = 1; w < WARPS; ++w) sum = join(sum, sm.warp[w]);
  }
  if (tid == 0) {
    const long long target = p.targets[r], at = target - p.vocab_base;
    const bool here = target >= 0 && at >= 0 && at < p.vocab;
    const float xt = here ? Vec<T>::one(row + at) : __uint_as_float(kAbsent);
    if (p.partial) {
      float* out = p.partial + (size_t)r * (4 + 2 * p.top);
      out[0] = sum.m, out[1] = sum.s, out[2] = sum.t, out[3] = xt;
    } else {
      const RowResult f = finish(sum, target, p.vocab_total, xt);
      reinterpret_cast<float2*>(p.lse)[r] = make_float2(f.m, f.log_s);
      p.logprob[r] = f.logprob;
      p.entropy[r] = f.entropy;
      sm.m = f.m;
      sm.log_s = f.log_s;
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const int K = p.top;
    for (int i = tid; i < cluster * K; i += kThreads) {
      const int c = i / K, e = i - c * K;
      const unsigned long long k = sm.best[c][e];
      if (k == 0 && cluster > 1) continue;  // (a row that is split has K real ones; a shard with fewer columns than K is not split)
      int place = e;                        // better ones of its own CTA, and of the others, which are in order too
#pragma unroll 4
      for (int w = 0; w < cluster; ++w) {
        int at = 0;
#pragma unroll
        for (int step = kMaxTopLogprobs / 2; step; step >>= 1) at += sm.best[w][at + step - 1] > k ? step : 0;
        at += sm.best[w][at] > k;
        place += w == c ? 0 : at;
      }
      if (place >= K) continue;
      if (p.partial) {
        float* out = p.partial + (size_t)r * (4 + 2 * K) + 4;
        out[place] = k ? value_of(k) : -INFINITY;
        out[K + place] = __int_as_float(k ? (int)(p.vocab_base + index_of(k)) : -1);
      } else {
        p.top_logprobs[(size_t)r * K + place] = (value_of(k) - sm.m) - sm.log_s;
        p.top_ids[(size_t)r * K + place] = p.vocab_base + index_of(k);
      }
    }
  }
}

// One CTA a row: a few numbers for every shard.
constexpr int kMergeThreads = 128, kMaxShards = 64;
__global__ void __launch_bounds__(kMergeThreads) merge_shards_kernel(const LogprobMergeParams p) {
  __shared__ unsigned long long keys[kMaxShards * kMaxTopLogprobs];
  __shared__ float s_m, s_log_s;
  ptx::griddep_wait();
  const int r = blockIdx.x, tid = threadIdx.x, K = p.top, words = 4 + 2 * K;
  const float* mine = p.partials + (size_t)r * words;
  const size_t step = (size_t)p.rows * words;
  if (tid == 0) {
    Sums a = nothing();
    float xt = __uint_as_float(kAbsent);
    for (int w = 0; w < p.shards; ++w) {
      const float* x = mine + w * step;
      Sums b;
      b.m = x[0], b.s = x[1], b.t = x[2];
      a = join(a, b);
      if (__float_as_uint(x[3]) != kAbsent) xt = x[3];
    }
    const RowResult f = finish(a, p.targets[r], p.vocab_total, xt);
    reinterpret_cast<float2*>(p.lse)[r] = make_float2(f.m, f.log_s);
    s_m = f.m;
    s_log_s = f.log_s;
    p.logprob[r] = f.logprob;
    p.entropy[r] = f.entropy;
  }
  const int n = p.shards * K;
  for (int i = tid; i < n; i += kMergeThreads) {
    const float* x = mine + (i / K) * step + 4 + i % K;
    const int id = __float_as_int(x[K]);
    keys[i] = id < 0 ? 0 : key_of(x[0], (uint32_t)id);
  }
  __syncthreads();
  for (int i = tid; i < n; i += kMergeThreads) {
    const unsigned long long k = keys[i];
    if (k == 0) continue;
    int place = 0;
    for (int j = 0; j < n && place < K; ++j) place += keys[j] > k;
    if (place < K) {
      p.top_logprobs[(size_t)r * K + place] = (value_of(k) - s_m) - s_log_s;
      p.top_ids[(size_t)r * K + place] = index_of(k);
    }
  }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------------------------
constexpr int kBwdThreads = 256, kBwdVecs = 4;

struct RowGrad {
  float m, log_s, entropy, whole, g_entropy;
};
__device__ __forceinline__ float grad_of(const RowGrad& g, float x) {
  const float lp = (x - g.m) - g.log_s, pr = ex2(lp * kLog2e);
  const float inner = g.whole + g.g_entropy * (lp + g.entropy);
  return pr == 0.f ? 0.f : -pr * inner;  // (-inf has no part in it)
}

template <typename T>
__global__ void __launch_bounds__(kBwdThreads) token_logprobs_backward_kernel(const LogprobBackwardParams p) {
  constexpr int N = Vec<T>::N;
  __shared__ RowGrad s_g;
  ptx::griddep_wait();  // (and no early start for the kernel behind it, which may take this gradient for a weight)
  const int tid = threadIdx.x, r = blockIdx.x;
  const T* row = static_cast<const T*>(p.logits) + (size_t)r * p.stride;
  T* out = static_cast<T*>(p.grad) + (size_t)r * p.grad_stride;
  const long long target = p.targets[r];
  const float g_lp = p.g_logprob && target >= 0 ? p.g_logprob[r] : 0.f;
  if (tid < 32) {
    float sum = p.g_top && tid < p.top ? p.g_top[(size_t)r * p.top + tid] : 0.f;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (tid == 0) {
      s_g.m = p.lse[2 * r];
      s_g.log_s = p.lse[2 * r + 1];
      s_g.entropy = p.entropy[r];
      s_g.whole = g_lp + sum;
      s_g.g_entropy = p.g_entropy ? p.g_entropy[r] : 0.f;
      if (target >= p.vocab_total && p.g_logprob) s_g.whole = __int_as_float(0x7fc00000);  // its log-probability is NaN
    }
  }
  __syncthreads();
  const RowGrad g = s_g;
  const Shape sh = shape_of(row, p.vocab);
  const T* vec0 = row + sh.head;
  const int first = (int)blockIdx.y * kBwdThreads * kBwdVecs, last = min(sh.vecs, first + kBwdThreads * kBwdVecs);
  uint4 w[kBwdVecs];
#pragma unroll
  for (int u = 0; u < kBwdVecs; ++u)
    if (first + tid + u * kBwdThreads < last) w[u] = ptx::ld_nc_v4(vec0 + (size_t)(first + tid + u * kBwdThreads) * N);
#pragma unroll
  for (int u = 0; u < kBwdVecs; ++u) {
    const int v = first + tid + u * kBwdThreads;
    if (v < last) {
      float x[N];
      Vec<T>::unpack(w[u], x);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = grad_of(g, x[i]);
      *reinterpret_cast<uint4*>(out + sh.head + (size_t)v * N) = Vec<T>::pack(x);
    }
  }
  // the ends of the row, with its first piece
  int lo = sh.head + min(first, sh.vecs) * N, hi = sh.head + last * N;
  if (blockIdx.y == 0) {
    if (tid < sh.head) out[tid] = Vec<T>::to(grad_of(g, Vec<T>::one(row + tid)));
    lo = 0;
  }
  if (blockIdx.y == gridDim.y - 1) {
    if (tid < sh.tail) {
      const int at = sh.head + sh.vecs * N + tid;
      out[at] = Vec<T>::to(grad_of(g, Vec<T>::one(row + at)));
    }
    hi = p.vocab;
  }
  __syncthreads();
  // the given token and the alternatives: the same element may be named several times, so each writes the whole of what it gets
  if (tid <= p.top) {
    auto id_of = [&](int j) { return (j == p.top ? (target < 0 ? -1ll : target) : (p.g_top ? p.top_ids[(size_t)r * p.top + j] : -1ll)); };
    auto of = [&](int j) { return j == p.top ? g_lp : p.g_top[(size_t)r * p.top + j]; };
    const long long id = id_of(tid), at = id - p.vocab_base;
    if (id >= 0 && at >= lo && at < hi) {
      float sum = 0.f;
      for (int j = 0; j <= p.top; ++j)
        if (id_of(j) == id) sum += of(j);
      out[at] = Vec<T>::to(grad_of(g, Vec<T>::one(row + at)) + sum);
    }
  }
}

template <typename T, int WARPS>
cudaError_t launch_forward(const LogprobParams& p, int cluster, cudaStream_t stream) {
  auto kern = p.top > 0 ? token_logprobs_kernel<T, WARPS, true> : token_logprobs_kernel<T, WARPS, false>;
  static DeviceOnce wide[2];
  if (cluster > 8 && wide[p.top > 0].pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    wide[p.top > 0].done();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows * cluster);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, cluster);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}

template <typename T>
cudaError_t forward(const LogprobParams& p, cudaStream_t stream) {
  const long long vecs = p.vocab / Vec<T>::N;
  if (vecs <= 512) return launch_forward<T, 4>(p, 1, stream);
  // a cluster for a row while the CTAs (six of 256 threads on an SM) do not fill the GPU and each still has four vectors for every thread
  int cluster = 1;
  while (cluster < kMaxCluster && (long long)p.rows * cluster * 2 <= 4 * 148 && vecs >= kClusterVecs * cluster * 2) cluster *= 2;
  return launch_forward<T, 8>(p, cluster, stream);
}

template <typename T>
cudaError_t backward(const LogprobBackwardParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const long long per = (long long)kBwdThreads * kBwdVecs * Vec<T>::N;
  cfg.gridDim = dim3((unsigned)p.rows, (unsigned)std::max(1ll, (p.vocab + per - 1) / per));
  cfg.blockDim = dim3(kBwdThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  cudaError_t e = cudaLaunchKernelEx(&cfg, token_logprobs_backward_kernel<T>, p);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}

bool sizes_ok(int rows, int vocab, int top, long long base, long long total) {
  return rows >= 0 && vocab >= 1 && top >= 0 && top <= kMaxTopLogprobs && base >= 0 && base + vocab <= total && total <= 0x7fffffffll && top <= total;
}

}  // namespace

cudaError_t token_logprobs(const LogprobParams& p, cudaStream_t stream) {
  if (!sizes_ok(p.rows, p.vocab, p.top, p.vocab_base, p.vocab_total) || (long long)p.rows * kMaxCluster > 0x7fffffffll) return cudaErrorInvalidValue;
  if (!p.partial && (p.vocab_base != 0 || p.vocab != p.vocab_total)) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  if (p.dtype == 0) return forward<__nv_bfloat16>(p, stream);
  if (p.dtype == 1) return forward<__half>(p, stream);
  return p.dtype == 2 ? forward<float>(p, stream) : cudaErrorInvalidValue;
}

cudaError_t token_logprobs_merge(const LogprobMergeParams& p, cudaStream_t stream) {
  if (p.rows < 0 || p.shards < 1 || p.shards > kMaxShards || p.top < 0 || p.top > kMaxTopLogprobs || p.top > p.vocab_total) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  cudaError_t e = cudaLaunchKernelEx(&cfg, merge_shards_kernel, p);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}

cudaError_t token_logprobs_backward(const LogprobBackwardParams& p, cudaStream_t stream) {
  if (!sizes_ok(p.rows, p.vocab, p.top, p.vocab_base, p.vocab_total)) return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  const int size = p.dtype == 2 ? 4 : 2;
  if (p.vocab / (kBwdThreads * kBwdVecs * 16 / size) >= 65535) return cudaErrorInvalidValue;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p.logits), b = reinterpret_cast<uintptr_t>(p.grad);
  if (((a ^ b) & 15) != 0 || ((p.stride - p.grad_stride) * size) % 16 != 0) return cudaErrorInvalidValue;
  if (p.dtype == 0) return backward<__nv_bfloat16>(p, stream);
  if (p.dtype == 1) return backward<__half>(p, stream);
  return p.dtype == 2 ? backward<float>(p, stream) : cudaErrorInvalidValue;
}

}  // namespace ccl
