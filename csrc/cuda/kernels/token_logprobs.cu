// Log-probability of given tokens, entropy and the best alternatives of each row of logits, in one pass; the gradient in another.
//
// Forward. A thread keeps a reference m, sum e^(x - m) and sum e^(x - m) (x - m); they join into log sum exp and the entropy
// H = log s - t / s. The reference is raised only when a value passes it by more than kLag, so the loop has no dependent maximum.
// Bound by memory (one read of the logits) as long as the exponentials keep up: one per element, 16 a clock and SM.
// A row belongs to one CTA; few rows are split over the CTAs of a cluster, which push their sums into the first one's shared memory.
//
// Alternatives. Nothing is sorted while the row streams by: every thread only remembers its largest value and the vector that it came from.
// With K of these as (value, lowest index first) keys, the K-th largest over all threads is a bound that K elements of the row reach, and only
// the threads whose own largest reaches it, exactly K of them, can hold an element that does. Those threads' elements (K out of 512
// shares of the row) are read once more, from L2, into a sorted list per warp (lane i holds the i-th best), and the lists are joined
// by counting for every candidate how many are better. Keys are unique, so the result does not depend on any order of execution, and
// rows of equal or masked values cost no more than others.
//
// Values that are masked with -inf or with the type's lowest value take no part in the sums (0 * inf is not computed); a row with a NaN or
// with +inf, or with nothing but -inf, has a NaN log-probability as log_softmax has.
#include "token_logprobs.h"

#include "gemm.h"
#include "ptx.cuh"

#include <algorithm>
#include <cfloat>

namespace ccl {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLag = 6.f;
constexpr int kMaxCluster = 16;
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

__device__ __forceinline__ unsigned long long exchange(unsigned long long k, int x, bool larger) {
  const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, x);
  return (other > k) == larger ? other : k;
}
// Sorts a bitonic sequence over the lanes, largest first.
__device__ __forceinline__ unsigned long long sort_bitonic(unsigned long long k, int lane) {
#pragma unroll
  for (int x = 16; x; x >>= 1) k = exchange(k, x, (lane & x) == 0);
  return k;
}
__device__ __forceinline__ unsigned long long sort_warp(unsigned long long k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int x = size >> 1; x; x >>= 1) k = exchange(k, x, ((lane & x) == 0) == ((lane & size) == 0));
  return k;
}
// Puts `cand` (the same in all lanes) into the list that the lanes hold, largest first; the last one falls out.
__device__ __forceinline__ void insert(unsigned long long& list, unsigned long long cand, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, list > cand));
  const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
  list = lane < at ? list : (lane == at ? cand : up);
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

// ---- vectors of 16 bytes ------------------------------------------------------------------------------------------------------------------
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
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
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[8]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(a[i] << 16), x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ float most(const uint4& w, const float (&)[8]) {
    const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(a[0], a[1]), __hmax2_nan(a[2], a[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint4 w;
    __nv_bfloat162* a = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    return w;
  }
  static __device__ __forceinline__ __nv_bfloat16 to(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[8]) {
    const __half2* a = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(a[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float most(const uint4& w, const float (&)[8]) {
    const __half2* a = reinterpret_cast<const __half2*>(&w);
    const __half2 m = __hmax2_nan(__hmax2_nan(a[0], a[1]), __hmax2_nan(a[2], a[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint4 w;
    __half2* a = reinterpret_cast<__half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    return w;
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
  float lse, logprob, entropy;
};
__device__ __forceinline__ RowResult finish(const Sums& a, long long target, long long total, float x_target) {
  RowResult r;
  const float log_s = logf(a.s);
  r.lse = a.m + log_s;
  r.entropy = log_s - kLn2 * a.t / a.s;
  r.logprob = target < 0 ? 0.f : (target >= total ? __int_as_float(0x7fc00000) : x_target - r.lse);
  return r;
}

template <int WARPS>
struct FwdSmem {
  Sums warp[WARPS];
  Sums rank[kMaxCluster];                               // in the cluster's first CTA
  unsigned long long lists[WARPS][32];                  // the threads' largest; later the warps' candidates
  unsigned long long best[kMaxCluster][32];             // in the cluster's first CTA: candidates of each CTA
  unsigned long long bound;
  int count[WARPS];
  float lse;
};

template <typename T, int WARPS, bool TOP>
__global__ void __launch_bounds__(WARPS * 32) token_logprobs_kernel(const LogprobParams p, int cluster) {
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

  Sums a = nothing();
  float top = 0.f;     // the thread's largest and the vector that it is in
  int top_vec = -1;
  auto take = [&](const uint4& w, int v) {
    float x[N];
    Vec<T>::unpack(w, x);
    const float most = Vec<T>::most(w, x);
    if (!(most - a.m <= kLag)) {
      if (TOP && (top_vec < 0 || most > top || (most != most && top == top))) top = most, top_vec = v;
      rebase(a, most);
    } else if (TOP && (top_vec < 0 || most > top)) {
      top = most, top_vec = v;
    }
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
    if (!(x_extra - a.m <= kLag)) rebase(a, x_extra);
    add(a, x_extra);
  }

  // ---- alternatives of this CTA's share -----------------------------------------------------------------------------------------------------
  if constexpr (TOP) {
    const int K = p.top;
    unsigned long long mine = top_vec >= 0 ? key_of(top, (uint32_t)top_vec) : 0;
    unsigned long long k = sort_warp(mine, lane);
    sm.lists[warp][lane] = k;
#pragma unroll
    for (int half = WARPS / 2; half; half >>= 1) {
      __syncthreads();
      if (warp < half) {
        const unsigned long long other = sm.lists[warp + half][31 - lane];
        k = sort_bitonic(k > other ? k : other, lane);
        sm.lists[warp][lane] = k;
      }
    }
    if (warp == 0 && lane == K - 1) sm.bound = k;
    __syncthreads();
    const unsigned long long bound = sm.bound;  // 0 when fewer than K threads have anything
    unsigned long long list = 0;
    auto offer = [&](unsigned long long cand) {  // 0: none
      unsigned left;
      while ((left = __ballot_sync(0xffffffffu, cand > __shfl_sync(0xffffffffu, list, K - 1)))) {
        const int src = __ffs(left) - 1;
        insert(list, __shfl_sync(0xffffffffu, cand, src), lane);
        if (lane == src) cand = 0;
      }
    };
    for (unsigned who = __ballot_sync(0xffffffffu, mine != 0 && mine >= bound); who; who &= who - 1) {
      const int first = v0 + warp * 32 + __ffs(who) - 1;
      for (int base = first; base < v1; base += 32 * kThreads) {
        const int vi = base + lane * kThreads;
        float x[N];
        if (vi < v1) Vec<T>::unpack(ptx::ld_nc_v4(vec0 + (size_t)vi * N), x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          // what is below the bound's value is no candidate
          unsigned long long cand = vi < v1 ? key_of(x[i], (uint32_t)(sh.head + vi * N + i)) : 0;
          if ((uint32_t)(cand >> 32) < (uint32_t)(bound >> 32)) cand = 0;
          offer(cand);
        }
      }
    }
    if (rank == 0 && warp < 2) offer(extra >= 0 ? key_of(x_extra, (uint32_t)extra) : 0);
    // the K best of the warps' lists: a candidate's place is the number of better ones
    if (lane >= K) list = 0;
    sm.lists[warp][lane] = list;  // (all have read `bound`; nobody reads the lists of the sort any more)
    if (lane == 0) sm.count[warp] = 0;
    __syncwarp();
    if (lane < K && list == 0) atomicAdd(&sm.count[warp], 1);
    __syncthreads();
    if (tid < kMaxTopLogprobs) sm.best[rank][tid] = 0;
    __syncthreads();
    if (list != 0) {
      int place = lane;  // better ones of its own list
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) continue;
        const int n = K - sm.count[w];
        for (int i = 0; i < n && sm.lists[w][i] > list; ++i) ++place;
      }
      if (place < K) sm.best[rank][place] = list;
    }
    __syncthreads();
  }

  // ---- sums of the CTA, then of the cluster ----------------------------------------------------------------------------------------------------
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, x);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, x);
    b.t = __shfl_xor_sync(0xffffffffu, a.t, x);
    a = join(a, b);
  }
  if (lane == 0) sm.warp[warp] = a;
  __syncthreads();
  if (cluster > 1) {
    ptx::cluster_wait();
    if (tid == 0) {
      a = sm.warp[0];
      for (int w = 1; w < WARPS; ++w) a = join(a, sm.warp[w]);
      const uint32_t dst = ptx::mapa(ptx::smem_u32(&sm.rank[rank]), 0);
      ptx::st_cluster_f32(dst, a.m);
      ptx::st_cluster_f32(dst + 4, a.s);
      ptx::st_cluster_f32(dst + 8, a.t);
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
  if (tid == 0) {
    a = cluster > 1 ? sm.rank[0] : sm.warp[0];
    const int n = cluster > 1 ? cluster : WARPS;
    for (int w = 1; w < n; ++w) a = join(a, cluster > 1 ? sm.rank[w] : sm.warp[w]);
    const long long target = p.targets[r], at = target - p.vocab_base;
    const bool here = target >= 0 && at >= 0 && at < p.vocab;
    const float xt = here ? Vec<T>::one(row + at) : __uint_as_float(kAbsent);
    if (p.partial) {
      float* out = p.partial + (size_t)r * (4 + 2 * p.top);
      out[0] = a.m, out[1] = a.s, out[2] = a.t, out[3] = xt;
    } else {
      const RowResult f = finish(a, target, p.vocab_total, xt);
      p.lse[r] = f.lse;
      p.logprob[r] = f.logprob;
      p.entropy[r] = f.entropy;
      sm.lse = f.lse;
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const int K = p.top;
    for (int i = tid; i < cluster * 32; i += kThreads) {
      const int c = i >> 5;
      const unsigned long long k = sm.best[c][i & 31];
      if ((i & 31) >= K) continue;
      int place = i & 31;
      if (k != 0)
        for (int w = 0; w < cluster; ++w) {
          if (w == c) continue;
          for (int e = 0; e < K && sm.best[w][e] > k; ++e) ++place;
        }
      else if (cluster > 1)
        continue;  // (there are K real ones: the vocabulary has at least K ids, and a shard is checked below)
      if (place >= K) continue;
      if (p.partial) {
        float* out = p.partial + (size_t)r * (4 + 2 * K) + 4;
        out[place] = k ? value_of(k) : -INFINITY;
        out[K + place] = __int_as_float(k ? (int)(p.vocab_base + index_of(k)) : -1);
      } else {
        p.top_logprobs[(size_t)r * K + place] = value_of(k) - sm.lse;
        p.top_ids[(size_t)r * K + place] = p.vocab_base + index_of(k);
      }
    }
  }
}

// One CTA a row: a few numbers for every shard.
constexpr int kMergeThreads = 128, kMaxShards = 64;
__global__ void __launch_bounds__(kMergeThreads) merge_shards_kernel(const LogprobMergeParams p) {
  __shared__ unsigned long long keys[kMaxShards * kMaxTopLogprobs];
  __shared__ float s_lse;
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
    p.lse[r] = s_lse = f.lse;
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
      p.top_logprobs[(size_t)r * K + place] = value_of(k) - s_lse;
      p.top_ids[(size_t)r * K + place] = index_of(k);
    }
  }
}

// ---- gradient -------------------------------------------------------------------------------------------------------------------------------
constexpr int kBwdThreads = 256, kBwdVecs = 4;

struct RowGrad {
  float lse, entropy, whole, g_entropy;
};
__device__ __forceinline__ float grad_of(const RowGrad& g, float x) {
  const float lp = x - g.lse, pr = ex2(lp * kLog2e);
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
      s_g.lse = p.lse[r];
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
  // a cluster for a row while the CTAs (two of 512 threads on an SM) do not fill the GPU and each still has a vector for every thread
  const long long vecs = p.vocab / Vec<T>::N;
  if (vecs <= 512) return launch_forward<T, 4>(p, 1, stream);
  int cluster = 1;
  while (cluster < kMaxCluster && (long long)p.rows * cluster * 2 <= 2 * 148 && vecs >= 512ll * cluster * 2) cluster *= 2;
  return launch_forward<T, 16>(p, cluster, stream);
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
