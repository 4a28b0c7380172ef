// Block tables and slot maps from request lengths, on the GPU: a decode step captured in a graph allocates its own pages.
//
// A prefix sum over the requests and then one entry for every token and every new page. The sums are small (a few words a request),
// so every CTA makes them for itself, in shared memory, and then writes its share of the entries, finding a token's request by binary
// search (1000 requests with 119702 new tokens: 12.5 us, half of it the two launches' sums; one cluster of sixteen for all of it took 13.0.
// Sixteen requests with 319 tokens: 4.7 us, less than the host's 7.5 for the call); what a plan changes in place (how much is held, the pool's state) is written by one CTA after all have read it: behind a
// barrier of the one cluster that a plan of ordinary size is, or by a second launch for a large one.
#include "kv_plan.h"

#include "gemm.h"
#include "ptx.cuh"

#include <algorithm>

namespace ccl {
namespace {

constexpr int kThreads = 1024;

// Inclusive sum over the CTA of one value a thread; `total` is the sum of all. s: 33 words.
__device__ __forceinline__ int block_scan(int v, int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, x);
    if (lane >= x) v += y;
  }
  __syncthreads();  // the previous use of s is over
  if (lane == 31) s[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = s[lane];
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, x);
      if (lane >= x) w += y;
    }
    s[lane] = w;
  }
  __syncthreads();
  total = s[31];
  return v + (warp > 0 ? s[warp - 1] : 0);
}
// The last r with from[r] <= i, for i < from[n]; entries of requests without anything are equal to the next one.
__device__ __forceinline__ int owner_of(const int* from, int n, int i) {
  int lo = 0, hi = n;  // from[lo] <= i < from[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

enum Mode { kAll, kEntries, kCommit };  // kAll: one cluster does both

template <int MODE>
__global__ void __launch_bounds__(kThreads) kv_plan_kernel(const KvPlanParams p) {
  extern __shared__ int dyn[];
  const int R = p.b.requests;
  int* s_start = dyn;            // [R + 1] first token
  int* s_base = s_start + R + 1; // [R + 1] first new page, counted over all requests
  int* s_held = s_base + R + 1;  // [R]
  __shared__ int s_scan[33];
  ptx::griddep_wait();
  const int tid = threadIdx.x;
  // indexes into the stack stay inside it whatever the state word says
  const int top = min(max(p.b.state[0], 0), p.b.capacity);
  long long blocks = 0, asked_blocks = 0, tokens = 0, asked_tokens = 0;  // sums over the chunks of requests before this one
  int refused = 0;
  for (int r0 = 0; r0 < R; r0 += kThreads) {
    const int r = r0 + tid;
    int len = -1, nt = 0, has = 0;
    if (r < R) {
      len = p.lengths[r];
      nt = p.new_tokens ? p.new_tokens[r] : 1;
      has = p.b.held[r];
    }
    const bool asks = len >= 0 && nt > 0;
    const long long want = asks ? ((long long)len + nt + p.block - 1) / p.block : 0;
    const bool fits = asks && want <= p.b.max_blocks && (long long)len + nt <= 0x7fffffffll;
    const int need = fits ? max(0, (int)want - max(has, 0)) : 0;
    int total;
    const int upto = block_scan(need, s_scan, total);  // at most 1024 * max_blocks
    const bool given = fits && (need == 0 || asked_blocks + upto <= top);
    asked_blocks += total;
    const int take = given ? need : 0;
    const int taken_upto = block_scan(take, s_scan, total);
    const long long base = blocks + taken_upto - take;
    blocks += total;
    // tokens: sums saturate at room + 1, which is all that matters of a sum that does not fit
    const int t = given ? min(nt, p.room + 1) : 0;
    const long long cap = (long long)p.room + 1;
    // (1024 values of up to room + 1 may pass 32 bits: halves)
    int total_lo, total_hi;
    const int lo_upto = block_scan(t & 0xffff, s_scan, total_lo), hi_upto = block_scan(t >> 16, s_scan, total_hi);
    const long long t_upto = lo_upto + ((long long)hi_upto << 16), t_total = total_lo + ((long long)total_hi << 16);
    const bool listed = given && asked_tokens + t_upto <= p.room;
    asked_tokens = min(asked_tokens + t_total, cap);
    const int mine = listed ? t : 0;
    const int listed_upto = block_scan(mine, s_scan, total);  // at most room
    if (r < R) {
      s_start[r] = (int)tokens + listed_upto - mine;
      s_base[r] = (int)base;
      s_held[r] = max(has, 0);
    }
    tokens += total;
    refused += __syncthreads_count(asks && !(p.room > 0 ? listed : given));
  }
  if (tid == 0) {
    s_start[R] = (int)tokens;
    s_base[R] = (int)blocks;
  }
  __syncthreads();
  const bool commits = MODE == kCommit || (MODE == kAll && blockIdx.x == 0);
  if (MODE == kAll && gridDim.x > 1) {  // everybody has read what is changed below
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (MODE != kCommit) {
    const int step = (int)gridDim.x * kThreads, first = (int)blockIdx.x * kThreads + tid;
    for (int i = first; i < (int)blocks; i += step) {
      const int r = owner_of(s_base, R, i);
      p.b.table[(size_t)r * p.b.max_blocks + s_held[r] + (i - s_base[r])] = p.b.free_blocks[top - 1 - i];
    }
    for (unsigned n = first; n < (unsigned)p.room; n += step) {  // (n + step may pass 2^31)
      const int i = (int)n;
      int r = -1, pos = -1, slot = -1;
      if (i < (int)tokens) {
        r = owner_of(s_start, R, i);
        pos = p.lengths[r] + (i - s_start[r]);
        const int col = pos / p.block;
        // a page that this plan hands out comes from the stack (its table entry may not be written yet)
        const int page = col < s_held[r] ? p.b.table[(size_t)r * p.b.max_blocks + col] : p.b.free_blocks[top - 1 - (s_base[r] + col - s_held[r])];
        slot = page * p.block + pos % p.block;
      }
      p.token_request[i] = r;
      p.positions[i] = pos;
      p.slots[i] = slot;
    }
    if (blockIdx.x == 0)
      for (int r = tid; r <= R; r += kThreads) p.starts[r] = s_start[r];
  }
  if (commits) {
    for (int r = tid; r < R; r += kThreads) {
      const int take = s_base[r + 1] - s_base[r];
      if (take > 0) p.b.held[r] = s_held[r] + take;
    }
    if (tid == 0) {
      p.b.state[0] = top - (int)blocks;
      p.b.state[1] = refused;
    }
  }
}

__global__ void __launch_bounds__(kThreads) kv_release_kernel(const uint8_t* finished, const KvBlocks b) {
  extern __shared__ int dyn[];
  const int R = b.requests;
  int* s_base = dyn;  // [R + 1]
  __shared__ int s_scan[33];
  ptx::griddep_wait();
  const int tid = threadIdx.x;
  const int top = min(max(b.state[0], 0), b.capacity);
  int blocks = 0;
  for (int r0 = 0; r0 < R; r0 += kThreads) {
    const int r = r0 + tid;
    const int n = r < R && finished[r] ? min(max(b.held[r], 0), b.max_blocks) : 0;
    int total;
    const int upto = block_scan(n, s_scan, total);
    if (r < R) s_base[r] = blocks + upto - n;
    blocks += total;
  }
  if (tid == 0) s_base[R] = blocks;
  __syncthreads();
  if (gridDim.x > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  const int step = (int)gridDim.x * kThreads;
  for (unsigned n = blockIdx.x * kThreads + tid; n < (unsigned)blocks; n += step) {
    const int i = (int)n, r = owner_of(s_base, R, i);
    int* entry = b.table + (size_t)r * b.max_blocks + (i - s_base[r]);
    const long long at = (long long)top + blocks - 1 - i;  // (counts that make no sense may add up to more than the pool, and to 2^31)
    if (at < b.capacity) b.free_blocks[at] = *entry;
    *entry = -1;
  }
  if (blockIdx.x == 0) {
    for (int r = tid; r < R; r += kThreads)
      if (finished[r]) b.held[r] = 0;
    if (tid == 0) b.state[0] = (int)min((long long)top + blocks, (long long)b.capacity);
  }
}

bool blocks_ok(const KvBlocks& b) {
  // sums of what requests hold, or ask for (at most max_blocks each), stay in 32 bits
  return b.requests >= 0 && b.requests <= kMaxPlanRequests && b.max_blocks >= 1 && (long long)std::max(b.requests, 1024) * b.max_blocks <= 0x7fffffffll && b.capacity >= 0;
}

template <typename F, typename... A>
cudaError_t go(F kern, int ctas, bool cluster, size_t smem, cudaStream_t stream, DeviceOnce& configured, A... args) {
  if (configured.pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * kMaxPlanRequests + 2) * 4);
    if (e != cudaSuccess) return e;
    configured.done();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  if (cluster && ctas > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = ctas;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}

}  // namespace

cudaError_t kv_plan(const KvPlanParams& p, cudaStream_t stream) {
  if (!blocks_ok(p.b) || p.room < 0 || p.room > 0x7ffffffe || p.block < 1 || (long long)p.b.capacity * p.block > 0x7fffffffll) return cudaErrorInvalidValue;
  static DeviceOnce all, entries, commit;
  const size_t smem = (3 * (size_t)p.b.requests + 2) * 4;
  const int one = 4 * kThreads;  // tokens that a CTA lists in four steps
  if (p.room <= 8 * one) {
    // a CTA for few tokens, a cluster of eight (the portable size) for more
    return go(kv_plan_kernel<kAll>, p.room <= one ? 1 : 8, true, smem, stream, all, p);
  }
  const int ctas = std::min(148, (p.room + one - 1) / one);
  cudaError_t e = go(kv_plan_kernel<kEntries>, ctas, false, smem, stream, entries, p);
  return e == cudaSuccess ? go(kv_plan_kernel<kCommit>, 1, false, smem, stream, commit, p) : e;
}

cudaError_t kv_release(const uint8_t* finished, const KvBlocks& b, cudaStream_t stream) {
  if (!blocks_ok(b)) return cudaErrorInvalidValue;
  if (b.requests == 0) return cudaSuccess;
  static DeviceOnce configured;
  const bool few = (long long)b.requests * b.max_blocks <= 4 * kThreads;
  return go(kv_release_kernel, few ? 1 : 8, true, ((size_t)b.requests + 1) * 4, stream, configured, finished, b);
}

}  // namespace ccl
