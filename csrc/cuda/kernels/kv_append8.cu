// Rotary embedding of prompt rows and their quantisation into the 8-bit cache's pages, one pass over the QKV projection.
//
// Bound by memory: q, k and v are read once, q and k written back rotated (bf16, for the prompt's own attention), k and v written as one
// byte each (16 x 1024 rows of 32 + 32 + 32 heads: 166 to 173 us, 4.7 to 4.9 TB/s; int8 180). A CTA takes `block` rows of the projection and a few heads of one kind (q, k or v). For k and v its unit is a cache block:
// one thread per 16 values (8 dims and the 8 that the rotation pairs them with) of a position, so that a whole block is in the registers
// of the CTA when its largest magnitude is known, and is read once. Rotary tables are loaded once for all heads of the CTA.
//
// Units. The rows of a request are consecutive; a unit starts at a row whose position starts a block, or that is a request's first. The
// CTA whose rows contain that start owns the unit. A unit that fills its block (with the tail's older values in front, when the request
// was in the middle of a block) goes to its page; one that does not goes to the tail. The first unit of a request may read the tail that
// its last unit writes, so the CTA of the first unit then writes the last one too, after its own.
#include "kv_cache8.cuh"

#include "gemm.h"

#include <algorithm>

namespace ccl {
namespace {

using namespace kv8;

__device__ __forceinline__ bool row_ok(const KvAppend8Params& p, int row) {
  const int r = p.requests[row], pos = p.positions[row];
  return r >= 0 && r < p.n_requests && pos >= 0 && pos < p.table_rows;
}

// Where the rows of `row`'s request end: behind `row` and inside the projection, whatever starts holds.
__device__ __forceinline__ int end_of(const KvAppend8Params& p, int request, int row) { return max(min(p.starts[request + 1], p.rows), row + 1); }

struct Unit {
  int row, n;        // its first row and how many
  int place;         // place of the first row in the block
  int request;
  int page;          // -1: outside the pool
};
// The unit that starts at `row`. Its rows stay inside the request and the rotary tables, whatever the arrays hold.
__device__ __forceinline__ Unit unit_at(const KvAppend8Params& p, int row) {
  Unit u;
  u.row = row;
  u.request = p.requests[row];
  const int pos = p.positions[row];
  u.place = pos & (p.cache.block - 1);
  u.n = min(min(end_of(p, u.request, row) - row, p.cache.block - u.place), p.table_rows - pos);
  const int slot = p.slots[row];
  u.page = slot < 0 ? -1 : slot / p.cache.block;
  if (u.page >= p.cache.num_blocks) u.page = -1;
  return u;
}

// D / 16 threads share a position: thread `j` has dims 8j .. 8j + 7 and those D / 2 further on. `there`: lo and hi hold them already.
template <int D, bool INT8, bool IS_K, int HEADS>
__device__ __forceinline__ void do_unit(const KvAppend8Params& p, const Unit& u, int kvh0, uint32_t (*s_amax)[32], bool there, uint4 (&lo)[HEADS], uint4 (&hi)[HEADS]) {
  constexpr int J = D / 16;
  const KvCache8& c = p.cache;
  const int tid = threadIdx.x, place = tid / J, j = tid - place * J;
  const int end = u.place + u.n;
  const bool full = end == c.block;
  const bool fresh = place >= u.place && place < end;
  const bool old = full && place < u.place;
  const size_t row = (size_t)u.row + place - u.place;
  __nv_bfloat16* tail0 = (IS_K ? c.k_tail : c.v_tail) + (((size_t)u.request * c.n_kv_heads + kvh0) * c.block + place) * D + j * 8;
  const size_t tail_step = (size_t)c.block * D;
  const __nv_bfloat16* src = p.qkv + row * p.qkv_stride + (size_t)(p.n_heads + (IS_K ? 0 : c.n_kv_heads) + kvh0) * D + j * 8;
  if (!there) {
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      lo[h] = hi[h] = make_uint4(0, 0, 0, 0);
      if ((fresh || old) && kvh0 + h < c.n_kv_heads) {
        const __nv_bfloat16* at = fresh ? src + h * D : tail0 + h * tail_step;
        lo[h] = *reinterpret_cast<const uint4*>(at);
        hi[h] = *reinterpret_cast<const uint4*>(at + D / 2);
      }
    }
  }
  if (IS_K && fresh) {
    const size_t pos = (size_t)p.positions[u.row] + place - u.place;
    const float4* cr = reinterpret_cast<const float4*>(p.cos + pos * (D / 2) + j * 8);
    const float4* sr = reinterpret_cast<const float4*>(p.sin + pos * (D / 2) + j * 8);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    __nv_bfloat16* dst = p.rotated + row * p.rotated_stride + (size_t)(p.n_heads + kvh0) * D + j * 8;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      if (kvh0 + h >= c.n_kv_heads) break;
      uint32_t* a = &lo[h].x;
      uint32_t* b = &hi[h].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0, y0, x1, y1;
        rotate(lo_f(a[i]), lo_f(b[i]), cs[2 * i], sn[2 * i], x0, y0);
        rotate(hi_f(a[i]), hi_f(b[i]), cs[2 * i + 1], sn[2 * i + 1], x1, y1);
        a[i] = pack_bf16(x0, x1);
        b[i] = pack_bf16(y0, y1);
      }
      *reinterpret_cast<uint4*>(dst + h * D) = lo[h];
      *reinterpret_cast<uint4*>(dst + h * D + D / 2) = hi[h];
    }
  }
  if (!full) {  // uniform
    if (fresh)
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        if (kvh0 + h >= c.n_kv_heads) break;
        *reinterpret_cast<uint4*>(tail0 + h * tail_step) = lo[h];
        *reinterpret_cast<uint4*>(tail0 + h * tail_step + D / 2) = hi[h];
      }
    return;
  }
  const int warps = (int)blockDim.x >> 5;
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    uint32_t seen = 0;
    const uint32_t* a = &lo[h].x;
    const uint32_t* b = &hi[h].x;
#pragma unroll
    for (int i = 0; i < 4; ++i) seen = amax_bits(amax_bits(seen, a[i]), b[i]);
    seen = __reduce_max_sync(0xffffffffu, seen);
    if ((tid & 31) == 0) s_amax[h][tid >> 5] = seen;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (kvh0 + h >= c.n_kv_heads || u.page < 0) break;
    const uint32_t seen = __reduce_max_sync(0xffffffffu, (tid & 31) < warps ? s_amax[h][tid & 31] : 0u);
    const float scale = scale_of<INT8>(bits_f(seen));
    const size_t sc = (size_t)u.page * c.n_kv_heads + kvh0 + h;
    uint8_t* dst = (IS_K ? c.k : c.v) + (sc * c.block + place) * D + j * 8;
    const uint4 x = lo[h], y = hi[h];
    const Divisor by = divisor(scale);
    *reinterpret_cast<uint2*>(dst) = make_uint2(codes4<INT8>(lo_f(x.x), hi_f(x.x), lo_f(x.y), hi_f(x.y), by), codes4<INT8>(lo_f(x.z), hi_f(x.z), lo_f(x.w), hi_f(x.w), by));
    *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(codes4<INT8>(lo_f(y.x), hi_f(y.x), lo_f(y.y), hi_f(y.y), by), codes4<INT8>(lo_f(y.z), hi_f(y.z), lo_f(y.w), hi_f(y.w), by));
    if (tid == 0) (IS_K ? c.k_scale : c.v_scale)[sc] = scale;
  }
  __syncthreads();  // s_amax is free again; what this unit read of the tail is read
}

template <int D, bool INT8, bool IS_K, int HEADS>
__device__ __forceinline__ void do_cache(const KvAppend8Params& p, int row0, int kvh0, uint32_t* s_starts, uint32_t (*s_amax)[32]) {
  constexpr int J = D / 16;
  const int tid = threadIdx.x, block = p.cache.block;
  // The usual unit starts with the CTA's first row and is as long: its values are asked for before that is known (three loads, one after the
  // other, would come first).
  uint4 lo[HEADS], hi[HEADS];
  {
    const size_t row = (size_t)row0 + tid / J;
    const __nv_bfloat16* src = p.qkv + row * p.qkv_stride + (size_t)(p.n_heads + (IS_K ? 0 : p.cache.n_kv_heads) + kvh0) * D + tid % J * 8;
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      lo[h] = hi[h] = make_uint4(0, 0, 0, 0);
      if (row < (size_t)p.rows && kvh0 + h < p.cache.n_kv_heads) {
        lo[h] = ptx::ld_nc_v4(src + h * D);
        hi[h] = ptx::ld_nc_v4(src + h * D + D / 2);
      }
    }
  }
  // which rows start a unit: a bit for each (block <= 128 rows; a row is looked at by one thread)
  if (tid < 4) s_starts[tid] = 0;
  __syncthreads();
  for (int i = tid; i < block; i += (int)blockDim.x) {
    const int row = row0 + i;
    if (row >= p.rows) continue;
    if (row_ok(p, row)) {
      if (row == 0 || p.requests[row - 1] != p.requests[row] || (p.positions[row] & (block - 1)) == 0) atomicOr(&s_starts[i >> 5], 1u << (i & 31));
    } else if (IS_K && p.zero_rest) {
      for (int h = 0; h < HEADS && kvh0 + h < p.cache.n_kv_heads; ++h)
        for (int d = 0; d < D; d += 8)
          *reinterpret_cast<uint4*>(p.rotated + (size_t)row * p.rotated_stride + (size_t)(p.n_heads + kvh0 + h) * D + d) = make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  for (int w = 0; w < (block + 31) / 32; ++w) {
    for (uint32_t left = s_starts[w]; left; left &= left - 1) {
      const int row = row0 + w * 32 + __ffs(left) - 1;
      const Unit u = unit_at(p, row);
      const int first = min(max(p.starts[u.request], 0), row);   // the request's first row
      const int place0 = p.positions[first] & (block - 1);
      const bool ends = u.place + u.n < block;                    // it does not fill its block: it goes to the tail
      if (ends && row != first && place0 != 0) continue;          // ... which the CTA of the first unit does
      do_unit<D, INT8, IS_K, HEADS>(p, u, kvh0, s_amax, row == row0 && u.n == block, lo, hi);
      if (row == first && place0 != 0 && !ends) {
        // its last row, or the last that has an angle
        const int last = min(end_of(p, u.request, row) - 1, row + (p.table_rows - 1 - p.positions[row]));
        const int tail_row = last - (p.positions[last] & (block - 1));  // where the last block starts
        if (last > row && tail_row >= row + u.n && row_ok(p, tail_row) && p.requests[tail_row] == u.request) {
          const Unit e = unit_at(p, tail_row);
          if (e.place == 0 && e.n < block) do_unit<D, INT8, IS_K, HEADS>(p, e, kvh0, s_amax, false, lo, hi);
        }
      }
    }
  }
}

template <int D, int HEADS>
__device__ __forceinline__ void do_q(const KvAppend8Params& p, int row0, int h0) {
  constexpr int J = D / 16;
  const int tid = threadIdx.x, i = tid / J, j = tid - i * J;
  const int row = row0 + i;
  if (row >= p.rows) return;
  const bool ok = row_ok(p, row);
  if (!ok && !p.zero_rest) return;
  const __nv_bfloat16* src = p.qkv + (size_t)row * p.qkv_stride + (size_t)h0 * D + j * 8;
  __nv_bfloat16* dst = p.rotated + (size_t)row * p.rotated_stride + (size_t)h0 * D + j * 8;
  uint4 lo[HEADS], hi[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    lo[h] = hi[h] = make_uint4(0, 0, 0, 0);
    if (ok && h0 + h < p.n_heads) {
      lo[h] = ptx::ld_nc_v4(src + h * D);
      hi[h] = ptx::ld_nc_v4(src + h * D + D / 2);
    }
  }
  float cs[8], sn[8];
  if (ok) {
    const size_t pos = p.positions[row];
    const float4* cr = reinterpret_cast<const float4*>(p.cos + pos * (D / 2) + j * 8);
    const float4* sr = reinterpret_cast<const float4*>(p.sin + pos * (D / 2) + j * 8);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
    sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w, sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h0 + h >= p.n_heads) break;
    uint32_t* a = &lo[h].x;
    uint32_t* b = &hi[h].x;
    if (ok)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x0, y0, x1, y1;
        rotate(lo_f(a[k]), lo_f(b[k]), cs[2 * k], sn[2 * k], x0, y0);
        rotate(hi_f(a[k]), hi_f(b[k]), cs[2 * k + 1], sn[2 * k + 1], x1, y1);
        a[k] = pack_bf16(x0, x1);
        b[k] = pack_bf16(y0, y1);
      }
    *reinterpret_cast<uint4*>(dst + h * D) = lo[h];
    *reinterpret_cast<uint4*>(dst + h * D + D / 2) = hi[h];
  }
}

// blockIdx.x: rows; blockIdx.y: groups of HEADS k heads, then of v heads, then of QHEADS q heads.
template <int D, bool INT8, int HEADS, int QHEADS, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) kv_append8_kernel(const KvAppend8Params p) {
  __shared__ uint32_t s_starts[4];
  __shared__ uint32_t s_amax[HEADS][32];
  // no early start for the kernel behind it: a GEMM fetches what it takes for weights before it waits, and this kernel's results may be that
  ptx::griddep_wait();
  const int row0 = (int)blockIdx.x * p.cache.block;
  const int kv_groups = (p.cache.n_kv_heads + HEADS - 1) / HEADS;
  const int y = blockIdx.y;
  if (y < kv_groups)
    do_cache<D, INT8, true, HEADS>(p, row0, y * HEADS, s_starts, s_amax);
  else if (y < 2 * kv_groups)
    do_cache<D, INT8, false, HEADS>(p, row0, (y - kv_groups) * HEADS, s_starts, s_amax);
  else
    do_q<D, QHEADS>(p, row0, (y - 2 * kv_groups) * QHEADS);
}

template <int D, bool INT8, int HEADS, int QHEADS, int THREADS, int CTAS>
cudaError_t launch(const KvAppend8Params& p, cudaStream_t stream) {
  const int kv_groups = (p.cache.n_kv_heads + HEADS - 1) / HEADS, q_groups = (p.n_heads + QHEADS - 1) / QHEADS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.rows + p.cache.block - 1) / p.cache.block), 2 * kv_groups + q_groups);
  cfg.blockDim = dim3(p.cache.block * (D / 16));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv_append8_kernel<D, INT8, HEADS, QHEADS, THREADS, CTAS>, p);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}
template <int D, bool INT8>
cudaError_t by_size(const KvAppend8Params& p, cudaStream_t s) {
  // Two heads of the cache and four of q a CTA, at 64 registers (us at 16 x 1024 rows of 32 + 32 + 32 heads in blocks of 32: two and two
  // heads 170, four and four 181, one and one 200; of 16: 162, of 64: 178, of 128: 202; int8 175, 180, 191 and 217).
  const int threads = p.cache.block * (D / 16);
  if (threads <= 256) return launch<D, INT8, 2, 4, 256, 4>(p, s);
  if (threads <= 512) return launch<D, INT8, 2, 4, 512, 2>(p, s);
  return launch<D, INT8, 2, 4, 1024, 1>(p, s);
}

}  // namespace

cudaError_t kv_append8(const KvAppend8Params& p, cudaStream_t stream) {
  auto aligned = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  const KvCache8& c = p.cache;
  if (p.rows == 0) return cudaSuccess;
  if (p.rows < 0 || p.n_requests < 0 || p.n_requests > c.requests || p.n_heads < 0 || c.n_kv_heads < 1 || p.table_rows < 0) return cudaErrorInvalidValue;
  if (c.block < 16 || c.block > 128 || (c.block & (c.block - 1)) != 0) return cudaErrorInvalidValue;
  if (2ll * c.n_kv_heads + p.n_heads > 65535) return cudaErrorInvalidValue;
  if (!aligned(p.qkv) || !aligned(p.rotated) || !aligned(c.k) || !aligned(c.v) || !aligned(c.k_tail) || !aligned(c.v_tail) || !aligned(p.cos) || !aligned(p.sin)) return cudaErrorInvalidValue;
  if (p.qkv_stride % 8 != 0 || p.rotated_stride % 8 != 0) return cudaErrorInvalidValue;
  if (c.head_dim == 128) return c.int8 ? by_size<128, true>(p, stream) : by_size<128, false>(p, stream);
  if (c.head_dim == 64) return c.int8 ? by_size<64, true>(p, stream) : by_size<64, false>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace ccl
