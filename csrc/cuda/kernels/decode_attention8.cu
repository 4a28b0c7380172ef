// Single-token attention over the 8-bit paged cache, fused with rotary embedding, append and the quantisation of a block that fills up.
//
// Bound by memory: 2 * head_dim bytes per cached position and KV head. Measured, of a copy's 6.55 TB/s: 7 sequences of 65521 positions, 64
// heads on 8, 941 MB: 154 to 168 us, 5.6 to 6.1 TB/s; 16 of 1087, 32 heads, 147 MB: 34.4 us, 4.3 TB/s, of which 2 us pass before the first
// page is asked for and the launch and the join take as long again; 33 of 0 to 2999, 32 heads on 8, 107 MB: 33 us, by the longest
// sequence, whose 16 rounds of a warp take 1.4 us each; one of 1000: 8 us, six dependent round trips.
// All query heads of a KV head (a tile of eight) go through one CTA, so that a code is read and widened once for them. Per 16 positions a
// warp multiplies transposed: scores^T = K q^T and then out^T = V^T p^T, with the eight query heads as the N side of m16n8k16. K's rows and
// V's columns are then the A operand, whose fragments ask of a thread four codes of a row (K) or of a column (V); since the sum over k does
// not care for its order, a thread takes 16 neighbouring bytes of a row and uses them as its k indices of four products (the queries are
// read in the same order), so that a thread reads 16 bytes at a time what it alone needs, with no barrier in the loop. (tcgen05 wants its
// operands in shared memory, widened: a round trip for every byte and 128 rows for at most 16; the products keep the tensor pipe busy for
// 14 % of the time that the bytes take to arrive.)
//
// Exactness. Codes widen to f16 without rounding. q is multiplied by a power of two and split into two f16 parts (22 bits), so scores are
// as exact as in fp32. The page's V scale joins the score, as log2(scale): weights 2^(s + log2 vs - m) multiply the codes in f16, kept
// within a factor of 2^15 of the running reference (f16 is what the codes are products with: 2^-11 of each weight, where the result is rounded to bf16,
// 2^-8; a second part would double V's products), and the sum of the softmax takes them divided by vs, in fp32. The reference m moves
// only when a score passes it by 2^15, and starts 2^8 below the maximum. The tail (bf16, at most a block) goes through the same products in
// bf16, q (the sum of its f16 parts) in three parts and the weights in two.
//
// A warp takes two units of 16 positions at a time, so that a fragment of q is read once for both, and has the next two pairs on their way:
// every thread copies (cp.async) what it will read itself, which needs no barrier. 16 KB of ring a warp let twelve warps share an SM.
#include "kv_cache8.cuh"

#include "gemm.h"

#include <algorithm>

namespace ccl {
namespace {

using namespace kv8;

// CTAs of 3, 4 or 6 warps (W): the GPU holds 592, 444 or 296 of them, twelve warps an SM. With sixteen query rows (NT 2) a warp's state takes
// twice the registers: CTAs of four, two an SM.
constexpr int ctas_per_sm(int NT, int W) { return NT == 1 ? 12 / W : 2; }
constexpr int kStages = 2;         // pairs of units on their way to a warp, or in use
constexpr int kMaxSplits = 64, kMaxCluster = 16;
constexpr int least_units(int W) { return 2 * W; }  // units of 16 positions per split at least: a pair for each warp
constexpr int kChunk = 512;        // units of a split where there are CTAs enough without splits
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 8.f;       // the reference starts this far (log2) below the maximum
constexpr float kRoom = 15.f;      // and moves when a weight would pass 2^15 (f16 ends at 2^16)

// Work split of one sequence and head tile: `per` units of 16 paged positions for each of `used` splits; the last one takes the tail too.
struct Split {
  int units, per, used;
};
__device__ __forceinline__ Split split_of(int pos, const DecodeAttn8Params& p) {
  Split s;
  s.units = (pos / p.cache.block) * (p.cache.block / 16);
  s.per = max(p.least, (s.units + p.nsplit - 1) / p.nsplit);
  s.used = max(1, (s.units + s.per - 1) / s.per);  // at most nsplit
  return s;
}
__device__ __forceinline__ bool position_ok(const DecodeAttn8Params& p, int pos) {
  return pos >= 0 && pos < p.table_rows && pos / p.cache.block < p.max_blocks;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float2 ld_cluster(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float f16_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
__device__ __forceinline__ float f16_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 or 8 bytes to shared memory, or zeros (`bytes` 0).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Four e4m3 codes -> two f16 pairs, exactly. The conversion instruction runs on a unit that starts 16 lanes a clock on a multiprocessor; for
// all of K and V it would bound the loop, so half of K goes the other way:
__device__ __forceinline__ void widen_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// ... 2^-8 of their values, on the integer units: a code's seven lower bits, moved to bit 7, are the f16 whose exponent is read with a bias
// that is 8 larger, denormals too. (The NaN code would be 480: a block with a NaN has a NaN scale, which spoils every score of its page.)
constexpr float kLowE4m3 = 256.f;
__device__ __forceinline__ void widen_e4m3_low(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t x = __byte_perm(w, 0, 0x1100), y = __byte_perm(w, 0, 0x3322);
  lo = ((x >> 1) & 0x3f803f80u) | (x & 0x80008000u);
  hi = ((y >> 1) & 0x3f803f80u) | (y & 0x80008000u);
}
// Four int8 codes -> (code + 128) * 2^-24 as denormal f16: K's products then have 128 * sum(q) too much, which is taken off the scores.
constexpr float kLowInt8 = 16777216.f;
__device__ __forceinline__ void widen_int8_low(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  lo = __byte_perm(w, 0, 0x4140);
  hi = __byte_perm(w, 0, 0x4342);
}
// Four int8 codes plus 128 -> the codes: 1024 + u as f16, minus 1152. (V's weights are not known beforehand, and its sums cancel: no bias.)
__device__ __forceinline__ void widen_biased(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));
  uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

template <int D, int NT, int W>
struct Smem {
  static constexpr int R = 8 * NT;       // query rows
  static constexpr int QP = D + 4;       // pitch (halves): eight rows start two banks apart
  static constexpr int OS = D / 8 + 2;   // the dims of a lane (floats), moved two banks on for each g
  static constexpr int OP = 8 * OS + 2;  // pitch (floats)
  static constexpr int kUnit = 16 * D;   // bytes of K, or of V, of a unit of 16 positions
  union {
    uint8_t ring[W][kStages][2][2 * kUnit];  // K and V of two units
    struct {                             // at the end
      float o[W][R * OP];           // out of each warp
      float2 joined[R * (D / 2 + 1)];    // of the CTA, for the others of its cluster: out, and {m, l} behind each row
    };
  };
  union {
    struct {
      __half qh[R * QP], ql[R * QP];     // q as two f16 parts
    };
    struct {
      float m[W][R], l[W][R];  // at the end
    };
  };
  float qs[R];                           // scale * log2 e over the power of two of the row
  float qc[R];                           // int8: what the codes' bias adds to a score
  uint4 new_k[D / 8], new_v[D / 8];      // the new token, bf16
  uint32_t amax[2][W];
  int bad;
};

// The new token of one sequence and KV head: k rotated, both as bf16 in shared memory. Two words (four values) a thread, of D / 2 threads;
// `load` needs no position.
struct NewToken {
  uint32_t a, b;
};
template <int D>
__device__ __forceinline__ NewToken load_new(const DecodeAttn8Params& p, int b, int kvh) {
  const int tid = threadIdx.x, i = tid & (D / 4 - 1);
  if (tid >= D / 2) return {0, 0};
  const int head = p.n_heads + kvh + (tid < D / 4 ? 0 : p.cache.n_kv_heads);  // the first D / 4 threads have k, the others v
  const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qkv + (size_t)b * p.qkv_stride + (size_t)head * D) + i;
  return {src[0], src[D / 4]};
}
template <int D>
__device__ __forceinline__ void store_new(NewToken w, float2 c, float2 s, uint4* k, uint4* v) {  // c, s: of dims 2i and 2i + 1
  const int tid = threadIdx.x, i = tid & (D / 4 - 1);
  if (tid >= D / 2) return;
  if (tid < D / 4) {  // dims 2i and 2i + 1 and the ones half a head further on
    float x0, y0, x1, y1;
    rotate(lo_f(w.a), lo_f(w.b), c.x, s.x, x0, y0);
    rotate(hi_f(w.a), hi_f(w.b), c.y, s.y, x1, y1);
    w.a = pack_bf16(x0, x1);
    w.b = pack_bf16(y0, y1);
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(tid < D / 4 ? k : v) + i;
  dst[0] = w.a;
  dst[D / 4] = w.b;
}

// Quantises the block that the new token completes. A CTA of its own does that, beside the attention (which reads this block from the
// tail): within the CTA that attends it took as long as 300 positions.
template <int D, bool INT8, int W>
__device__ __forceinline__ void quantise_block(const DecodeAttn8Params& p, int b, int kvh, uint4* fresh_k, uint4* fresh_v, uint32_t (*amax)[W]) {
  constexpr int kThreads = W * 32;
  const KvCache8& c = p.cache;
  const int tid = threadIdx.x, pos = p.positions[b];
  if (!position_ok(p, pos) || (pos & (c.block - 1)) != c.block - 1) return;
  const int page = p.table[(size_t)b * p.max_blocks + pos / c.block];
  if ((unsigned)page >= (unsigned)c.num_blocks) return;
  const int i2 = tid & (D / 4 - 1);
  store_new<D>(load_new<D>(p, b, kvh), reinterpret_cast<const float2*>(p.cos + (size_t)pos * (D / 2))[i2], reinterpret_cast<const float2*>(p.sin + (size_t)pos * (D / 2))[i2], fresh_k, fresh_v);
  __syncthreads();
  const size_t at = ((size_t)b * c.n_kv_heads + kvh) * c.block * D, sc = (size_t)page * c.n_kv_heads + kvh;
  const uint4* k = reinterpret_cast<const uint4*>(c.k_tail + at);
  const uint4* v = reinterpret_cast<const uint4*>(c.v_tail + at);
  const int last = (c.block - 1) * (D / 8), n = last + D / 8;  // pieces of eight values; from `last` on: the new token
  constexpr int U = 8;                                          // of K, and of V, in flight
  uint4 x[U], y[U];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      x[u] = y[u] = make_uint4(0, 0, 0, 0);
      if (i < n) {
        x[u] = *(i >= last ? fresh_k + (i - last) : k + i);
        y[u] = *(i >= last ? fresh_v + (i - last) : v + i);
      }
    }
  };
  auto most = [](uint32_t seen, const uint4& w) { return amax_bits(amax_bits(amax_bits(amax_bits(seen, w.x), w.y), w.z), w.w); };
  uint32_t seen_k = 0, seen_v = 0;
  for (int i0 = tid; i0 < n; i0 += U * kThreads) {
    fetch(i0);
#pragma unroll
    for (int u = 0; u < U; ++u) seen_k = most(seen_k, x[u]), seen_v = most(seen_v, y[u]);
  }
  seen_k = __reduce_max_sync(0xffffffffu, seen_k);
  seen_v = __reduce_max_sync(0xffffffffu, seen_v);
  if ((tid & 31) == 0) amax[0][tid >> 5] = seen_k, amax[1][tid >> 5] = seen_v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) seen_k = max(seen_k, amax[0][w]), seen_v = max(seen_v, amax[1][w]);
  const float scale_k = scale_of<INT8>(bits_f(seen_k)), scale_v = scale_of<INT8>(bits_f(seen_v));
  uint2* to_k = reinterpret_cast<uint2*>(c.k + sc * c.block * D);
  uint2* to_v = reinterpret_cast<uint2*>(c.v + sc * c.block * D);
  const Divisor by_k = divisor(scale_k), by_v = divisor(scale_v);
  auto codes8 = [](const uint4& w, const Divisor& scale) {
    return make_uint2(codes4<INT8>(lo_f(w.x), hi_f(w.x), lo_f(w.y), hi_f(w.y), scale), codes4<INT8>(lo_f(w.z), hi_f(w.z), lo_f(w.w), hi_f(w.w), scale));
  };
  for (int i0 = tid; i0 < n; i0 += U * kThreads) {
    if (n > U * kThreads) fetch(i0);  // (a block of one round is still there)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      if (i < n) {
        to_k[i] = codes8(x[u], by_k);
        to_v[i] = codes8(y[u], by_v);
      }
    }
  }
  if (tid == 0) {
    c.k_scale[sc] = scale_k;
    c.v_scale[sc] = scale_v;
  }
}

template <int D, int NT, bool INT8, int W>
__global__ void __launch_bounds__(W * 32, ctas_per_sm(NT, W)) decode_attention8_kernel(const DecodeAttn8Params p) {
  constexpr int R = 8 * NT, kThreads = W * 32;
  constexpr int KJ = D / 64;        // 16-byte loads of a K row by a thread
  constexpr int VW = D / 32;        // words of a V row by a thread
  constexpr int NM = D / 16;        // products over the dims
  using S = Smem<D, NT, W>;
  extern __shared__ __align__(16) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);

  ptx::griddep_wait();
  const KvCache8& c = p.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / c.n_kv_heads;
  const int tiles = (group + R - 1) / R;
  // the grid: nsplit CTAs for every pair of a head tile and a sequence; then, the last to start, one for each sequence and KV head whose
  // block may fill up
  const int pairs = p.batch * c.n_kv_heads * tiles;
  const int pair = blockIdx.x / p.nsplit, split = blockIdx.x - pair * p.nsplit;
  if (pair >= pairs) {
    const int i = (pair - pairs) * p.nsplit + split;
    if (i < p.batch * c.n_kv_heads) quantise_block<D, INT8, W>(p, i % p.batch, i / p.batch, sm.new_k, sm.new_v, sm.amax);
    return;
  }
  const int b = pair % p.batch, kvh = pair / p.batch / tiles, tile = pair / p.batch - kvh * tiles;
  const int rows = min(R, group - tile * R);
  const int head0 = kvh * group + tile * R;
  const int pos = p.positions[b];
  // what needs no position is asked for with it: q (LPR lanes share a row; a lane has two words of it, half a head apart), the new token
  constexpr int LPR = D / 4, RPW = 32 / LPR, QI = (R + W * RPW - 1) / (W * RPW);
  const int q_word = lane % LPR;
  uint32_t q_lo[QI], q_hi[QI];
  auto q_row = [&](int i) { return (i * W + warp) * RPW + lane / LPR; };
#pragma unroll
  for (int i = 0; i < QI; ++i) {
    q_lo[i] = q_hi[i] = 0;
    if (q_row(i) < rows) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.qkv + (size_t)b * p.qkv_stride + (size_t)(head0 + q_row(i)) * D) + q_word;
      q_lo[i] = src[0];
      q_hi[i] = src[D / 4];
    }
  }
  const NewToken fresh = load_new<D>(p, b, kvh);
  // The loop's units, in pairs: pair n of this warp is pair warp + W n of the split; a lane looks up the page of one unit of a window of 16 pairs.
  auto unit_of = [&](int n, int h) { return 2 * (warp + W * n) + h; };
  const int in_block = 31 - __clz(c.block / 16);  // log2 of the units of a block
  const int* table = p.table + (size_t)b * p.max_blocks;
  __nv_bfloat16* out = p.out + (size_t)b * p.out_stride + (size_t)head0 * D;
  if (!position_ok(p, pos)) {
    if (split == 0)
      for (int i = tid; i < rows * D; i += kThreads) out[i] = __float2bfloat16(0.f);
    return;
  }
  const Split sp = split_of(pos, p);
  if (split >= sp.used) return;
  const bool owns_tail = split == sp.used - 1;
  // The angles of this lane's dims, for its rows of q and, in the first warp, for k. Behind the loop's loads they would wait for all of those
  // of the GPU (5 us instead of 1).
  const float2 cs = reinterpret_cast<const float2*>(p.cos + (size_t)pos * (D / 2))[q_word], sn = reinterpret_cast<const float2*>(p.sin + (size_t)pos * (D / 2))[q_word];

  // ---- the loop's loads -------------------------------------------------------------------------------------------------------------
  const int u0 = split * sp.per, units = max(0, min(sp.units - u0, sp.per));
  const int n_pairs = max(0, ((units + 1) / 2 - warp + W - 1) / W);
  const int place = pos & (c.block - 1);
  // the tail's units of 16 positions follow the pairs, the first of them with the last warp
  const int tail_units = owns_tail ? place / 16 + 1 : 0;
  const int n_all = n_pairs + max(0, (tail_units - (W - 1 - warp) + W - 1) / W);
  auto tail_first = [&](int n) { return ((W - 1 - warp) + W * (n - n_pairs)) * 16; };
  const size_t tail_at = ((size_t)b * c.n_kv_heads + kvh) * c.block * D;
  bool bad = false;
  auto page_of = [&](int n) {  // of window n / 16, for this lane
    const int u = unit_of(n + (lane >> 1), lane & 1);
    if (u >= units) return 0;
    const int page = table[(u0 + u) >> in_block];
    if ((unsigned)page < (unsigned)c.num_blocks) return page;
    bad = true;
    return 0;
  };
  int pages = page_of(0), pages_next = page_of(16);
  float ks_next = 1.f, vs_next = 1.f;
  auto scales_of = [&](int n) {
    if (unit_of(n + (lane >> 1), lane & 1) >= units) return;
    const size_t at = (size_t)pages * c.n_kv_heads + kvh;
    ks_next = c.k_scale[at];
    vs_next = c.v_scale[at];
  };
  // A thread copies what it will read itself: K's rows g and g + 8, V's rows 2t, 2t + 1, 2t + 8, 2t + 9.
  const uint32_t page_bytes = (uint32_t)c.n_kv_heads * c.block * D;  // at most 2^30
  const uint8_t* k_base = c.k + (size_t)kvh * c.block * D + g * D + t * 16;
  const uint8_t* v_base = c.v + (size_t)kvh * c.block * D + 2 * t * D + g * (D / 8);
  const uint32_t ring = ptx::smem_u32(sm.ring[warp]);
  // A row of V that a load brings in stays together in shared memory (scattered by thread, its 16 bytes would be written one after the
  // other: 5.2 instead of 7.0 TB/s); its pieces change places with the row, so that they are read without conflicts.
  const uint32_t v_place = t * D + (D == 128 ? (g ^ (2 * t)) * 16 : (g ^ (2 * (t & 2))) * 8);
  size_t at[kStages][2];
  auto load_k = [&](int n, size_t (&where)[2]) {
    if (n < n_pairs) {
      if (n > 0 && (n & 15) == 0) {
        pages = pages_next;
        scales_of(n);
        pages_next = page_of(n + 16);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int u = unit_of(n, h);
        const uint32_t page = __shfl_sync(0xffffffffu, pages, 2 * (n & 15) + h);
        where[h] = (size_t)page * page_bytes + (uint32_t)(((u0 + u) & ((1 << in_block) - 1)) * 16 * D);
        const uint8_t* k = k_base + where[h];
        const uint32_t dst = ring + ((n % kStages) * 2 * 2 + h) * S::kUnit + lane * 16, bytes = u < units ? 16 : 0;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          copy16(dst + j * 1024, k + j * 64, bytes);
          copy16(dst + j * 1024 + 512, k + 8 * D + j * 64, bytes);
        }
      }
    } else if (n < n_all) {  // bf16: one unit is as long as two of codes; the new position is not in the tail yet
      const int r = tail_first(n) + g;
      const __nv_bfloat16* k = c.k_tail + tail_at + (size_t)g * D + (size_t)tail_first(n) * D + t * 8;
      const uint32_t dst = ring + (n % kStages) * 4 * S::kUnit + lane * 16, b0 = r < place ? 16 : 0, b8 = r + 8 < place ? 16 : 0;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        copy16(dst + j * 1024, r < place ? k + j * 32 : c.k_tail, b0);
        copy16(dst + j * 1024 + 512, r + 8 < place ? k + 8 * D + j * 32 : c.k_tail, b8);
      }
    }
    copies_done();
  };
  auto load_v = [&](int n, const size_t (&where)[2]) {
    if (n < n_pairs) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* v = v_base + where[h];
        const uint32_t dst = ring + ((n % kStages) * 2 * 2 + 2 + h) * S::kUnit + v_place, bytes = unit_of(n, h) < units ? D / 8 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* row = v + ((i & 1) + (i >> 1) * 8) * D;
          if constexpr (D == 128)
            copy16(dst + i * 512, row, bytes);
          else
            copy8(dst + i * 256, row, bytes);
        }
      }
    } else if (n < n_all) {
      const uint32_t dst = ring + ((n % kStages) * 4 + 2) * S::kUnit + lane * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = tail_first(n) + 2 * t + (i & 1) + (i >> 1) * 8;
        const __nv_bfloat16* v = r < place ? c.v_tail + tail_at + (size_t)r * D + g * (D / 8) : c.v_tail;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) copy16(dst + (i * (D / 64) + j) * 512, v + j * 8, r < place ? 16 : 0);
      }
    }
    copies_done();
  };
  scales_of(0);
#pragma unroll
  for (int n = 0; n < kStages; ++n) {
    load_k(n, at[n]);
    load_v(n, at[n]);
  }

  // ---- q: rotate, split; the new token ------------------------------------------------------------------------------------------
#pragma unroll
  for (int i = 0; i < QI; ++i) {
    const int r = q_row(i);
    float z[2][2];  // [half][dim]
    rotate(lo_f(q_lo[i]), lo_f(q_hi[i]), cs.x, sn.x, z[0][0], z[1][0]);
    rotate(hi_f(q_lo[i]), hi_f(q_hi[i]), cs.y, sn.y, z[0][1], z[1][1]);
    float most = fmaxf(fmaxf(fabsf(z[0][0]), fabsf(z[0][1])), fmaxf(fabsf(z[1][0]), fabsf(z[1][1])));
#pragma unroll
    for (int x = LPR / 2; x; x >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
    const int e = (int)(__float_as_uint(most) >> 23);  // biased exponent; 0 for a row of zeros, 255 for an infinity
    // the largest element at 2^9 .. 2^10, after the factor that half of an e4m3 K's dims get (2^8, and finite with it)
    const int up = e == 0 || e == 255 ? 127 : min(INT8 ? 254 : 246, 127 + (INT8 ? 9 : 1) + 127 - e);
    const float mult = __uint_as_float((uint32_t)up << 23), to_f16 = !INT8 && (q_word & 2) ? mult * kLowE4m3 : mult;
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = r * S::QP + h * (D / 2) + 2 * q_word;
      const bool row = R % (W * RPW) == 0 || r < R;
      const __half2 hi = __floats2half2_rn(z[h][0] * to_f16, z[h][1] * to_f16);
      const __half2 lo = __floats2half2_rn(z[h][0] * to_f16 - __low2float(hi), z[h][1] * to_f16 - __high2float(hi));
      if (row) {
        *reinterpret_cast<__half2*>(&sm.qh[at]) = hi;
        *reinterpret_cast<__half2*>(&sm.ql[at]) = lo;
      }
      sum += (__low2float(hi) + __low2float(lo)) + (__high2float(hi) + __high2float(lo));
    }
    if constexpr (INT8) {
#pragma unroll
      for (int x = LPR / 2; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    }
    if (q_word == 0 && r < R) {
      sm.qs[r] = p.scale * kLog2e / mult;
      sm.qc[r] = 128.f * sum * (p.scale * kLog2e / mult);
    }
  }
  if (owns_tail) store_new<D>(fresh, cs, sn, sm.new_k, sm.new_v);  // (q_word is the word that a thread of k has)
  if (tid == 0) sm.bad = 0;
  __syncthreads();

  // ---- state of the softmax: column 2t and 2t + 1 of each tile of eight queries ---------------------------------------------------
  float o[NT][NM][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int a = 0; a < NT; ++a) {
#pragma unroll
    for (int i = 0; i < NM; ++i) o[a][i][0] = o[a][i][1] = o[a][i][2] = o[a][i][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[a][h] = -INFINITY;
      l[a][h] = 0.f;
    }
  }

  // Scores (rows: positions g, g + 8 of each unit; columns: queries) into weights. Moves the references where a score passes them by kRoom.
  auto weigh = [&](auto& s, const float* over_v) {
    constexpr int H = sizeof(s[0]) / sizeof(s[0][0]);
    bool over = false;
    float top[NT][2];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[a][e] = fmaxf(s[a][0][e], s[a][0][e + 2]);
#pragma unroll
        for (int h = 1; h < H; ++h) top[a][e] = fmaxf(top[a][e], fmaxf(s[a][h][e], s[a][h][e + 2]));
        over = over || top[a][e] - m[a][e] > kRoom;
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t0 = top[a][e];
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 4));
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 8));
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 16));
          if (t0 - m[a][e] > kRoom) {
            const float corr = exp2_fast(m[a][e] - (t0 - kHead));
            m[a][e] = t0 - kHead;
            l[a][e] *= corr;
#pragma unroll
            for (int i = 0; i < NM; ++i) {
              o[a][i][e] *= corr;
              o[a][i][e + 2] *= corr;
            }
          }
        }
    }
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][h][e] = exp2_fast(s[a][h][e] - m[a][e & 1]);
        l[a][0] += (s[a][h][0] + s[a][h][2]) * over_v[h];
        l[a][1] += (s[a][h][1] + s[a][h][3]) * over_v[h];
      }
  };

  // ---- the pages -----------------------------------------------------------------------------------------------------------------
  float f[NT][2], off[NT][2];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      f[a][e] = sm.qs[a * 8 + 2 * t + e] * (INT8 ? kLowInt8 : 1.f);
      off[a][e] = INT8 ? sm.qc[a * 8 + 2 * t + e] : 0.f;
    }
  // K of pair n -> its products with q (two sums, which join later).
  auto scores = [&](int n, float (&s)[2][NT][2][4]) {
    const uint8_t* stage = &sm.ring[warp][0][0][0] + (n % kStages) * 4 * S::kUnit;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][a][0][e] = s[0][a][1][e] = s[1][a][0][e] = s[1][a][1][e] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      uint4 x[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4* kr = reinterpret_cast<const uint4*>(stage + h * S::kUnit) + lane;
        x[h][0] = kr[j * 64];
        x[h][1] = kr[j * 64 + 32];
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0[2], a1[2], a2[2], a3[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t r0 = w == 0 ? x[h][0].x : (w == 1 ? x[h][0].y : (w == 2 ? x[h][0].z : x[h][0].w));
          const uint32_t r8 = w == 0 ? x[h][1].x : (w == 1 ? x[h][1].y : (w == 2 ? x[h][1].z : x[h][1].w));
          if constexpr (INT8) {
            widen_int8_low(r0, a0[h], a2[h]);
            widen_int8_low(r8, a1[h], a3[h]);
          } else if (w & 1) {
            widen_e4m3_low(r0, a0[h], a2[h]);
            widen_e4m3_low(r8, a1[h], a3[h]);
          } else {
            widen_e4m3(r0, a0[h], a2[h]);
            widen_e4m3(r8, a1[h], a3[h]);
          }
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          const int q = (a * 8 + g) * S::QP + j * 64 + t * 16 + w * 4;
          const uint2 hi = *reinterpret_cast<const uint2*>(&sm.qh[q]), lo = *reinterpret_cast<const uint2*>(&sm.ql[q]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma(s[0][a][h], a0[h], a1[h], a2[h], a3[h], hi.x, hi.y);
            mma(s[1][a][h], a0[h], a1[h], a2[h], a3[h], lo.x, lo.y);
          }
        }
      }
    }
  };
  // The scores of the pair after the next are not asked for before K of the next one is read, and so on: while the weights and values of
  // pair n go their way (exponentials, transposes, products one after the other), the products of pair n + 1 have nothing to wait for.
  // In the order of asking: .. K(n + 1) V(n) | K(n + 2) V(n + 1): two more than are waited for.
  float ks = 1.f, lvs = 0.f, ivs = 1.f;  // of the window's lane
  float acc[2][NT][2][4];
  size_t where[2] = {0, 0};  // of pair n + 2, whose V is still to be asked for
  wait_copies<2 * kStages - 1>();
  if (n_pairs > 0) {
    scores(0, acc);
    load_k(kStages, where);
  } else {
    copies_done();
  }
  int n = 0;
  for (; n < n_pairs; ++n) {
    if ((n & 15) == 0) {
      // (an infinite scale, that of a page with an infinity, stands for 0 * inf in every position: NaN)
      ks = ks_next + (ks_next - ks_next);
      lvs = log2f(vs_next + (vs_next - vs_next));
      ivs = __frcp_rn(vs_next);
    }
    float s[NT][2][4], uiv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int src = 2 * (n & 15) + h;
      const float uks = __shfl_sync(0xffffffffu, ks, src), ulv = __shfl_sync(0xffffffffu, lvs, src);
      uiv[h] = __shfl_sync(0xffffffffu, ivs, src);
      const bool there = unit_of(n, h) < units;
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float rest = INT8 ? ulv - off[a][e & 1] * uks : ulv;
          const float x = (acc[0][a][h][e] + acc[1][a][h][e]) * (f[a][e & 1] * uks) + rest;
          s[a][h][e] = x + (x - x);  // (what passes fp32 is NaN: -inf would be that or nothing, by what else the warp has)
          if (h == 1 && !there) s[a][h][e] = -INFINITY;
        }
    }
    wait_copies<2>();
    size_t next[2] = {0, 0};
    if (n + 1 < n_pairs) {
      scores(n + 1, acc);
      load_k(n + 1 + kStages, next);  // where K(n + 1) was
    } else {
      copies_done();
    }
    weigh(s, uiv);
    uint32_t b0[NT][2], b1[NT][2];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        b0[a][h] = transpose8x8(pack_f16(s[a][h][0], s[a][h][1]));
        b1[a][h] = transpose8x8(pack_f16(s[a][h][2], s[a][h][3]));
      }
    const uint8_t* stage = &sm.ring[warp][0][0][0] + (n % kStages) * 4 * S::kUnit;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t vr[4][VW];
      const uint8_t* vp = stage + (2 + h) * S::kUnit + v_place;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(vp + i * 512);
          vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(vp + i * 256);
          vr[i][0] = x.x, vr[i][1] = x.y;
        }
        if constexpr (INT8) {
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[i][w] ^= 0x80808080u;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t a0, a1, a2, a3;
          const uint32_t y = __byte_perm(vr[0][w], vr[1][w], x ? 0x7362 : 0x5140), z = __byte_perm(vr[2][w], vr[3][w], x ? 0x7362 : 0x5140);
          if constexpr (INT8) {
            widen_biased(y, a0, a1);
            widen_biased(z, a2, a3);
          } else {
            widen_e4m3(y, a0, a1);
            widen_e4m3(z, a2, a3);
          }
#pragma unroll
          for (int a = 0; a < NT; ++a) mma(o[a][2 * w + x], a0, a1, a2, a3, b0[a][h], b1[a][h]);
        }
      }
    }
    load_v(n + kStages, where);
    where[0] = next[0];
    where[1] = next[1];
  }

  // ---- the tail, q in three bf16 parts and the weights in two ------------------------------------------------------------------------
  for (; n < n_all; ++n) {
    const int first = tail_first(n);
    const uint4* stage = reinterpret_cast<const uint4*>(&sm.ring[warp][0][0][0] + (n % kStages) * 4 * S::kUnit) + lane;
    float s[NT][1][4];
#pragma unroll
    for (int a = 0; a < NT; ++a) s[a][0][0] = s[a][0][1] = s[a][0][2] = s[a][0][3] = 0.f;
    wait_copies<2>();
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint4 x0 = *(first + g == place ? sm.new_k + j * 4 + t : stage + j * 64);
      const uint4 x8 = *(first + g + 8 == place ? sm.new_k + j * 4 + t : stage + j * 64 + 32);
      const uint32_t r0[4] = {x0.x, x0.y, x0.z, x0.w}, r8[4] = {x8.x, x8.y, x8.z, x8.w};
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          const int at = (a * 8 + g) * S::QP + j * 32 + t * 8 + w * 4;
          const uint2 hi = *reinterpret_cast<const uint2*>(&sm.qh[at]), lo = *reinterpret_cast<const uint2*>(&sm.ql[at]);
          float z[4] = {f16_lo(hi.x) + f16_lo(lo.x), f16_hi(hi.x) + f16_hi(lo.x), f16_lo(hi.y) + f16_lo(lo.y), f16_hi(hi.y) + f16_hi(lo.y)};
          uint32_t part[3][2];
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // (the dims that e4m3's K has 2^-8 of)
              if (i == 0 && !INT8 && w == 1) z[2 * e] *= 1.f / kLowE4m3, z[2 * e + 1] *= 1.f / kLowE4m3;
              part[i][e] = pack_bf16(z[2 * e], z[2 * e + 1]);
              z[2 * e] -= lo_f(part[i][e]);
              z[2 * e + 1] -= hi_f(part[i][e]);
            }
#pragma unroll
          for (int i = 2; i >= 0; --i) mma_bf16(s[a][0], r0[2 * w], r8[2 * w], r0[2 * w + 1], r8[2 * w + 1], part[i][0], part[i][1]);  // the small parts first
        }
    }
    load_k(n + kStages, where);
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (what passes fp32 is NaN: the sign of its infinity may be that of a small part)
        const float x = s[a][0][e] * (f[a][e & 1] * (INT8 ? 1.f / kLowInt8 : 1.f)) + (s[a][0][e] - s[a][0][e]);
        s[a][0][e] = first + g + (e >> 1) * 8 <= place ? x : -INFINITY;
      }
    const float one[1] = {1.f};
    weigh(s, one);
    // two bf16 parts of the weights, the upper half of their bits and the rest, which is never zero: an infinity stays one
    uint32_t b0[2][NT], b1[2][NT];
    auto rest = [](float w) { return fmaxf(w - __uint_as_float(__float_as_uint(w) & 0xffff0000u), 7.5231638e-37f); };
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const float* w = s[a][0];
      b0[0][a] = transpose8x8(__byte_perm(__float_as_uint(w[0]), __float_as_uint(w[1]), 0x7632));
      b1[0][a] = transpose8x8(__byte_perm(__float_as_uint(w[2]), __float_as_uint(w[3]), 0x7632));
      b0[1][a] = transpose8x8(pack_bf16(rest(w[0]), rest(w[1])));
      b1[1][a] = transpose8x8(pack_bf16(rest(w[2]), rest(w[3])));
    }
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      uint4 v[4];  // zeros behind the new position
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = *(first + 2 * t + (i & 1) + (i >> 1) * 8 == place ? sm.new_v + g * (D / 64) + j : stage + 2 * S::kUnit / 16 + (i * (D / 64) + j) * 32);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        auto word = [&](int i) { return w == 0 ? v[i].x : (w == 1 ? v[i].y : (w == 2 ? v[i].z : v[i].w)); };
        const uint32_t a0 = __byte_perm(word(0), word(1), 0x5410), a1 = __byte_perm(word(0), word(1), 0x7632);
        const uint32_t a2 = __byte_perm(word(2), word(3), 0x5410), a3 = __byte_perm(word(2), word(3), 0x7632);
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          mma_bf16(o[a][j * 4 + w], a0, a1, a2, a3, b0[1][a], b1[1][a]);
          mma_bf16(o[a][j * 4 + w], a0, a1, a2, a3, b0[0][a], b1[0][a]);
        }
      }
    }
    load_v(n + kStages, where);
  }
  wait_copies<0>();
  if (owns_tail && tile == 0)
    if (tid < D / 4) {  // append; nobody reads this place before the next launch
      const int i = tid % (D / 8);
      __nv_bfloat16* to = (tid < D / 8 ? c.k_tail : c.v_tail) + tail_at + (size_t)place * D;
      reinterpret_cast<uint4*>(to)[i] = (tid < D / 8 ? sm.new_k : sm.new_v)[i];
    }
  if (bad) sm.bad = 1;

  // The kernel behind this one may be placed now; at the start it would take places that are left by CTAs of different lengths.
  ptx::griddep_launch_dependents();
  __syncthreads();  // the rings and q are not needed any more

  // ---- join the warps --------------------------------------------------------------------------------------------------------------
#pragma unroll
  for (int a = 0; a < NT; ++a) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[a][h] += __shfl_xor_sync(0xffffffffu, l[a][h], 4);
      l[a][h] += __shfl_xor_sync(0xffffffffu, l[a][h], 8);
      l[a][h] += __shfl_xor_sync(0xffffffffu, l[a][h], 16);
      if (g == 0) {
        sm.m[warp][a * 8 + 2 * t + h] = m[a][h];
        sm.l[warp][a * 8 + 2 * t + h] = l[a][h];
      }
    }
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(&sm.o[warp][(a * 8 + 2 * t + e) * S::OP + g * S::OS + 2 * i]) = make_float2(o[a][i][e], o[a][i][e + 2]);
  }
  __syncthreads();
  const bool any_bad = sm.bad != 0;
  constexpr int PR = D / 2;  // pairs of dims of a row
#pragma unroll 4
  for (int i = tid; i < rows * PR; i += kThreads) {
    const int r = i / PR, d = 2 * (i % PR);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm.m[w][r]);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float x = sm.m[w][r] == -INFINITY ? 0.f : exp2_fast(sm.m[w][r] - M);
      const float2 v = *reinterpret_cast<const float2*>(&sm.o[w][r * S::OP + d / (D / 8) * S::OS + d % (D / 8)]);
      L += sm.l[w][r] * x;
      x0 += v.x * x;
      x1 += v.y * x;
    }
    // (a sum below zero: a page outside the pool)
    if (sp.used == 1) {
      const float inv = 1.f / L;
      reinterpret_cast<uint32_t*>(out + (size_t)r * D)[d / 2] = any_bad ? 0 : pack_bf16(x0 * inv, x1 * inv);
    } else if (p.cluster) {
      sm.joined[r * (PR + 1) + d / 2] = make_float2(x0, x1);
      if (d == 0) sm.joined[r * (PR + 1) + PR] = make_float2(M, any_bad ? -1.f : L);
    } else {
      float* part = p.partials + (((size_t)b * p.n_heads + head0 + r) * p.nsplit + split) * (D + 2);
      *reinterpret_cast<float2*>(part + 2 + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(part) = make_float2(M, any_bad ? -1.f : L);
    }
  }
  if (sp.used == 1 || !p.cluster) return;
  // ---- join the splits, which are the CTAs of the cluster (those without work have left): each takes its share of the rows -------------
  ptx::cluster_arrive();
  ptx::cluster_wait();
  for (int i = split * kThreads + tid; i < rows * PR; i += sp.used * kThreads) {
    const int r = i / PR, at = r * (PR + 1);
    const uint32_t out_at = ptx::smem_u32(&sm.joined[at + i % PR]), ml_at = ptx::smem_u32(&sm.joined[at + PR]);
    float2 ml[kMaxCluster], x[kMaxCluster];
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k)
      if (k < sp.used) {
        ml[k] = ld_cluster(ptx::mapa(ml_at, k));
        x[k] = ld_cluster(ptx::mapa(out_at, k));
      }
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k)
      if (k < sp.used) M = fmaxf(M, ml[k].x);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
    bool zero = false;
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k)
      if (k < sp.used) {
        const float w = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - M);
        zero = zero || ml[k].y < 0.f;
        L += ml[k].y * w;
        x0 += x[k].x * w;
        x1 += x[k].y * w;
      }
    reinterpret_cast<uint32_t*>(out + (size_t)r * D)[i % PR] = zero ? 0 : pack_bf16(x0 / L, x1 / L);
  }
  ptx::cluster_arrive();  // nobody leaves while its results are read
  ptx::cluster_wait();
}

// Joins the splits of a sequence that has more than one, where they are too many for a cluster.
template <int D>
__global__ void __launch_bounds__(D) merge_splits_kernel(const DecodeAttn8Params p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int pos = p.positions[b];
  if (!position_ok(p, pos)) return;
  const int used = split_of(pos, p).used;
  if (used == 1) return;
  const float* part = p.partials + ((size_t)b * p.n_heads + h) * p.nsplit * (D + 2);
  float M = -INFINITY;
  for (int i = 0; i < used; ++i) M = fmaxf(M, part[(size_t)i * (D + 2)]);
  float L = 0.f, acc = 0.f;
  bool zero = false;
#pragma unroll 4
  for (int i = 0; i < used; ++i) {
    const float* x = part + (size_t)i * (D + 2);
    const float w = x[0] == -INFINITY ? 0.f : exp2_fast(x[0] - M);
    zero = zero || x[1] < 0.f;
    L += x[1] * w;
    acc += x[2 + d] * w;
  }
  p.out[(size_t)b * p.out_stride + (size_t)h * D + d] = __float2bfloat16(zero ? 0.f : acc / L);
}

template <int D, int NT, bool INT8, int W>
cudaError_t launch(const DecodeAttn8Params& p, cudaStream_t stream) {
  auto kern = decode_attention8_kernel<D, NT, INT8, W>;
  static DeviceOnce configured;
  if (configured.pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D, NT, W>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    configured.done();
  }
  const int group = p.n_heads / p.cache.n_kv_heads, tiles = (group + 8 * NT - 1) / (8 * NT);
  const long long pairs = (long long)p.batch * p.cache.n_kv_heads * tiles, quantisers = (long long)p.batch * p.cache.n_kv_heads;
  const long long ctas = (pairs + (quantisers + p.nsplit - 1) / p.nsplit) * p.nsplit;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = sizeof(Smem<D, NT, W>);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  // Placed before its predecessor has ended, a CTA hides its launch (16 sequences of 1087: 34.6 instead of 36.9 us, launched one by one; one of 1000:
  // 8.1 instead of 10.3). But clusters go where that one leaves room for all their CTAs, and of long pieces some SMs then have two and others
  // none for long (7 sequences of 65521 in clusters of five, behind themselves: 166 us with, 157 without).
  const bool short_pieces = (long long)p.max_blocks * p.cache.block <= 512LL * p.nsplit;
  cfg.numAttrs = short_pieces || !p.cluster ? pdl_launch_attr(&attr[0]) : 0;
  if (p.cluster) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = p.nsplit;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return e;
  launch_count_add(1);
  if (p.nsplit == 1 || p.cluster) return cudaSuccess;
  cfg.gridDim = dim3(p.n_heads, p.batch);
  cfg.blockDim = dim3(D);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  e = cudaLaunchKernelEx(&cfg, merge_splits_kernel<D>, p);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}
template <int D, int NT, int W>
cudaError_t by_code(const DecodeAttn8Params& p, cudaStream_t s) {
  return p.cache.int8 ? launch<D, NT, true, W>(p, s) : launch<D, NT, false, W>(p, s);
}
template <int D>
cudaError_t by_shape(const DecodeAttn8Params& p, cudaStream_t s) {
  if (p.n_heads / p.cache.n_kv_heads > 8) return by_code<D, 2, 4>(p, s);
  return p.warps == 3 ? by_code<D, 1, 3>(p, s) : (p.warps == 4 ? by_code<D, 1, 4>(p, s) : by_code<D, 1, 6>(p, s));
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace

void decode_attention8_split(DecodeAttn8Params& p) {
  const int group = p.n_heads / p.cache.n_kv_heads;
  const int tile = group > 8 ? 2 : 1, r = 8 * tile;  // query rows of a CTA
  const long long pairs = (long long)p.batch * p.cache.n_kv_heads * ((group + r - 1) / r);
  // At most: how long the sequences are only the GPU knows. A table that is much wider than they are costs (16 of 1087: 34 us in one of 8192 positions,
  // 72 in one of 32768, 215 in one of 131072).
  const long long units = (long long)p.max_blocks * (p.cache.block / 16);
  // The CTAs whose number comes nearest to what the GPU holds (us at W 6 / 4 / 3: 512 pairs, 16 sequences of 1087, 41 / 43 / 34; 264 pairs, 33
  // ragged ones, 33 / 37 / 37; 56 pairs of 65521 positions 157 / 163 / 161; 32 of 1000 8.1 / 8.4 / 8.4). Of equals those that fit at once,
  // and then the larger.
  double best = 0;
  long long best_waves = 0;
  for (int W : {6, 4, 3}) {
    if (tile == 2 && W != 4) continue;
    const int places = 148 * ctas_per_sm(tile, W);
    // As many CTAs as the GPU holds at a time, or, where there are more pairs than that, splits of kChunk units; none shorter than a pair of
    // units for each warp.
    const int least = pairs <= places ? least_units(W) : kChunk;
    const long long want = pairs <= places ? places / pairs : (units + kChunk - 1) / kChunk;
    int nsplit = (int)std::max(1ll, std::min({want, (long long)kMaxSplits, (units + least - 1) / least}));
    // The CTAs of a sequence are a cluster, which joins their results without a second launch, unless there is so much for so few heads
    // that more of them pay.
    if (nsplit > kMaxCluster && units <= kMaxCluster * 64) nsplit = kMaxCluster;
    const long long ctas = pairs * nsplit, waves = (ctas + places - 1) / places;
    const double fill = (double)ctas / (double)(waves * places);
    if (fill > best + 1e-9 || (fill > best - 1e-9 && waves < best_waves)) {
      best = fill;
      best_waves = waves;
      p.warps = W;
      p.nsplit = nsplit;
      p.least = least;
    }
  }
  p.cluster = p.nsplit > 1 && p.nsplit <= kMaxCluster;
}

size_t decode_attention8_partial_floats(const DecodeAttn8Params& p) {
  return p.nsplit > 1 && !p.cluster ? (size_t)p.batch * p.n_heads * p.nsplit * (p.cache.head_dim + 2) : 0;
}

cudaError_t decode_attention8(const DecodeAttn8Params& p, cudaStream_t stream) {
  const KvCache8& c = p.cache;
  if (p.batch == 0) return cudaSuccess;
  if (p.batch < 0 || p.batch > 65535 || p.nsplit < 1 || c.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % c.n_kv_heads != 0 || p.n_heads > 65535) return cudaErrorInvalidValue;
  if (c.block < 16 || c.block > 128 || (c.block & (c.block - 1)) != 0 || p.max_blocks < 1 || c.num_blocks < 1 || c.requests < p.batch) return cudaErrorInvalidValue;
  if (p.nsplit > 1 && !p.cluster && !p.partials) return cudaErrorInvalidValue;
  if (!aligned16(p.qkv) || !aligned16(c.k) || !aligned16(c.v) || !aligned16(c.k_tail) || !aligned16(c.v_tail) || !aligned16(p.out)) return cudaErrorInvalidValue;
  if (p.qkv_stride % 8 != 0 || p.out_stride % 8 != 0) return cudaErrorInvalidValue;
  if (c.head_dim == 128) return by_shape<128>(p, stream);
  if (c.head_dim == 64) return by_shape<64>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace ccl
