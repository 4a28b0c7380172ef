// Single-token attention over the 8-bit paged cache, fused with rotary embedding, append and the quantisation of a block that fills up.
//
// Bound by memory: 2 * head_dim bytes per cached position and KV head. All query heads of a KV head (a tile of eight) go through one CTA,
// so that a code is read and widened once for them. Per 16 positions a warp multiplies transposed: scores^T = K q^T and then
// out^T = V^T p^T, with the eight query heads as the N side of m16n8k16. K's rows and V's columns are then the A operand, whose fragments
// ask of a thread four codes of a row (K) or of a column (V); since the sum over k does not care for its order, a thread takes 16
// neighbouring bytes of a row and uses them as its k indices of four products (the queries are read in the same order), so that all of K
// and V goes from global memory into the registers that the products read, 16 bytes a load and whole lines a warp, with no shared memory
// and no barrier in the loop. (tcgen05 wants its operands in shared memory, widened: a round trip for every byte and 128 rows for at most
// 16; with eight rows the products take a sixth of the time that the bytes take to arrive.)
//
// Exactness. Codes widen to f16 without rounding. q is multiplied by a power of two that brings its largest element to 2^9 .. 2^10 and
// split into two f16 parts (22 bits), so scores are as exact as in fp32. The page's V scale joins the score, as log2(scale): weights
// 2^(s + log2 vs - m) multiply the codes in f16, kept within a factor of 2^15 of the running reference, and the sum of the softmax takes
// them divided by vs, in fp32. The reference m moves only when a score passes it by 2^15, and starts 2^8 below the maximum.
// The tail (bf16, at most a block) is done in fp32 on the CUDA cores.
#include "kv_cache8.cuh"

#include "gemm.h"

#include <algorithm>

namespace ccl {
namespace {

using namespace kv8;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMinUnits = 16;      // units of 16 positions per split at least: four for each warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 8.f;       // the reference starts this far (log2) below the maximum
constexpr float kRoom = 15.f;      // and moves when a weight would pass 2^15 (f16 ends at 2^16)

// Work split of one sequence: `per` units of 16 paged positions for each of `used` splits; the last one takes the tail too.
struct Split {
  int units, per, used;
};
__device__ __forceinline__ Split split_of(int pos, int block, int nsplit) {
  Split s;
  s.units = (pos / block) * (block / 16);
  s.per = max(kMinUnits, (s.units + nsplit - 1) / nsplit);
  s.used = max(1, (s.units + s.per - 1) / s.per);
  return s;
}
__device__ __forceinline__ bool position_ok(const DecodeAttn8Params& p, int pos) {
  return pos >= 0 && pos < p.table_rows && pos / p.cache.block < p.max_blocks;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four codes -> two f16 pairs, exactly.
template <bool INT8>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (INT8) {
    w ^= 0x80808080u;  // 0 .. 255 in the mantissa of 1024 + u, then minus 1152
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

template <int D, int NT>
struct Smem {
  static constexpr int R = 8 * NT;       // query rows
  static constexpr int QP = D + 4;       // pitch (halves): eight rows start two banks apart
  static constexpr int OP = D + 4;       // pitch (floats)
  __half qh[R * QP], ql[R * QP];         // q as two f16 parts
  float qf[R * D];                       // q in fp32, for the tail
  float o[kWarps][R * OP];               // out of each warp
  float m[kWarps][R], l[kWarps][R];
  float qs[R];                           // scale * log2 e over the power of two of the row
  uint32_t new_k[D / 2], new_v[D / 2];   // the new token, bf16
  uint32_t amax[2][kWarps];
  int bad;
};

// Quantises the block that the new token completes. `src`: 0 for K, 1 for V.
template <int D, bool INT8>
__device__ __forceinline__ void quantise_block(const __nv_bfloat16* tail, const uint32_t* fresh, int block, uint32_t (&amax)[kWarps], uint8_t* page, float* scale_out) {
  const int tid = threadIdx.x, n = block * D / 4;  // pieces of four values
  const int last = (block - 1) * (D / 4);          // from here on: the new token
  auto piece = [&](int i) {
    return i >= last ? make_uint2(fresh[(i - last) * 2], fresh[(i - last) * 2 + 1]) : *reinterpret_cast<const uint2*>(tail + (size_t)i * 4);
  };
  uint32_t seen = 0;
  for (int i = tid; i < n; i += kThreads) {
    const uint2 w = piece(i);
    seen = amax_bits(amax_bits(seen, w.x), w.y);
  }
  seen = __reduce_max_sync(0xffffffffu, seen);
  if ((tid & 31) == 0) amax[tid >> 5] = seen;
  __syncthreads();
  seen = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) seen = max(seen, amax[w]);
  const float scale = scale_of<INT8>(bits_f(seen));
  for (int i = tid; i < n; i += kThreads) {
    const uint2 w = piece(i);
    *reinterpret_cast<uint32_t*>(page + (size_t)i * 4) = codes4<INT8>(lo_f(w.x), hi_f(w.x), lo_f(w.y), hi_f(w.y), scale);
  }
  if (tid == 0) *scale_out = scale;
}

template <int D, int NT, bool INT8>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) decode_attention8_kernel(const DecodeAttn8Params p) {
  constexpr int R = 8 * NT;
  constexpr int KJ = D / 64;        // 16-byte loads of a K row by a thread
  constexpr int VW = D / 32;        // words of a V row by a thread
  constexpr int NM = D / 16;        // products over the dims
  using S = Smem<D, NT>;
  extern __shared__ __align__(16) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);

  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const KvCache8& c = p.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / c.n_kv_heads;
  const int tiles = (group + R - 1) / R;
  const int kvh = blockIdx.y / tiles, tile = blockIdx.y - kvh * tiles;
  const int rows = min(R, group - tile * R);
  const int head0 = kvh * group + tile * R;
  const int b = blockIdx.z, split = blockIdx.x;
  const int pos = p.positions[b];
  __nv_bfloat16* out = p.out + (size_t)b * p.out_stride + (size_t)head0 * D;
  if (!position_ok(p, pos)) {
    if (split == 0)
      for (int i = tid; i < rows * D; i += kThreads) out[i] = __float2bfloat16(0.f);
    return;
  }
  const Split sp = split_of(pos, c.block, p.nsplit);
  if (split >= sp.used) return;
  const bool owns_tail = split == sp.used - 1;
  const int* table = p.table + (size_t)b * p.max_blocks;

  // ---- the loop's loads: unit n of this warp is unit u0 + warp + 4 n of the sequence -------------------------------------------
  const int u0 = split * sp.per, u1 = min(sp.units, u0 + sp.per);
  const int n_units = max(0, (u1 - u0 - warp + kWarps - 1) / kWarps);
  const int in_block = 31 - __clz(c.block / 16);  // log2 of the units of a block
  bool bad = false;
  auto page_of = [&](int n) {  // of the window's lane
    int page = 0;
    if (n < n_units) {
      page = table[(u0 + warp + kWarps * n) >> in_block];
      if ((unsigned)page >= (unsigned)c.num_blocks) {
        bad = true;
        page = 0;
      }
    }
    return page;
  };
  // a window of 32 units: each lane looks up one page and its scales
  int pages = page_of(lane), pages_next = page_of(32 + lane);
  float ks_next = 1.f, vs_next = 1.f;
  auto scales_of = [&](int n) {
    if (n < n_units) {
      const size_t at = (size_t)pages * c.n_kv_heads + kvh;
      ks_next = c.k_scale[at];
      vs_next = c.v_scale[at];
    }
  };
  uint4 kr[2][KJ];
  uint32_t vr[4][VW];
  size_t at = 0;  // byte offset of the unit in both pools
  auto load_k = [&](int n) {
    if (n >= n_units) return;  // uniform
    if (n > 0 && (n & 31) == 0) {
      pages = pages_next;
      scales_of(n + lane);
      pages_next = page_of(n + 32 + lane);
    }
    const int page = __shfl_sync(0xffffffffu, pages, n & 31);
    const int u = u0 + warp + kWarps * n;
    at = (((size_t)page * c.n_kv_heads + kvh) * c.block + (size_t)(u & ((1 << in_block) - 1)) * 16) * D;
    const uint8_t* k = c.k + at + g * D + t * 16;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      kr[0][j] = ptx::ld_nc_v4(k + j * 64);
      kr[1][j] = ptx::ld_nc_v4(k + 8 * D + j * 64);
    }
  };
  auto load_v = [&](int n) {
    if (n >= n_units) return;
    const uint8_t* v = c.v + at + g * (D / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* row = v + (2 * t + (i & 1) + (i >> 1) * 8) * D;
      if constexpr (VW == 4) {
        const uint4 x = ptx::ld_nc_v4(row);
        vr[i][0] = x.x, vr[i][1] = x.y, vr[i][2] = x.z, vr[i][3] = x.w;
      } else {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(row));
        vr[i][0] = x.x, vr[i][1] = x.y;
      }
    }
  };
  scales_of(lane);
  load_k(0);
  load_v(0);

  // ---- q: rotate, split; the new token ------------------------------------------------------------------------------------------
  const __nv_bfloat16* qkv = p.qkv + (size_t)b * p.qkv_stride;
  const float* cosr = p.cos + (size_t)pos * (D / 2);
  const float* sinr = p.sin + (size_t)pos * (D / 2);
  constexpr int PP = D / 64;  // rotated pairs of a lane
  for (int r = warp; r < R; r += kWarps) {
    float x[PP], y[PP], most = 0.f;
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int d = lane + 32 * i;
      x[i] = y[i] = 0.f;
      if (r < rows) {
        const __nv_bfloat16* src = qkv + (size_t)(head0 + r) * D;
        rotate(__bfloat162float(src[d]), __bfloat162float(src[d + D / 2]), cosr[d], sinr[d], x[i], y[i]);
      }
      most = fmaxf(most, fmaxf(fabsf(x[i]), fabsf(y[i])));
    }
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
    const int e = (int)(__float_as_uint(most) >> 23);  // biased exponent; 0 for a row of zeros, 255 for an infinity
    const int up = e == 0 || e == 255 ? 127 : min(254, 127 + 9 + 127 - e);
    const float mult = __uint_as_float((uint32_t)up << 23);
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int d = lane + 32 * i;
      const float z[2] = {x[i], y[i]};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int dd = d + h * (D / 2);
        const float v = z[h] * mult;
        const __half hi = __float2half_rn(v);
        sm.qh[r * S::QP + dd] = hi;
        sm.ql[r * S::QP + dd] = __float2half_rn(v - __half2float(hi));
        sm.qf[r * D + dd] = z[h];
      }
    }
    if (lane == 0) sm.qs[r] = p.scale * kLog2e / mult;
  }
  const int place = pos & (c.block - 1);
  const size_t tail_at = ((size_t)b * c.n_kv_heads + kvh) * c.block * D;
  if (owns_tail && tid < D / 2) {
    // thread i < D/4 holds dims 2i, 2i + 1 of K and their partners; the others V
    const __nv_bfloat16* kn = qkv + (size_t)(p.n_heads + kvh) * D;
    const __nv_bfloat16* vn = kn + (size_t)c.n_kv_heads * D;
    if (tid < D / 4) {
      const uint32_t a = reinterpret_cast<const uint32_t*>(kn)[tid], h = reinterpret_cast<const uint32_t*>(kn)[tid + D / 4];
      float x0, y0, x1, y1;
      rotate(lo_f(a), lo_f(h), cosr[2 * tid], sinr[2 * tid], x0, y0);
      rotate(hi_f(a), hi_f(h), cosr[2 * tid + 1], sinr[2 * tid + 1], x1, y1);
      sm.new_k[tid] = pack_bf16(x0, x1);
      sm.new_k[tid + D / 4] = pack_bf16(y0, y1);
    } else {
      const int i = tid - D / 4;
      sm.new_v[i] = reinterpret_cast<const uint32_t*>(vn)[i];
      sm.new_v[i + D / 4] = reinterpret_cast<const uint32_t*>(vn)[i + D / 4];
    }
  }
  if (tid == 0) sm.bad = 0;
  __syncthreads();

  // ---- state of the softmax: column 2t and 2t + 1 of each tile of eight queries ---------------------------------------------------
  float o[NT][NM][4], m[NT][2], l[NT][2], f[NT][2];
#pragma unroll
  for (int a = 0; a < NT; ++a) {
#pragma unroll
    for (int i = 0; i < NM; ++i) o[a][i][0] = o[a][i][1] = o[a][i][2] = o[a][i][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[a][h] = -INFINITY;
      l[a][h] = 0.f;
      f[a][h] = sm.qs[a * 8 + 2 * t + h];
    }
  }

  // ---- the tail, one position per warp at a time: lanes share the dims -------------------------------------------------------------
  if (owns_tail) {
    constexpr int E = D / 32;  // dims of a lane
    if (tile == 0 && tid < D / 2) {  // append; nobody reads this place before the next launch
      reinterpret_cast<uint32_t*>(c.k_tail + tail_at + (size_t)place * D)[tid] = sm.new_k[tid];
      reinterpret_cast<uint32_t*>(c.v_tail + tail_at + (size_t)place * D)[tid] = sm.new_v[tid];
    }
    float to[R][E], tm[R], tl[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      tm[r] = -INFINITY;
      tl[r] = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) to[r][i] = 0.f;
    }
    for (int j = warp; j <= place; j += kWarps) {
      const uint32_t* kp = j == place ? sm.new_k : reinterpret_cast<const uint32_t*>(c.k_tail + tail_at + (size_t)j * D);
      const uint32_t* vp = j == place ? sm.new_v : reinterpret_cast<const uint32_t*>(c.v_tail + tail_at + (size_t)j * D);
      float kk[E], vv[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const uint32_t kw = kp[lane * (E / 2) + i], vw = vp[lane * (E / 2) + i];
        kk[2 * i] = lo_f(kw), kk[2 * i + 1] = hi_f(kw);
        vv[2 * i] = lo_f(vw), vv[2 * i + 1] = hi_f(vw);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= rows) break;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += sm.qf[r * D + lane * E + i] * kk[i];
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= p.scale * kLog2e;
        const float mn = fmaxf(tm[r], s);
        const float corr = exp2_fast(tm[r] - mn), w = exp2_fast(s - mn);
        tl[r] = tl[r] * corr + w;
#pragma unroll
        for (int i = 0; i < E; ++i) to[r][i] = to[r][i] * corr + w * vv[i];
        tm[r] = mn;
      }
    }
    // into the layout of the products, through this warp's part of shared memory
    const float up = 256.f;  // 2^kHead
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < E; ++i) sm.o[warp][r * S::OP + lane * E + i] = to[r][i] * up;
      if (lane == 0) {
        sm.m[warp][r] = tm[r] - kHead;
        sm.l[warp][r] = tl[r] * up;
      }
    }
    __syncwarp();
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
      for (int i = 0; i < NM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[a][i][e] = sm.o[warp][(a * 8 + 2 * t + (e & 1)) * S::OP + g * (D / 8) + 2 * i + (e >> 1)];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m[a][h] = sm.m[warp][a * 8 + 2 * t + h];
        l[a][h] = g == 0 ? sm.l[warp][a * 8 + 2 * t + h] : 0.f;
      }
    }
    __syncwarp();
  }

  // ---- the pages -----------------------------------------------------------------------------------------------------------------
  float ks = 1.f, lvs = 0.f, ivs = 1.f;  // of the window's lane
  for (int n = 0; n < n_units; ++n) {
    if ((n & 31) == 0) {
      ks = ks_next;
      lvs = log2f(vs_next);
      ivs = __frcp_rn(vs_next);
    }
    float s[NT][4], s2[NT][4];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[a][e] = s2[a][e] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const uint32_t r0[4] = {kr[0][j].x, kr[0][j].y, kr[0][j].z, kr[0][j].w}, r8[4] = {kr[1][j].x, kr[1][j].y, kr[1][j].z, kr[1][j].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t a0, a1, a2, a3;
        widen<INT8>(r0[w], a0, a2);
        widen<INT8>(r8[w], a1, a3);
#pragma unroll
        for (int a = 0; a < NT; ++a) {
          const int q = (a * 8 + g) * S::QP + j * 64 + t * 16 + w * 4;
          const uint2 h = *reinterpret_cast<const uint2*>(&sm.qh[q]), lo = *reinterpret_cast<const uint2*>(&sm.ql[q]);
          mma(s[a], a0, a1, a2, a3, h.x, h.y);
          mma(s2[a], a0, a1, a2, a3, lo.x, lo.y);
        }
      }
    }
    load_k(n + 1);
    const float uks = __shfl_sync(0xffffffffu, ks, n & 31), ulv = __shfl_sync(0xffffffffu, lvs, n & 31), uiv = __shfl_sync(0xffffffffu, ivs, n & 31);
    bool over = false;
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[a][e] = (s[a][e] + s2[a][e]) * (f[a][e & 1] * uks) + ulv;
      over = over || fmaxf(s[a][0], s[a][2]) - m[a][0] > kRoom || fmaxf(s[a][1], s[a][3]) - m[a][1] > kRoom;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(s[a][h], s[a][h + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          if (top - m[a][h] > kRoom) {
            const float corr = exp2_fast(m[a][h] - (top - kHead));
            m[a][h] = top - kHead;
            l[a][h] *= corr;
#pragma unroll
            for (int i = 0; i < NM; ++i) {
              o[a][i][h] *= corr;
              o[a][i][h + 2] *= corr;
            }
          }
        }
    }
    uint32_t b0[NT], b1[NT];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const float w0 = exp2_fast(s[a][0] - m[a][0]), w1 = exp2_fast(s[a][1] - m[a][1]);
      const float w2 = exp2_fast(s[a][2] - m[a][0]), w3 = exp2_fast(s[a][3] - m[a][1]);
      l[a][0] += (w0 + w2) * uiv;
      l[a][1] += (w1 + w3) * uiv;
      b0[a] = transpose8x8(pack_f16(w0, w1));
      b1[a] = transpose8x8(pack_f16(w2, w3));
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t a0, a1, a2, a3;
        widen<INT8>(__byte_perm(vr[0][w], vr[1][w], h ? 0x7362 : 0x5140), a0, a1);
        widen<INT8>(__byte_perm(vr[2][w], vr[3][w], h ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
        for (int a = 0; a < NT; ++a) mma(o[a][2 * w + h], a0, a1, a2, a3, b0[a], b1[a]);
      }
    }
    load_v(n + 1);
  }
  if (bad) sm.bad = 1;

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
      for (int e = 0; e < 4; ++e) sm.o[warp][(a * 8 + 2 * t + (e & 1)) * S::OP + g * (D / 8) + 2 * i + (e >> 1)] = o[a][i][e];
  }
  __syncthreads();
  const bool any_bad = sm.bad != 0;
  for (int r = tid / D; r < rows; r += kThreads / D) {
    const int d = tid & (D - 1);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.m[w][r]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float x = sm.m[w][r] == -INFINITY ? 0.f : exp2_fast(sm.m[w][r] - M);
      L += sm.l[w][r] * x;
      acc += sm.o[w][r * S::OP + d] * x;
    }
    if (sp.used == 1) {
      out[(size_t)r * D + d] = __float2bfloat16(any_bad ? 0.f : acc / L);
    } else {
      float* part = p.partials + (((size_t)b * p.n_heads + head0 + r) * p.nsplit + split) * (D + 2);
      part[2 + d] = acc;
      if (d == 0) {
        part[0] = any_bad ? INFINITY : M;
        part[1] = L;
      }
    }
  }

  // ---- the block is full: quantise it ------------------------------------------------------------------------------------------------
  if (owns_tail && tile == 0 && place == c.block - 1) {
    const int page = table[pos / c.block];
    if ((unsigned)page < (unsigned)c.num_blocks) {
      const size_t at8 = ((size_t)page * c.n_kv_heads + kvh) * c.block * D, sc = (size_t)page * c.n_kv_heads + kvh;
      quantise_block<D, INT8>(c.k_tail + tail_at, sm.new_k, c.block, sm.amax[0], c.k + at8, c.k_scale + sc);
      quantise_block<D, INT8>(c.v_tail + tail_at, sm.new_v, c.block, sm.amax[1], c.v + at8, c.v_scale + sc);
    }
  }
}

// Joins the splits of a sequence that has more than one.
template <int D>
__global__ void __launch_bounds__(D) merge_splits_kernel(const DecodeAttn8Params p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int pos = p.positions[b];
  if (!position_ok(p, pos)) return;
  const int used = split_of(pos, p.cache.block, p.nsplit).used;
  if (used == 1) return;
  const float* part = p.partials + ((size_t)b * p.n_heads + h) * p.nsplit * (D + 2);
  float M = -INFINITY;
  for (int i = 0; i < used; ++i) M = fmaxf(M, part[(size_t)i * (D + 2)]);
  float L = 0.f, acc = 0.f;
#pragma unroll 4
  for (int i = 0; i < used; ++i) {
    const float* x = part + (size_t)i * (D + 2);
    const float w = x[0] == -INFINITY ? 0.f : exp2_fast(x[0] - M);
    L += x[1] * w;
    acc += x[2 + d] * w;
  }
  p.out[(size_t)b * p.out_stride + (size_t)h * D + d] = __float2bfloat16(M == INFINITY ? 0.f : acc / L);
}

template <int D, int NT, bool INT8>
cudaError_t launch(const DecodeAttn8Params& p, cudaStream_t stream) {
  auto kern = decode_attention8_kernel<D, NT, INT8>;
  static DeviceOnce configured;
  if (configured.pending()) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D, NT>));
    if (e != cudaSuccess) return e;
    configured.done();
  }
  const int group = p.n_heads / p.cache.n_kv_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.nsplit, p.cache.n_kv_heads * ((group + 8 * NT - 1) / (8 * NT)), p.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Smem<D, NT>);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = pdl_launch_attr(&attr[0]);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return e;
  launch_count_add(1);
  if (p.nsplit == 1) return cudaSuccess;
  cfg.gridDim = dim3(p.n_heads, p.batch);
  cfg.blockDim = dim3(D);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, merge_splits_kernel<D>, p);
  if (e == cudaSuccess) launch_count_add(1);
  return e;
}
template <int D, int NT>
cudaError_t by_code(const DecodeAttn8Params& p, cudaStream_t s) {
  return p.cache.int8 ? launch<D, NT, true>(p, s) : launch<D, NT, false>(p, s);
}
template <int D>
cudaError_t by_tile(const DecodeAttn8Params& p, cudaStream_t s) {
  return p.n_heads / p.cache.n_kv_heads > 8 ? by_code<D, 2>(p, s) : by_code<D, 1>(p, s);
}

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace

int decode_attention8_splits(const DecodeAttn8Params& p) {
  const int group = p.n_heads / p.cache.n_kv_heads;
  const int r = group > 8 ? 16 : 8;
  const long long pairs = (long long)p.batch * p.cache.n_kv_heads * ((group + r - 1) / r);
  // about four CTAs for every place (four on an SM), so that sequences of different lengths even out, of at least kMinUnits units
  const long long cap = ((long long)p.max_blocks * (p.cache.block / 16) + kMinUnits - 1) / kMinUnits;
  return (int)std::max(1ll, std::min({4ll * 4 * 148 / std::max(1ll, pairs), cap, 64ll}));
}

size_t decode_attention8_partial_floats(const DecodeAttn8Params& p) {
  return p.nsplit > 1 ? (size_t)p.batch * p.n_heads * p.nsplit * (p.cache.head_dim + 2) : 0;
}

cudaError_t decode_attention8(const DecodeAttn8Params& p, cudaStream_t stream) {
  const KvCache8& c = p.cache;
  if (p.batch == 0) return cudaSuccess;
  if (p.batch < 0 || p.batch > 65535 || p.nsplit < 1 || c.n_kv_heads < 1 || p.n_heads < 1 || p.n_heads % c.n_kv_heads != 0 || p.n_heads > 65535) return cudaErrorInvalidValue;
  if (c.block < 16 || c.block > 128 || (c.block & (c.block - 1)) != 0 || p.max_blocks < 1 || c.requests < p.batch) return cudaErrorInvalidValue;
  if (p.nsplit > 1 && !p.partials) return cudaErrorInvalidValue;
  if (!aligned16(p.qkv) || !aligned16(c.k) || !aligned16(c.v) || !aligned16(c.k_tail) || !aligned16(c.v_tail) || !aligned16(p.out)) return cudaErrorInvalidValue;
  if (p.qkv_stride % 8 != 0 || p.out_stride % 8 != 0) return cudaErrorInvalidValue;
  if (c.head_dim == 128) return by_tile<128>(p, stream);
  if (c.head_dim == 64) return by_tile<64>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace ccl
