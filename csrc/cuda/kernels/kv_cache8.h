// Host interface of the 8-bit paged KV cache: prompt append and single-token attention (no torch dependency).
//
// Layout. `block` (16, 32, 64 or 128) consecutive positions of one KV head share a page: 8-bit codes (e4m3 or int8, ties to even) and one
// fp32 scale for K and one for V. The block that a sequence is still filling is kept in bf16, its "tail"; when its last position arrives it
// is quantised, once: scale = max(amax / qmax, 2^-40) with qmax 448 or 127, code = round(x / scale). A page is therefore always full, and
// no value is rounded to 8 bits twice.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ccl {

struct KvCache8 {
  uint8_t* k;                // [num_blocks, n_kv_heads, block, head_dim]
  uint8_t* v;
  float* k_scale;            // [num_blocks, n_kv_heads]
  float* v_scale;
  __nv_bfloat16* k_tail;     // [requests, n_kv_heads, block, head_dim]
  __nv_bfloat16* v_tail;
  int num_blocks, n_kv_heads, block, head_dim, requests;
  bool int8;                 // codes: int8, else e4m3
};

// Rotary embedding and append of `rows` rows of a QKV projection (n_heads q heads, then k heads, then v heads). Row t belongs to
// request `requests[t]`, has position `positions[t]` and goes to `slots[t]` = page * block + place (kv_plan's arrays; the rows of a
// request are consecutive and so are their positions). A row whose request or position is outside the tables is skipped.
struct KvAppend8Params {
  const __nv_bfloat16* qkv;
  long long qkv_stride;      // elements, a multiple of 8
  __nv_bfloat16* rotated;    // [rows, (n_heads + n_kv_heads) * head_dim]: q and k after the rotation
  long long rotated_stride;
  const int* starts;         // [n_requests + 1] first row of each request
  const int* requests;       // [rows]
  const int* positions;
  const int* slots;
  const float* cos;          // [table_rows, head_dim / 2]
  const float* sin;
  int rows, n_requests, n_heads, table_rows;
  bool zero_rest;            // rows without a token: zeros in `rotated` (else left as they are)
  KvCache8 cache;
};
cudaError_t kv_append8(const KvAppend8Params& p, cudaStream_t stream);

// One new token for each of `batch` sequences: rotary embedding, append to the tail (and, when it fills the block, to its page),
// attention over positions 0 .. positions[b]. A position outside the block table or the rotary tables (-1: no sequence in this row)
// gives a row of zeros and writes nothing; a page number outside the pool, a row of zeros.
struct DecodeAttn8Params {
  const __nv_bfloat16* qkv;
  long long qkv_stride;
  const int* positions;      // [batch]
  const int* table;          // [batch, max_blocks]
  const float* cos;
  const float* sin;
  __nv_bfloat16* out;        // [batch, out_stride]
  long long out_stride;
  float* partials;           // decode_attention8_partial_floats() floats; unused when there is one split
  int batch, n_heads, max_blocks, table_rows;
  int nsplit, least, warps;  // set by decode_attention8_split()
  bool cluster;
  float scale;               // 1 / sqrt(head_dim)
  KvCache8 cache;
};
void decode_attention8_split(DecodeAttn8Params& p);
size_t decode_attention8_partial_floats(const DecodeAttn8Params& p);  // with the split set
cudaError_t decode_attention8(const DecodeAttn8Params& p, cudaStream_t stream);

}  // namespace ccl
