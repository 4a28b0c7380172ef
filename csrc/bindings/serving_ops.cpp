// Dispatcher registration of the serving operators on one GPU: paged 8-bit KV cache and token log-probabilities.
//
// Each op has one function that checks its arguments and gives its results' shapes, which the CUDA and the Meta kernel share, so that
// tracing refuses what a launch would refuse.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>
#include <torch/torch.h>

#include <cmath>

#include "cuda/kernels/kv_cache8.h"
#include "cuda/kernels/kv_plan.h"
#include "cuda/kernels/token_logprobs.h"

namespace {

using at::Tensor;
using c10::optional;

void ok(cudaError_t e, const char* op) { TORCH_CHECK(e == cudaSuccess, op, ": ", cudaGetErrorString(e)); }
cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream(); }

// Uninitialised tensors beside `like`.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  if (like.is_cuda()) return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
  return at::empty(sizes, like.options().dtype(type));
}
// Several small ones, on a GPU in one allocation: each costs the host a microsecond, of nine in a call.
template <size_t N>
std::array<Tensor, N> fresh_together(const Tensor& like, const std::array<std::pair<at::DimVector, at::ScalarType>, N>& what) {
  std::array<Tensor, N> out;
  if (!like.is_cuda()) {
    for (size_t i = 0; i < N; ++i) out[i] = fresh(what[i].first, what[i].second, like);
    return out;
  }
  auto bytes_of = [](const std::pair<at::DimVector, at::ScalarType>& w) {
    int64_t n = (int64_t)c10::elementSize(w.second);
    for (int64_t d : w.first) n *= d;
    return (n + 15) / 16 * 16;
  };
  int64_t total = 0;
  for (const auto& w : what) total += bytes_of(w);
  const Tensor all = at::detail::empty_cuda({total}, at::kByte, like.device(), c10::nullopt);
  int64_t at = 0;
  for (size_t i = 0; i < N; ++i) {
    out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(what[i].second));
    auto* t = out[i].unsafeGetTensorImpl();
    t->set_storage_offset(at / (int64_t)c10::elementSize(what[i].second));
    t->set_sizes_contiguous(what[i].first);
    at += bytes_of(what[i]);
  }
  return out;
}

// A tensor of this type, rank, device and layout (all dimensions dense).
void expect(const Tensor& t, const char* op, const char* name, at::ScalarType type, int64_t dim, const Tensor& like) {
  TORCH_CHECK(t.scalar_type() == type, op, ": ", name, " must be ", type, ", not ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must have ", dim, " dimension(s), not ", t.dim());
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(), ", the first argument on ", like.device());
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
}
// Rows of a 2-D bf16 tensor that the kernels read or write 16 bytes at a time.
void expect_rows(const Tensor& t, const char* op, const char* name, const Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.dim() == 2, op, ": ", name, " must be a 2-D bf16 tensor");
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " is on ", t.device(), ", the first argument on ", like.device());
  TORCH_CHECK(t.size(1) == 0 || t.stride(1) == 1, op, ": ", name, "'s innermost dimension must be contiguous");
  TORCH_CHECK(t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)), op, ": ", name, "'s row stride must be a multiple of 8 elements and no shorter than a row");
  TORCH_CHECK(t.size(0) <= 0x7fffffff, op, ": ", name, " has too many rows");
}
void expect_aligned(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, op, ": ", name, " must start at a multiple of 16 bytes");
}
bool overlap(const Tensor& a, const Tensor& b) {
  auto range = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) == 0) return std::make_pair((uintptr_t)0, (uintptr_t)0);
      n += (t.size(d) - 1) * t.stride(d);
    }
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::make_pair(at, at + n * t.element_size());
  };
  const auto x = range(a), y = range(b);
  return x.first < y.second && y.first < x.second;
}

// ---- blocks of a pool -------------------------------------------------------------------------------------------------------------------
void check_blocks(const char* op, const Tensor& first, const Tensor& table, const Tensor& held, const Tensor& free_blocks, const Tensor& state) {
  expect(table, op, "table", at::kInt, 2, first);
  expect(held, op, "held", at::kInt, 1, first);
  expect(free_blocks, op, "free", at::kInt, 1, first);
  expect(state, op, "state", at::kInt, 1, first);
  const int64_t n = first.size(0);
  TORCH_CHECK(table.size(0) == n && held.size(0) == n, op, ": table and held must have one row for each of the ", n, " requests");
  TORCH_CHECK(n <= ccl::kMaxPlanRequests, op, ": at most ", ccl::kMaxPlanRequests, " requests, not ", n);
  TORCH_CHECK(table.size(1) >= 1 && std::max<int64_t>(n, 1024) * table.size(1) <= 0x7fffffff, op, ": a table of ", n, " x ", table.size(1), " entries is empty or too large");
  TORCH_CHECK(state.size(0) == 2, op, ": state has two words");
  TORCH_CHECK(free_blocks.size(0) <= 0x7fffffff, op, ": too many blocks");
}
ccl::KvBlocks blocks_of(const Tensor& table, const Tensor& held, const Tensor& free_blocks, const Tensor& state) {
  return {table.data_ptr<int>(), held.data_ptr<int>(), free_blocks.data_ptr<int>(), state.data_ptr<int>(), (int)table.size(0), (int)table.size(1), (int)free_blocks.size(0)};
}

using Plan = std::tuple<Tensor, Tensor, Tensor, Tensor>;
Plan plan_shapes(const Tensor& lengths, const optional<Tensor>& new_tokens, const Tensor& table, const Tensor& held, const Tensor& free_blocks, const Tensor& state, int64_t block, int64_t room) {
  const char* op = "kv_plan";
  expect(lengths, op, "lengths", at::kInt, 1, lengths);
  if (new_tokens) {
    expect(*new_tokens, op, "new_tokens", at::kInt, 1, lengths);
    TORCH_CHECK(new_tokens->size(0) == lengths.size(0), op, ": new_tokens must have one entry for each request");
  }
  check_blocks(op, lengths, table, held, free_blocks, state);
  TORCH_CHECK(block == 16 || block == 32 || block == 64 || block == 128, op, ": block_size must be 16, 32, 64 or 128, not ", block);
  TORCH_CHECK(room >= 0 && room < 0x7fffffff, op, ": max_tokens must be between 0 and 2^31 - 2");
  TORCH_CHECK(free_blocks.size(0) * block <= 0x7fffffff, op, ": slots are 32-bit: ", free_blocks.size(0), " blocks of ", block, " are too many");
  auto t = fresh_together<4>(lengths, {{{{lengths.size(0) + 1}, at::kInt}, {{room}, at::kInt}, {{room}, at::kInt}, {{room}, at::kInt}}});
  return {t[0], t[1], t[2], t[3]};
}
Plan kv_plan_cuda(const Tensor& lengths, const optional<Tensor>& new_tokens, Tensor& table, Tensor& held, Tensor& free_blocks, Tensor& state, int64_t block, int64_t room) {
  c10::cuda::CUDAGuard g(lengths.device());
  Plan out = plan_shapes(lengths, new_tokens, table, held, free_blocks, state, block, room);
  ccl::KvPlanParams p;
  p.lengths = lengths.data_ptr<int>();
  p.new_tokens = new_tokens ? new_tokens->data_ptr<int>() : nullptr;
  p.starts = std::get<0>(out).data_ptr<int>();
  p.token_request = std::get<1>(out).data_ptr<int>();
  p.positions = std::get<2>(out).data_ptr<int>();
  p.slots = std::get<3>(out).data_ptr<int>();
  p.room = (int)room;
  p.block = (int)block;
  p.b = blocks_of(table, held, free_blocks, state);
  ok(ccl::kv_plan(p, stream()), "kv_plan");
  return out;
}
Plan kv_plan_meta(const Tensor& lengths, const optional<Tensor>& new_tokens, Tensor& table, Tensor& held, Tensor& free_blocks, Tensor& state, int64_t block, int64_t room) {
  return plan_shapes(lengths, new_tokens, table, held, free_blocks, state, block, room);
}

void check_release(const Tensor& finished, const Tensor& table, const Tensor& held, const Tensor& free_blocks, const Tensor& state) {
  expect(finished, "kv_release", "finished", at::kBool, 1, finished);
  check_blocks("kv_release", finished, table, held, free_blocks, state);
}
void kv_release_cuda(const Tensor& finished, Tensor& table, Tensor& held, Tensor& free_blocks, Tensor& state) {
  check_release(finished, table, held, free_blocks, state);
  c10::cuda::CUDAGuard g(finished.device());
  ok(ccl::kv_release(reinterpret_cast<const uint8_t*>(finished.data_ptr<bool>()), blocks_of(table, held, free_blocks, state), stream()), "kv_release");
}
void kv_release_meta(const Tensor& finished, Tensor& table, Tensor& held, Tensor& free_blocks, Tensor& state) { check_release(finished, table, held, free_blocks, state); }

// ---- the 8-bit cache ------------------------------------------------------------------------------------------------------------------------
void check_cache(const char* op, const Tensor& like, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt, const Tensor& cos, const Tensor& sin) {
  TORCH_CHECK(k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kChar, op, ": the cache's codes must be float8_e4m3fn or int8, not ", k.scalar_type());
  expect(k, op, "k", k.scalar_type(), 4, like);
  expect(v, op, "v", k.scalar_type(), 4, like);
  expect(ks, op, "k_scale", at::kFloat, 2, like);
  expect(vs, op, "v_scale", at::kFloat, 2, like);
  expect(kt, op, "k_tail", at::kBFloat16, 4, like);
  expect(vt, op, "v_tail", at::kBFloat16, 4, like);
  TORCH_CHECK(v.sizes() == k.sizes() && vt.sizes() == kt.sizes(), op, ": k and v must have the same sizes");
  const int64_t kv = k.size(1), block = k.size(2), dim = k.size(3);
  TORCH_CHECK(kv >= 1 && kv <= 65535, op, ": 1 to 65535 KV heads, not ", kv);
  TORCH_CHECK(block == 16 || block == 32 || block == 64 || block == 128, op, ": pages hold 16, 32, 64 or 128 positions, not ", block);
  TORCH_CHECK(dim == 64 || dim == 128, op, ": head_dim must be 64 or 128, not ", dim);
  TORCH_CHECK(ks.size(0) == k.size(0) && ks.size(1) == kv && vs.sizes() == ks.sizes(), op, ": scales must be [num_blocks, kv_heads]");
  TORCH_CHECK(kt.size(1) == kv && kt.size(2) == block && kt.size(3) == dim, op, ": tails must be [requests, kv_heads, block, head_dim]");
  TORCH_CHECK(k.size(0) * block <= 0x7fffffff && kt.size(0) <= 0x7fffffff, op, ": too many blocks or requests");
  TORCH_CHECK(k.size(0) >= 1, op, ": a pool without pages");  // (what is not there is read from page 0, with a weight of zero)
  expect(cos, op, "cos", at::kFloat, 2, like);
  expect(sin, op, "sin", at::kFloat, 2, like);
  TORCH_CHECK(cos.size(1) == dim / 2 && sin.sizes() == cos.sizes() && cos.size(0) <= 0x7fffffff, op, ": cos and sin must be [positions, head_dim / 2]");
}
ccl::KvCache8 cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& kt, const Tensor& vt) {
  ccl::KvCache8 c;
  c.k = static_cast<uint8_t*>(k.data_ptr());
  c.v = static_cast<uint8_t*>(v.data_ptr());
  c.k_scale = ks.data_ptr<float>();
  c.v_scale = vs.data_ptr<float>();
  c.k_tail = static_cast<__nv_bfloat16*>(kt.data_ptr());
  c.v_tail = static_cast<__nv_bfloat16*>(vt.data_ptr());
  c.num_blocks = (int)k.size(0);
  c.n_kv_heads = (int)k.size(1);
  c.block = (int)k.size(2);
  c.head_dim = (int)k.size(3);
  c.requests = (int)kt.size(0);
  c.int8 = k.scalar_type() == at::kChar;
  return c;
}
void expect_cache_aligned(const char* op, const Tensor& k, const Tensor& v, const Tensor& kt, const Tensor& vt, const Tensor& cos, const Tensor& sin) {
  expect_aligned(k, op, "k");
  expect_aligned(v, op, "v");
  expect_aligned(kt, op, "k_tail");
  expect_aligned(vt, op, "v_tail");
  expect_aligned(cos, op, "cos");
  expect_aligned(sin, op, "sin");
}

#define CACHE_ARGS Tensor &k, Tensor &v, Tensor &ks, Tensor &vs, Tensor &kt, Tensor &vt
#define CONST_CACHE_ARGS const Tensor &k, const Tensor &v, const Tensor &ks, const Tensor &vs, const Tensor &kt, const Tensor &vt
#define PLAN_ARGS const Tensor &starts, const Tensor &requests, const Tensor &positions, const Tensor &slots

void check_append(const Tensor& qkv, PLAN_ARGS, CONST_CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, const Tensor* out) {
  const char* op = "kv_append_8bit";
  expect_rows(qkv, op, "qkv", qkv);
  check_cache(op, qkv, k, v, ks, vs, kt, vt, cos, sin);
  expect(starts, op, "starts", at::kInt, 1, qkv);
  expect(requests, op, "requests", at::kInt, 1, qkv);
  expect(positions, op, "positions", at::kInt, 1, qkv);
  expect(slots, op, "slots", at::kInt, 1, qkv);
  const int64_t n = qkv.size(0);
  TORCH_CHECK(requests.size(0) == n && positions.size(0) == n && slots.size(0) == n, op, ": the plan must list ", n, " tokens, one for each row of qkv");
  TORCH_CHECK(starts.size(0) >= 1 && starts.size(0) - 1 <= kt.size(0), op, ": the plan has more requests than the cache has tails");
  TORCH_CHECK(n_heads >= 0 && n_heads + 2 * k.size(1) <= 65535, op, ": n_heads must be between 0 and 65535 with the KV heads");
  TORCH_CHECK(qkv.size(1) >= (n_heads + 2 * k.size(1)) * k.size(3), op, ": a row of qkv must hold ", n_heads, " + 2 x ", k.size(1), " heads of ", k.size(3));
  if (out) {
    expect_rows(*out, op, "out", qkv);
    TORCH_CHECK(out->size(0) == n && out->size(1) == (n_heads + k.size(1)) * k.size(3), op, ": out must be [", n, ", ", (n_heads + k.size(1)) * k.size(3), "]");
  }
}
void append(const Tensor& qkv, PLAN_ARGS, CONST_CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, const Tensor& out, bool zero_rest) {
  const char* op = "kv_append_8bit";
  expect_cache_aligned(op, k, v, kt, vt, cos, sin);
  expect_aligned(qkv, op, "qkv");
  expect_aligned(out, op, "out");
  ccl::KvAppend8Params p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.qkv_stride = qkv.size(0) > 1 ? qkv.stride(0) : 0;
  p.rotated = static_cast<__nv_bfloat16*>(out.data_ptr());
  p.rotated_stride = out.size(0) > 1 ? out.stride(0) : 0;
  p.starts = starts.data_ptr<int>();
  p.requests = requests.data_ptr<int>();
  p.positions = positions.data_ptr<int>();
  p.slots = slots.data_ptr<int>();
  p.cos = cos.data_ptr<float>();
  p.sin = sin.data_ptr<float>();
  p.rows = (int)qkv.size(0);
  p.n_requests = (int)starts.size(0) - 1;
  p.n_heads = (int)n_heads;
  p.table_rows = (int)cos.size(0);
  p.zero_rest = zero_rest;
  p.cache = cache_of(k, v, ks, vs, kt, vt);
  ok(ccl::kv_append8(p, stream()), op);
}
Tensor kv_append_8bit_cuda(const Tensor& qkv, PLAN_ARGS, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads) {
  check_append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, nullptr);
  c10::cuda::CUDAGuard g(qkv.device());
  Tensor out = fresh({qkv.size(0), (n_heads + k.size(1)) * k.size(3)}, at::kBFloat16, qkv);
  append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, out, true);
  return out;
}
Tensor kv_append_8bit_meta(const Tensor& qkv, PLAN_ARGS, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads) {
  check_append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, nullptr);
  return fresh({qkv.size(0), (n_heads + k.size(1)) * k.size(3)}, at::kBFloat16, qkv);
}
void kv_append_8bit_out_cuda(const Tensor& qkv, PLAN_ARGS, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, Tensor& out) {
  check_append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, &out);
  for (const Tensor* t : std::initializer_list<const Tensor*>{&qkv, &k, &v, &kt, &vt})
    TORCH_CHECK(!overlap(*t, out), "kv_append_8bit: out shares memory with qkv or the cache");
  c10::cuda::CUDAGuard g(qkv.device());
  append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, out, false);
}
void kv_append_8bit_out_meta(const Tensor& qkv, PLAN_ARGS, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, Tensor& out) {
  check_append(qkv, starts, requests, positions, slots, k, v, ks, vs, kt, vt, cos, sin, n_heads, &out);
}

void check_attention(const Tensor& qkv, const Tensor& positions, const Tensor& table, CONST_CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, const Tensor* out) {
  const char* op = "decode_attention_8bit";
  expect_rows(qkv, op, "qkv", qkv);
  check_cache(op, qkv, k, v, ks, vs, kt, vt, cos, sin);
  expect(positions, op, "positions", at::kInt, 1, qkv);
  expect(table, op, "table", at::kInt, 2, qkv);
  const int64_t n = qkv.size(0);
  TORCH_CHECK(n <= 65535, op, ": at most 65535 sequences, not ", n);
  TORCH_CHECK(positions.size(0) == n, op, ": positions must have one entry for each of the ", n, " rows of qkv");
  TORCH_CHECK(table.size(0) >= n && kt.size(0) >= n, op, ": the table and the tails must have a row for each of the ", n, " sequences");
  TORCH_CHECK(table.size(1) >= 1 && table.size(1) * k.size(2) <= 0x7fffffff, op, ": a table of ", table.size(1), " blocks is empty or too long");
  TORCH_CHECK(n_heads >= 1 && n_heads <= 65535 && n_heads % k.size(1) == 0, op, ": n_heads must be a multiple of the ", k.size(1), " KV heads, at most 65535");
  TORCH_CHECK(qkv.size(1) >= (n_heads + 2 * k.size(1)) * k.size(3), op, ": a row of qkv must hold ", n_heads, " + 2 x ", k.size(1), " heads of ", k.size(3));
  if (out) {
    expect_rows(*out, op, "out", qkv);
    TORCH_CHECK(out->size(0) == n && out->size(1) == n_heads * k.size(3), op, ": out must be [", n, ", ", n_heads * k.size(3), "]");
  }
}
void attention(const Tensor& qkv, const Tensor& positions, const Tensor& table, CONST_CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, const Tensor& out) {
  const char* op = "decode_attention_8bit";
  if (qkv.size(0) == 0) return;
  expect_cache_aligned(op, k, v, kt, vt, cos, sin);
  expect_aligned(qkv, op, "qkv");
  expect_aligned(out, op, "out");
  ccl::DecodeAttn8Params p;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.qkv_stride = qkv.size(0) > 1 ? qkv.stride(0) : 0;
  p.positions = positions.data_ptr<int>();
  p.table = table.data_ptr<int>();
  p.cos = cos.data_ptr<float>();
  p.sin = sin.data_ptr<float>();
  p.out = static_cast<__nv_bfloat16*>(out.data_ptr());
  p.out_stride = out.size(0) > 1 ? out.stride(0) : 0;
  p.batch = (int)qkv.size(0);
  p.n_heads = (int)n_heads;
  p.max_blocks = (int)table.size(1);
  p.table_rows = (int)cos.size(0);
  p.scale = 1.0f / std::sqrt((float)k.size(3));
  p.cache = cache_of(k, v, ks, vs, kt, vt);
  ccl::decode_attention8_split(p);
  p.partials = nullptr;
  Tensor partials;  // of this call alone: two calls, or two captured graphs, never share it
  if (const size_t n = ccl::decode_attention8_partial_floats(p)) {
    partials = fresh({(int64_t)n}, at::kFloat, qkv);
    p.partials = partials.data_ptr<float>();
  }
  ok(ccl::decode_attention8(p, stream()), op);
}
Tensor decode_attention_8bit_cuda(const Tensor& qkv, const Tensor& positions, const Tensor& table, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads) {
  check_attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, nullptr);
  c10::cuda::CUDAGuard g(qkv.device());
  Tensor out = fresh({qkv.size(0), n_heads * k.size(3)}, at::kBFloat16, qkv);
  attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, out);
  return out;
}
Tensor decode_attention_8bit_meta(const Tensor& qkv, const Tensor& positions, const Tensor& table, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads) {
  check_attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, nullptr);
  return fresh({qkv.size(0), n_heads * k.size(3)}, at::kBFloat16, qkv);
}
void decode_attention_8bit_out_cuda(const Tensor& qkv, const Tensor& positions, const Tensor& table, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, Tensor& out) {
  check_attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, &out);
  for (const Tensor* t : std::initializer_list<const Tensor*>{&qkv, &k, &v, &kt, &vt})
    TORCH_CHECK(!overlap(*t, out), "decode_attention_8bit: out shares memory with qkv or the cache");
  c10::cuda::CUDAGuard g(qkv.device());
  attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, out);
}
void decode_attention_8bit_out_meta(const Tensor& qkv, const Tensor& positions, const Tensor& table, CACHE_ARGS, const Tensor& cos, const Tensor& sin, int64_t n_heads, Tensor& out) {
  check_attention(qkv, positions, table, k, v, ks, vs, kt, vt, cos, sin, n_heads, &out);
}

// ---- log-probabilities ------------------------------------------------------------------------------------------------------------------------
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : (t.scalar_type() == at::kHalf ? 1 : 2); }
void check_logits(const char* op, const Tensor& logits, const Tensor& targets, int64_t top, int64_t base, int64_t total) {
  const auto t = logits.scalar_type();
  TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, op, ": logits must be bf16, fp16 or fp32, not ", t);
  TORCH_CHECK(logits.dim() == 2, op, ": logits must be [rows, vocabulary], not ", logits.dim(), "-dimensional");
  TORCH_CHECK(logits.size(1) >= 1, op, ": an empty vocabulary");
  TORCH_CHECK(logits.size(1) == 1 || logits.stride(1) == 1, op, ": the vocabulary's dimension must be contiguous");
  TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1), op, ": rows of logits must not overlap");
  expect(targets, op, "targets", at::kLong, 1, logits);
  TORCH_CHECK(targets.size(0) == logits.size(0), op, ": targets must have one id for each of the ", logits.size(0), " rows");
  TORCH_CHECK(top >= 0 && top <= ccl::kMaxTopLogprobs && top <= total, op, ": top must be between 0 and ", ccl::kMaxTopLogprobs, " and no larger than the vocabulary, not ", top);
  TORCH_CHECK(base >= 0 && total <= 0x7fffffff && base + logits.size(1) <= total, op, ": columns ", base, " to ", base + logits.size(1), " do not lie in a vocabulary of ", total);
  TORCH_CHECK(logits.size(0) <= 0x7ffffff, op, ": too many rows");
}
long long row_stride(const Tensor& logits) { return logits.size(0) > 1 ? logits.stride(0) : logits.size(1); }

using Logprobs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
Logprobs logprob_shapes(int64_t rows, int64_t top, const Tensor& like) {
  auto t = fresh_together<5>(like, {{{{rows}, at::kFloat}, {{rows}, at::kFloat}, {{rows, 2}, at::kFloat}, {{rows, top}, at::kFloat}, {{rows, top}, at::kLong}}});
  return {t[0], t[1], t[2], t[3], t[4]};
}
ccl::LogprobParams logprob_params(const Tensor& logits, const Tensor& targets, int64_t top, int64_t base, int64_t total) {
  ccl::LogprobParams p = {};
  p.logits = logits.data_ptr();
  p.stride = row_stride(logits);
  p.dtype = dtype_of(logits);
  p.rows = (int)logits.size(0);
  p.vocab = (int)logits.size(1);
  p.top = (int)top;
  p.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  p.vocab_base = base;
  p.vocab_total = total;
  return p;
}
Logprobs token_logprobs_cuda(const Tensor& logits, const Tensor& targets, int64_t top) {
  check_logits("token_logprobs", logits, targets, top, 0, logits.dim() == 2 ? logits.size(1) : 0);
  c10::cuda::CUDAGuard g(logits.device());
  Logprobs out = logprob_shapes(logits.size(0), top, logits);
  auto p = logprob_params(logits, targets, top, 0, logits.size(1));
  p.logprob = std::get<0>(out).data_ptr<float>();
  p.entropy = std::get<1>(out).data_ptr<float>();
  p.lse = std::get<2>(out).data_ptr<float>();
  p.top_logprobs = std::get<3>(out).data_ptr<float>();
  p.top_ids = reinterpret_cast<long long*>(std::get<4>(out).data_ptr<int64_t>());
  ok(ccl::token_logprobs(p, stream()), "token_logprobs");
  return out;
}
Logprobs token_logprobs_meta(const Tensor& logits, const Tensor& targets, int64_t top) {
  check_logits("token_logprobs", logits, targets, top, 0, logits.dim() == 2 ? logits.size(1) : 0);
  return logprob_shapes(logits.size(0), top, logits);
}
Tensor token_logprobs_shard_cuda(const Tensor& logits, const Tensor& targets, int64_t top, int64_t base, int64_t total) {
  check_logits("token_logprobs", logits, targets, top, base, total);
  c10::cuda::CUDAGuard g(logits.device());
  Tensor out = fresh({logits.size(0), 4 + 2 * top}, at::kFloat, logits);
  auto p = logprob_params(logits, targets, top, base, total);
  p.partial = out.data_ptr<float>();
  ok(ccl::token_logprobs(p, stream()), "token_logprobs");
  return out;
}
Tensor token_logprobs_shard_meta(const Tensor& logits, const Tensor& targets, int64_t top, int64_t base, int64_t total) {
  check_logits("token_logprobs", logits, targets, top, base, total);
  return fresh({logits.size(0), 4 + 2 * top}, at::kFloat, logits);
}
void check_merge(const Tensor& partials, const Tensor& targets, int64_t top, int64_t total) {
  const char* op = "token_logprobs_merge";
  expect(partials, op, "partials", at::kFloat, 3, partials);
  expect(targets, op, "targets", at::kLong, 1, partials);
  TORCH_CHECK(partials.size(0) >= 1 && partials.size(0) <= 64, op, ": 1 to 64 shards, not ", partials.size(0));
  TORCH_CHECK(top >= 0 && top <= ccl::kMaxTopLogprobs && top <= total, op, ": top must be between 0 and ", ccl::kMaxTopLogprobs, " and no larger than the vocabulary");
  TORCH_CHECK(partials.size(1) == targets.size(0) && partials.size(2) == 4 + 2 * top, op, ": partials must be [shards, rows, 4 + 2 * top]");
}
Logprobs token_logprobs_merge_cuda(const Tensor& partials, const Tensor& targets, int64_t top, int64_t total) {
  check_merge(partials, targets, top, total);
  c10::cuda::CUDAGuard g(partials.device());
  Logprobs out = logprob_shapes(partials.size(1), top, partials);
  ccl::LogprobMergeParams p;
  p.partials = partials.data_ptr<float>();
  p.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  p.vocab_total = total;
  p.shards = (int)partials.size(0);
  p.rows = (int)partials.size(1);
  p.top = (int)top;
  p.logprob = std::get<0>(out).data_ptr<float>();
  p.entropy = std::get<1>(out).data_ptr<float>();
  p.lse = std::get<2>(out).data_ptr<float>();
  p.top_logprobs = std::get<3>(out).data_ptr<float>();
  p.top_ids = reinterpret_cast<long long*>(std::get<4>(out).data_ptr<int64_t>());
  ok(ccl::token_logprobs_merge(p, stream()), "token_logprobs_merge");
  return out;
}
Logprobs token_logprobs_merge_meta(const Tensor& partials, const Tensor& targets, int64_t top, int64_t total) {
  check_merge(partials, targets, top, total);
  return logprob_shapes(partials.size(1), top, partials);
}

void check_backward(const Tensor& logits, const Tensor& targets, const Tensor& lse, const Tensor& entropy, const Tensor& top_ids, const optional<Tensor>& g_lp, const optional<Tensor>& g_ent,
                    const optional<Tensor>& g_top, int64_t base, int64_t total) {
  const char* op = "token_logprobs_backward";
  TORCH_CHECK(top_ids.dim() == 2, op, ": top_ids must be [rows, top]");
  check_logits(op, logits, targets, top_ids.size(1), base, total);
  const int64_t n = logits.size(0);
  expect(lse, op, "lse", at::kFloat, 2, logits);
  expect(entropy, op, "entropy", at::kFloat, 1, logits);
  expect(top_ids, op, "top_ids", at::kLong, 2, logits);
  TORCH_CHECK(lse.size(0) == n && lse.size(1) == 2 && entropy.size(0) == n && top_ids.size(0) == n, op, ": lse, entropy and top_ids must have ", n, " rows");
  if (g_lp) expect(*g_lp, op, "the gradient of logprob", at::kFloat, 1, logits);
  if (g_ent) expect(*g_ent, op, "the gradient of entropy", at::kFloat, 1, logits);
  if (g_top) expect(*g_top, op, "the gradient of top_logprobs", at::kFloat, 2, logits);
  TORCH_CHECK((!g_lp || g_lp->size(0) == n) && (!g_ent || g_ent->size(0) == n) && (!g_top || g_top->sizes() == top_ids.sizes()), op, ": gradients must have the results' sizes");
}
// A backward pass in a graph's capture, of a leaf that an eager graph still holds: the engine would let the default stream, where that one's
// gradients are accumulated, wait for the capturing one, which ends the capture and with it the process.
void refuse_held_leaf(const Tensor& logits) {
  if (!logits.requires_grad() || !logits.is_leaf() || c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(logits);
  const auto at = accumulator ? accumulator->stream() : c10::nullopt;
  TORCH_CHECK(!at || at->id() != 0, "token_logprobs: backward in a graph's capture while results of the same logits from the default stream are alive: delete those before");
}
Tensor token_logprobs_backward_cuda(const Tensor& logits, const Tensor& targets, const Tensor& lse, const Tensor& entropy, const Tensor& top_ids, const optional<Tensor>& g_lp,
                                    const optional<Tensor>& g_ent, const optional<Tensor>& g_top, int64_t base, int64_t total) {
  check_backward(logits, targets, lse, entropy, top_ids, g_lp, g_ent, g_top, base, total);
  c10::cuda::CUDAGuard g(logits.device());
  refuse_held_leaf(logits);
  const int64_t n = logits.size(0), vocab = logits.size(1), size = logits.element_size();
  // the gradient's rows lie as the logits' rows do relative to 16 bytes, so that one vector of the one is one of the other
  const int64_t per = 16 / size, shift = (int64_t)(reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16) / size;
  const int64_t stride = vocab + ((row_stride(logits) - vocab) % per + per) % per;
  Tensor whole = fresh({shift + n * stride}, logits.scalar_type(), logits);
  Tensor grad = whole.as_strided({n, vocab}, {stride, 1}, shift);
  ccl::LogprobBackwardParams p = {};
  p.logits = logits.data_ptr();
  p.stride = row_stride(logits);
  p.dtype = dtype_of(logits);
  p.rows = (int)n;
  p.vocab = (int)vocab;
  p.top = (int)top_ids.size(1);
  p.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  p.vocab_base = base;
  p.vocab_total = total;
  p.lse = lse.data_ptr<float>();
  p.entropy = entropy.data_ptr<float>();
  p.top_ids = reinterpret_cast<const long long*>(top_ids.data_ptr<int64_t>());
  p.g_logprob = g_lp ? g_lp->data_ptr<float>() : nullptr;
  p.g_entropy = g_ent ? g_ent->data_ptr<float>() : nullptr;
  p.g_top = g_top && p.top > 0 ? g_top->data_ptr<float>() : nullptr;
  p.grad = grad.data_ptr();
  p.grad_stride = stride;
  ok(ccl::token_logprobs_backward(p, stream()), "token_logprobs_backward");
  return grad;
}
Tensor token_logprobs_backward_meta(const Tensor& logits, const Tensor& targets, const Tensor& lse, const Tensor& entropy, const Tensor& top_ids, const optional<Tensor>& g_lp,
                                    const optional<Tensor>& g_ent, const optional<Tensor>& g_top, int64_t base, int64_t total) {
  check_backward(logits, targets, lse, entropy, top_ids, g_lp, g_ent, g_top, base, total);
  const int64_t vocab = logits.size(1), per = 16 / logits.element_size();
  return at::empty_strided({logits.size(0), vocab}, {vocab + ((row_stride(logits) - vocab) % per + per) % per, 1}, logits.options());
}

// The gradient of the whole-vocabulary form (a Python function does as much, for about 20 us more of the host's time a step).
class TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t top) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("ccl::token_logprobs", "").typed<Logprobs(const Tensor&, const Tensor&, int64_t)>();
    auto [logprob, entropy, lse, top_logprobs, top_ids] = op.call(logits, targets, top);
    ctx->save_for_backward({logits, targets, lse, entropy, top_ids});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({lse, top_ids});
    return {logprob, entropy, lse, top_logprobs, top_ids};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    auto given = [&](int i) { return grads[i].defined() ? optional<Tensor>(grads[i].contiguous()) : optional<Tensor>(); };
    const auto g_lp = given(0), g_ent = given(1), g_top = given(3);
    if (!g_lp && !g_ent && !g_top) return {Tensor(), Tensor(), Tensor()};
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("ccl::token_logprobs_backward", "")
                         .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, const optional<Tensor>&,
                                       const optional<Tensor>&, int64_t, int64_t)>();
    const auto s = ctx->get_saved_variables();
    return {op.call(s[0], s[1], s[2], s[3], s[4], g_lp, g_ent, g_top, 0, s[0].size(1)), Tensor(), Tensor()};
  }
};
Logprobs token_logprobs_autograd(const Tensor& logits, const Tensor& targets, int64_t top) {
  TORCH_CHECK(!logits._fw_grad(0).defined(), "token_logprobs: forward-mode derivatives are not implemented");  // (below autograd they would be dropped)
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto out = TokenLogprobs::apply(logits, targets, top);
    return {out[0], out[1], out[2], out[3], out[4]};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("ccl::token_logprobs", "").typed<Logprobs(const Tensor&, const Tensor&, int64_t)>();
  return op.call(logits, targets, top);
}

// No derivative goes through the 8-bit cache: one in forward mode is an error, and so is a backward pass that comes to a result. (torch's own kernel for
// that costs the host a microsecond more a call.)
void kv_autograd(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const std::string& name = op.schema().name();
  torch::autograd::edge_list edges;
  for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size())) {
    if (!v.isTensor()) continue;
    const Tensor& t = v.toTensor();
    TORCH_CHECK(!t._fw_grad(0).defined(), name, ": forward-mode derivatives are not implemented");
    if (t.requires_grad() && at::GradMode::is_enabled()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  }
  TORCH_CHECK(edges.empty() || !op.schema().returns().empty(), name, ": with out there are no derivatives, and an argument requires one");
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
  if (edges.empty()) return;
  Tensor out = stack->back().toTensor();
  torch::autograd::set_history(out, std::make_shared<torch::autograd::NotImplemented>(name, std::move(edges)));
}

}  // namespace

#define CACHE_SCHEMA "Tensor(a!) k, Tensor(b!) v, Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor(e!) k_tail, Tensor(f!) v_tail, Tensor cos, Tensor sin, int n_heads"
#define PLAN_SCHEMA "Tensor starts, Tensor requests, Tensor positions, Tensor slots"

TORCH_LIBRARY_FRAGMENT(ccl, m) {
  m.def("kv_plan(Tensor lengths, Tensor? new_tokens, Tensor(a!) table, Tensor(b!) held, Tensor(c!) free, Tensor(d!) state, int block_size, int max_tokens) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("kv_release(Tensor finished, Tensor(a!) table, Tensor(b!) held, Tensor(c!) free, Tensor(d!) state) -> ()");
  m.def("kv_append_8bit(Tensor qkv, " PLAN_SCHEMA ", " CACHE_SCHEMA ") -> Tensor");
  m.def("kv_append_8bit_out(Tensor qkv, " PLAN_SCHEMA ", " CACHE_SCHEMA ", Tensor(g!) out) -> ()");
  m.def("decode_attention_8bit(Tensor qkv, Tensor positions, Tensor table, " CACHE_SCHEMA ") -> Tensor");
  m.def("decode_attention_8bit_out(Tensor qkv, Tensor positions, Tensor table, " CACHE_SCHEMA ", Tensor(g!) out) -> ()");
  m.def("token_logprobs(Tensor logits, Tensor targets, int top) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("token_logprobs_shard(Tensor logits, Tensor targets, int top, int vocab_base, int vocab_total) -> Tensor");
  m.def("token_logprobs_merge(Tensor partials, Tensor targets, int top, int vocab_total) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("token_logprobs_backward(Tensor logits, Tensor targets, Tensor lse, Tensor entropy, Tensor top_ids, Tensor? g_logprob, Tensor? g_entropy, Tensor? g_top, int vocab_base, int vocab_total) -> Tensor");
}

TORCH_LIBRARY_IMPL(ccl, CUDA, m) {
  m.impl("kv_plan", &kv_plan_cuda);
  m.impl("kv_release", &kv_release_cuda);
  m.impl("kv_append_8bit", &kv_append_8bit_cuda);
  m.impl("kv_append_8bit_out", &kv_append_8bit_out_cuda);
  m.impl("decode_attention_8bit", &decode_attention_8bit_cuda);
  m.impl("decode_attention_8bit_out", &decode_attention_8bit_out_cuda);
  m.impl("token_logprobs", &token_logprobs_cuda);
  m.impl("token_logprobs_shard", &token_logprobs_shard_cuda);
  m.impl("token_logprobs_merge", &token_logprobs_merge_cuda);
  m.impl("token_logprobs_backward", &token_logprobs_backward_cuda);
}

TORCH_LIBRARY_IMPL(ccl, Meta, m) {
  m.impl("kv_plan", &kv_plan_meta);
  m.impl("kv_release", &kv_release_meta);
  m.impl("kv_append_8bit", &kv_append_8bit_meta);
  m.impl("kv_append_8bit_out", &kv_append_8bit_out_meta);
  m.impl("decode_attention_8bit", &decode_attention_8bit_meta);
  m.impl("decode_attention_8bit_out", &decode_attention_8bit_out_meta);
  m.impl("token_logprobs", &token_logprobs_meta);
  m.impl("token_logprobs_shard", &token_logprobs_shard_meta);
  m.impl("token_logprobs_merge", &token_logprobs_merge_meta);
  m.impl("token_logprobs_backward", &token_logprobs_backward_meta);
}

TORCH_LIBRARY_IMPL(ccl, Autograd, m) {
  m.impl("token_logprobs", &token_logprobs_autograd);
  // errors, not zeros: a second derivative, and any of the parts that a group's form is made of
  for (const char* op : {"token_logprobs_backward", "token_logprobs_shard", "token_logprobs_merge"}) m.impl(op, torch::autograd::autogradNotImplementedFallback());
  for (const char* op : {"kv_append_8bit", "kv_append_8bit_out", "decode_attention_8bit", "decode_attention_8bit_out"}) m.impl(op, torch::CppFunction::makeFromBoxedFunction<&kv_autograd>());
}
