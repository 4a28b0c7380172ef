// Host interface of the paged cache's bookkeeping on the GPU (no torch dependency).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ccl {

constexpr int kMaxPlanRequests = 16384;  // a request takes 12 bytes of shared memory

// The pool and who holds what of it. `free_blocks` is a stack: its first state[0] entries are the free pages.
struct KvBlocks {
  int* table;        // [requests, max_blocks]: pages of each request, in order; -1 behind them
  int* held;         // [requests] how many
  int* free_blocks;  // [capacity]
  int* state;        // {free pages, requests that the last plan could not serve}
  int requests, max_blocks, capacity;
};

// Gives every request r with new_tokens[r] > 0 (null: 1 each) and lengths[r] >= 0 the pages for lengths[r] + new_tokens[r] positions, and
// lists the new tokens, request after request: starts[r], and requests / positions / slots (page * block + place) of `room` entries, -1
// behind the last token. First come, first served: from the first request that the free pages do not suffice for, none gets pages; from
// the first whose tokens do not fit `room`, none is listed (room 0: nothing is listed and nothing counts as refused for it); one that
// needs more than max_blocks is passed over. state[1] counts requests with new tokens that were not served.
struct KvPlanParams {
  const int* lengths;
  const int* new_tokens;
  int* starts;       // [requests + 1]
  int* token_request;
  int* positions;
  int* slots;
  int room, block;
  KvBlocks b;
};
cudaError_t kv_plan(const KvPlanParams& p, cudaStream_t stream);

// Takes back the pages of the requests with finished[r] != 0; what was planned last comes back to where it was.
cudaError_t kv_release(const uint8_t* finished, const KvBlocks& b, cudaStream_t stream);

}  // namespace ccl
