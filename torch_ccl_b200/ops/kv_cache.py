"""A paged KV cache in 8 bits: who holds which page, prompt append, and single-token attention.

    blocks = KVBlocks.empty(requests=64, max_blocks=128, num_blocks=4096)       # one pool for all layers
    cache = KVCache8.empty(4096, n_kv_heads, block_size, head_dim, requests=64) # one per layer

    plan = kv_plan(lengths, new_tokens, blocks, block_size, max_tokens)         # prompts: pages and a slot for every token
    for each layer: rotated = kv_append_8bit(qkv, plan, cache, cos, sin, n_heads)
    ...
    kv_plan(positions, None, blocks, block_size)                                # one token each: a page where one is needed
    for each layer: out = decode_attention_8bit(qkv, positions, blocks.table, cache, cos, sin, n_heads)
    ...
    kv_release(finished, blocks)

`block_size` consecutive positions of one KV head share a page of 8-bit codes with one fp32 scale for K and one for V. The block that a
sequence is still filling is held in bf16, in its "tail", and is quantised once, when its last position arrives:
scale = max(amax / qmax, 2^-40) with qmax 448 (float8_e4m3fn) or 127 (int8), code = round(x / scale). Attention of position p reads the
blocks before p // block_size from their pages and the rest from the tail.

A sequence therefore goes on at its next position, or at one that its tail still has (a position of the block that it is filling, whose later
ones are then written again). It cannot go back to an earlier block: the tail holds another one by then. A page belongs to one request.
A request that a plan did not serve (`blocks.held[r] * block_size` says how many positions it has pages for) has to wait with its position until one
does: a block that fills up without a page is lost, and a page that is handed out for it later has what its last owner left there.

Row r of `lengths`, `blocks.table`, the tails and a decode step's qkv belong to the same request; to work on some of them pass slices of
all (`KVBlocks.rows`, `KVCache8.rows`). All calls run on the current stream of their tensors' device, allocate through torch's allocator
only and can be captured in a CUDA graph. No gradient goes through them: asking for one is an error. Two calls
that change the same pool, or append to the same rows, must be ordered by the caller.
"""
from typing import NamedTuple

import torch

_ops = torch.ops.ccl


class KVBlocks(NamedTuple):
    """The pages of a pool and who holds them; the same for every layer's cache."""

    table: torch.Tensor  # int32 [requests, max_blocks]: pages of each request in order, -1 behind them
    held: torch.Tensor   # int32 [requests]: how many
    free: torch.Tensor   # int32 [num_blocks]: a stack whose first state[0] entries are free pages
    state: torch.Tensor  # int32 [2]: {free pages, requests that the last kv_plan could not serve}

    @staticmethod
    def empty(requests, max_blocks, num_blocks, device="cuda"):
        i32 = dict(dtype=torch.int32, device=device)
        state = torch.zeros(2, **i32)
        state[0] = num_blocks
        # the lowest page is handed out first
        return KVBlocks(torch.full((requests, max_blocks), -1, **i32), torch.zeros(requests, **i32),
                        torch.arange(num_blocks - 1, -1, -1, **i32), state)

    def rows(self, first, last):
        """Requests first .. last - 1, over the same pool."""
        return KVBlocks(self.table[first:last], self.held[first:last], self.free, self.state)


class KVPlan(NamedTuple):
    """The new tokens of a `kv_plan`, request after request; -1 behind the last one."""

    starts: torch.Tensor     # int32 [requests + 1]: first token of each request
    requests: torch.Tensor   # int32 [max_tokens]
    positions: torch.Tensor  # int32 [max_tokens]
    slots: torch.Tensor      # int32 [max_tokens]: page * block_size + place in the page


class KVCache8(NamedTuple):
    """One layer's 8-bit pages, their scales, and the bf16 blocks that are still being filled."""

    k: torch.Tensor        # float8_e4m3fn or int8 [num_blocks, kv_heads, block_size, head_dim]
    v: torch.Tensor
    k_scale: torch.Tensor  # fp32 [num_blocks, kv_heads]
    v_scale: torch.Tensor
    k_tail: torch.Tensor   # bf16 [requests, kv_heads, block_size, head_dim]
    v_tail: torch.Tensor

    @staticmethod
    def empty(num_blocks, n_kv_heads, block_size, head_dim, requests, dtype=torch.float8_e4m3fn, device="cuda"):
        """block_size 16, 32, 64 or 128; head_dim 64 or 128; dtype float8_e4m3fn or int8."""
        page, tail = (num_blocks, n_kv_heads, block_size, head_dim), (requests, n_kv_heads, block_size, head_dim)
        codes = [torch.zeros(page, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
        scales = [torch.ones(num_blocks, n_kv_heads, device=device) for _ in range(2)]
        tails = [torch.zeros(tail, dtype=torch.bfloat16, device=device) for _ in range(2)]
        return KVCache8(*codes, *scales, *tails)

    def rows(self, first, last):
        """The tails of requests first .. last - 1, over the same pages."""
        return KVCache8(*self[:4], self.k_tail[first:last], self.v_tail[first:last])


def kv_plan(lengths, new_tokens, blocks, block_size, max_tokens=0):
    """Gives requests the pages that `new_tokens[r]` more positions after `lengths[r]` need (int32 [requests] each; new_tokens None: one
    more each) and lists the new tokens, up to `max_tokens` of them. A request with a negative length or no new tokens is passed over.
    What a request already holds counts, so that the same plan made twice takes nothing twice. First come, first served: from the first
    request that the free pages do not suffice for, none gets any; from the first whose tokens do not fit max_tokens (if that is not 0), none is listed;
    one that would pass the table's width gets nothing. `blocks.state[1]` says how many requests were not served. The arrays of a plan share
    one allocation."""
    return KVPlan(*_ops.kv_plan.default(lengths, new_tokens, *blocks, block_size, max_tokens))


def kv_release(finished, blocks):
    """Takes back the pages of the requests r with finished[r] (bool [requests])."""
    _ops.kv_release.default(finished, *blocks)


def kv_append_8bit(qkv, plan, cache, cos, sin, n_heads, out=None):
    """Rotary embedding and append of the rows of `qkv` (bf16 [tokens, (n_heads + 2 kv_heads) * head_dim]: q heads, k heads, v heads; one row
    for each entry of the plan). Returns [tokens, (n_heads + kv_heads) * head_dim]: q and k after the rotation. Rows without a token
    are zeros there; rows of `out`, if it is given, are left as they are. cos, sin: fp32 [positions, head_dim / 2]."""
    if out is None:
        return _ops.kv_append_8bit.default(qkv, *plan, *cache, cos, sin, n_heads)
    _ops.kv_append_8bit_out.default(qkv, *plan, *cache, cos, sin, n_heads, out)
    return out


def decode_attention_8bit(qkv, positions, table, cache, cos, sin, n_heads, out=None):
    """One new token per sequence: rotary embedding, append, attention over positions 0 .. positions[b]; returns bf16
    [batch, n_heads * head_dim]. n_heads may be any multiple of the KV heads. A position outside the table or the rotary tables (-1: no
    sequence in this row) gives a row of zeros and appends nothing; so does a row that reads a page number outside the pool, except
    that its token is appended. A page with an infinite or NaN scale, which is what a block with an infinity or a NaN is given, and scores that
    pass fp32, give NaN for the heads that read them. (A NaN among the codes of a page with a finite scale, which nothing here
    writes, is read as some number.)"""
    if out is None:
        return _ops.decode_attention_8bit.default(qkv, positions, table, *cache, cos, sin, n_heads)
    _ops.decode_attention_8bit_out.default(qkv, positions, table, *cache, cos, sin, n_heads, out)
    return out
