"""Log-probabilities of given tokens, entropy and the best alternatives, over a whole vocabulary or the shards of a group."""
from typing import NamedTuple, Optional

import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

_ops = torch.ops.ccl


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                 # fp32 [rows]
    entropy: torch.Tensor                 # fp32 [rows], in nats
    top_logprobs: Optional[torch.Tensor]  # fp32 [rows, top], best first
    top_ids: Optional[torch.Tensor]       # int64 [rows, top]


def _forward(logits, targets, top, group):
    """({logprob, entropy, lse, top_logprobs, top_ids}, first column's id, vocabulary) of the shards of a group"""
    world, rank = dist.get_world_size(group), dist.get_rank(group)
    base, total = rank * logits.shape[-1], world * logits.shape[-1]
    mine = _ops.token_logprobs_shard.default(logits, targets, top, base, total)
    every = mine.new_empty((world,) + mine.shape)
    if mine.numel():
        _ops.all_gather_copy_out.default(mine, list(every), group.group_name)
    return _ops.token_logprobs_merge.default(every, targets, top, total), base, total


class _ShardLogprobs(torch.autograd.Function):
    """Of a rank's shard; the whole vocabulary's gradient is registered with the op."""

    @staticmethod
    def forward(ctx, logits, targets, top, group):
        (logprob, entropy, lse, top_logprobs, top_ids), ctx.base, ctx.total = _forward(logits, targets, top, group)
        ctx.save_for_backward(logits, targets, lse, entropy, top_ids)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_ids)
        return logprob, entropy, top_logprobs, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None
        logits, targets, lse, entropy, top_ids = ctx.saved_tensors
        g = [None if t is None else t.contiguous() for t in (g_logprob, g_entropy, g_top)]
        return _ops.token_logprobs_backward.default(logits, targets, lse, entropy, top_ids, *g, ctx.base, ctx.total), None, None, None


def token_logprobs(logits, targets, top=0, group=None):
    """log softmax(logits)[row, targets[row]] and the entropy of every row, with the `top` (0 to 32) best ids and their log-probabilities:
    a `TokenLogprobs`, differentiable in the logits (bf16, fp16 or fp32 [rows, vocabulary]; rows may be strided) once and in reverse mode.

    targets: int64 [rows]; a negative one stands for "no token" (log-probability 0, no gradient from it), one past the vocabulary gives NaN.
    Equal logits are ordered by id; a NaN counts as larger than everything, as in torch.topk. Sums are in fp32. A gradient may
    be captured in a graph if no result of the same logits (where they are a leaf) from the default stream is alive; one that is, is an error.
    The results of a call share one allocation: what is kept for long, or saved, is best cloned.

    group: `logits` are this rank's equal shard of the vocabulary (rank 0 has the first ids); every rank passes the same targets, gets
    the whole vocabulary's results, and the gradient of its own shard. None: `logits` have the whole vocabulary."""
    if group is None:
        logprob, entropy, _, top_logprobs, top_ids = _ops.token_logprobs.default(logits, targets, top)
    elif torch.is_grad_enabled() and logits.requires_grad:
        logprob, entropy, top_logprobs, top_ids = _ShardLogprobs.apply(logits, targets, top, group)
    else:
        (logprob, entropy, _, top_logprobs, top_ids), _, _ = _forward(logits, targets, top, group)
    return TokenLogprobs(logprob, entropy, top_logprobs, top_ids) if top else TokenLogprobs(logprob, entropy, None, None)
