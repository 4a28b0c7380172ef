"""What the serving operators refuse (paged 8-bit KV cache, token log-probabilities), and the shapes they promise, on meta tensors: the same
checks run before a launch."""
import pytest
import torch

import oneccl_bindings_for_pytorch  # noqa: F401
from torch_ccl_b200 import ops

BF16 = torch.bfloat16


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def i32(*shape):
    return meta(*shape, dtype=torch.int32)


def make(requests=4, max_blocks=8, num_blocks=64, kv=2, block=16, dim=128, dtype=torch.float8_e4m3fn, heads=4, tokens=100):
    a = dict(blocks=ops.KVBlocks.empty(requests, max_blocks, num_blocks, "meta"),
             cache=ops.KVCache8(*[meta(num_blocks, kv, block, dim, dtype=dtype) for _ in range(2)], meta(num_blocks, kv), meta(num_blocks, kv),
                                *[meta(requests, kv, block, dim, dtype=BF16) for _ in range(2)]),
             cos=meta(max_blocks * block, dim // 2), sin=meta(max_blocks * block, dim // 2), heads=heads,
             plan=ops.KVPlan(i32(requests + 1), i32(tokens), i32(tokens), i32(tokens)),
             rows=meta(tokens, (heads + 2 * kv) * dim, dtype=BF16), qkv=meta(requests, (heads + 2 * kv) * dim, dtype=BF16), positions=i32(requests))
    return a


def append(a, **k):
    return ops.kv_append_8bit(a["rows"], a["plan"], a["cache"], a["cos"], a["sin"], a["heads"], **k)


def attend(a, **k):
    return ops.decode_attention_8bit(a["qkv"], a["positions"], a["blocks"].table, a["cache"], a["cos"], a["sin"], a["heads"], **k)


def test_schemas_are_registered():
    for name in ["kv_plan", "kv_release", "kv_append_8bit", "kv_append_8bit_out", "decode_attention_8bit", "decode_attention_8bit_out", "token_logprobs",
                 "token_logprobs_shard", "token_logprobs_merge", "token_logprobs_backward"]:
        for key in ("CUDA", "Meta"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key(f"ccl::{name}", key)
    assert "Tensor(a!) k" in str(torch.ops.ccl.decode_attention_8bit.default._schema)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_shapes(block, dim, dtype):
    a = make(block=block, dim=dim, dtype=dtype)
    p = ops.kv_plan(i32(4), i32(4), a["blocks"], block, 100)
    assert [t.shape[0] for t in p] == [5, 100, 100, 100] and all(t.dtype == torch.int32 for t in p)
    assert ops.kv_plan(i32(4), None, a["blocks"], block).slots.shape == (0,)
    assert ops.kv_release(meta(4, dtype=torch.bool), a["blocks"]) is None
    assert append(a).shape == (100, 6 * dim)
    assert attend(a).shape == (4, 4 * dim)
    out = meta(4, 4 * dim, dtype=BF16)
    assert attend(a, out=out) is out


def test_plan_refuses():
    b = ops.KVBlocks.empty(4, 8, 64, "meta")
    with pytest.raises(RuntimeError, match="lengths must be Int"):
        ops.kv_plan(meta(4, dtype=torch.int64), None, b, 16)
    with pytest.raises(RuntimeError, match="one entry for each request"):
        ops.kv_plan(i32(4), i32(3), b, 16)
    with pytest.raises(RuntimeError, match="one row for each of the 5"):
        ops.kv_plan(i32(5), None, b, 16)
    with pytest.raises(RuntimeError, match="block_size"):
        ops.kv_plan(i32(4), None, b, 48)
    with pytest.raises(RuntimeError, match="max_tokens"):
        ops.kv_plan(i32(4), None, b, 16, -1)
    with pytest.raises(RuntimeError, match="slots are 32-bit"):
        ops.kv_plan(i32(4), None, b._replace(free=i32(1 << 25)), 128)
    with pytest.raises(RuntimeError, match="at most 16384 requests"):
        ops.kv_plan(i32(16385), None, ops.KVBlocks.empty(16385, 8, 64, "meta"), 16)
    with pytest.raises(RuntimeError, match="state has two words"):
        ops.kv_plan(i32(4), None, b._replace(state=i32(1)), 16)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.kv_plan(i32(4), None, b._replace(table=i32(4, 16)[:, :8]), 16)
    with pytest.raises(RuntimeError, match="finished must be Bool"):
        ops.kv_release(i32(4), b)


def test_cache_refuses():
    for change, words in [(dict(block=8), "16, 32, 64 or 128"), (dict(block=48), "16, 32, 64 or 128"), (dict(dim=96), "head_dim must be 64 or 128"),
                          (dict(dim=256), "head_dim must be 64 or 128"), (dict(dtype=torch.float8_e5m2), "float8_e4m3fn or int8"), (dict(dtype=torch.uint8), "float8_e4m3fn or int8")]:
        a = make(**change)
        with pytest.raises(RuntimeError, match=words):
            attend(a)
        with pytest.raises(RuntimeError, match=words):
            append(a)
    a = make()
    for wrong in [a["cache"]._replace(v=meta(64, 2, 16, 64, dtype=torch.float8_e4m3fn)), a["cache"]._replace(k_scale=meta(64, 1)), a["cache"]._replace(v_tail=meta(3, 2, 16, 128, dtype=BF16)),
                  a["cache"]._replace(k_tail=meta(4, 2, 16, 128, dtype=torch.float16)), a["cache"]._replace(v=meta(64, 2, 16, 128, dtype=torch.int8))]:
        with pytest.raises(RuntimeError):
            attend(dict(a, cache=wrong))
        with pytest.raises(RuntimeError):
            append(dict(a, cache=wrong))


def test_a_pool_without_pages_is_refused():
    a = make(num_blocks=0)
    with pytest.raises(RuntimeError, match="a pool without pages"):
        attend(a)
    with pytest.raises(RuntimeError, match="a pool without pages"):
        append(a)


def test_append_refuses():
    a = make()
    with pytest.raises(RuntimeError, match="one for each row of qkv"):
        append(dict(a, plan=a["plan"]._replace(slots=i32(99))))
    with pytest.raises(RuntimeError, match="more requests than the cache has tails"):
        append(dict(a, plan=a["plan"]._replace(starts=i32(6))))
    with pytest.raises(RuntimeError, match="must hold 5"):
        append(dict(a, heads=5))
    with pytest.raises(RuntimeError, match="n_heads"):
        append(dict(a, heads=-1))
    with pytest.raises(RuntimeError, match="bf16"):
        append(dict(a, rows=meta(100, 8 * 128, dtype=torch.float16)))
    with pytest.raises(RuntimeError, match="row stride"):
        append(dict(a, rows=meta(100, 8 * 128 + 4, dtype=BF16)[:, :8 * 128]))
    with pytest.raises(RuntimeError, match="out must be"):
        append(a, out=meta(100, 6 * 128 + 8, dtype=BF16))


def test_attention_refuses():
    a = make()
    with pytest.raises(RuntimeError, match="multiple of the 2 KV heads"):
        attend(dict(a, heads=3))
    with pytest.raises(RuntimeError, match="positions must have one entry"):
        attend(dict(a, positions=i32(3)))
    with pytest.raises(RuntimeError, match="a row for each of the 5"):
        attend(dict(a, qkv=meta(5, 8 * 128, dtype=BF16), positions=i32(5)))
    with pytest.raises(RuntimeError, match="cos and sin"):
        attend(dict(a, cos=meta(128, 32)))
    with pytest.raises(RuntimeError, match="at most 65535 sequences"):
        attend(dict(make(requests=65536, max_blocks=1), cos=meta(16, 64), sin=meta(16, 64)))
    with pytest.raises(RuntimeError, match="out must be"):
        attend(a, out=meta(4, 3 * 128, dtype=BF16))


def test_logprobs():
    t = meta(5, dtype=torch.int64)
    for dtype in (BF16, torch.float16, torch.float32):
        got = ops.token_logprobs(meta(5, 1000, dtype=dtype), t, top=7)
        assert got.logprob.shape == got.entropy.shape == (5,) and got.top_ids.shape == got.top_logprobs.shape == (5, 7) and got.top_ids.dtype == torch.int64
    assert ops.token_logprobs(meta(5, 1000), t).top_ids is None
    x = meta(5, 1000).requires_grad_(True)
    got = ops.token_logprobs(x, t, top=3)
    g, = torch.autograd.grad(got.logprob.sum() + got.top_logprobs.sum(), x)
    assert g.shape == x.shape and not got.top_ids.requires_grad
    for logits, targets, top, words in [
            (meta(5, 1000, dtype=torch.float64), t, 0, "bf16, fp16 or fp32"), (meta(1000), t, 0, "rows, vocabulary"), (meta(5, 0), t, 0, "empty vocabulary"),
            (meta(1000, 5).t(), t, 0, "contiguous"), (meta(5, 1000), meta(4, dtype=torch.int64), 0, "one id for each"), (meta(5, 1000), i32(5), 0, "targets must be Long"),
            (meta(5, 1000), t, 33, "between 0 and 32"), (meta(5, 1000), t, -1, "between 0 and 32"), (meta(5, 20), t, 21, "no larger than the vocabulary"),
            (meta(1, 1000).expand(5, 1000), t, 0, "must not overlap")]:
        with pytest.raises(RuntimeError, match=words):
            ops.token_logprobs(logits, targets, top)
    shard = torch.ops.ccl.token_logprobs_shard(meta(5, 500), t, 4, 500, 1000)
    assert shard.shape == (5, 12)
    with pytest.raises(RuntimeError, match="do not lie in a vocabulary"):
        torch.ops.ccl.token_logprobs_shard(meta(5, 500), t, 4, 501, 1000)
    assert torch.ops.ccl.token_logprobs_merge(meta(2, 5, 12), t, 4, 1000)[0].shape == (5,)
    with pytest.raises(RuntimeError, match="4 \\+ 2 \\* top"):
        torch.ops.ccl.token_logprobs_merge(meta(2, 5, 13), t, 4, 1000)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_of_logprobs_are_refused(grad):
    """Of the whole vocabulary's form and of a group's parts; not a derivative of zero."""
    import torch.autograd.forward_ad as fw

    t = meta(5, dtype=torch.int64)
    calls = [lambda x: ops.token_logprobs(x, t, top=3).logprob, lambda x: torch.ops.ccl.token_logprobs_shard(x, t, 3, 0, 1000),
             lambda x: torch.ops.ccl.token_logprobs_merge(x.view(2, 250, 10), meta(250, dtype=torch.int64), 3, 1000)[0]]
    for call in calls:
        x = meta(5, 1000).requires_grad_(grad)
        with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            call(fw.make_dual(x, meta(5, 1000)))
        with torch.no_grad(), fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            call(fw.make_dual(x, meta(5, 1000)))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            torch.func.jvp(call, (meta(5, 1000),), (meta(5, 1000),))
        call(x)


def test_derivatives_of_a_groups_parts_are_refused():
    t = meta(5, dtype=torch.int64)
    part = torch.ops.ccl.token_logprobs_shard(meta(5, 500).requires_grad_(True), t, 3, 0, 1000)
    with pytest.raises(RuntimeError, match="not implemented"):
        part.sum().backward()
    lp = torch.ops.ccl.token_logprobs_merge(meta(2, 5, 10).requires_grad_(True), t, 3, 1000)[0]
    with pytest.raises(RuntimeError, match="not implemented"):
        lp.sum().backward()


@pytest.mark.parametrize("call,rows", [(append, "rows"), (attend, "qkv")])
def test_derivatives_through_the_cache_are_refused(call, rows):
    """In forward mode at the call, in reverse mode when a backward pass comes to the result; without a derivative nothing is in the way."""
    import torch.autograd.forward_ad as fw

    a = make()
    x = a[rows]
    width = 6 * 128 if call is append else 4 * 128
    out = meta(x.shape[0], width, dtype=BF16)
    with fw.dual_level():
        for k in ({}, {"out": out}):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dict(a, **{rows: fw.make_dual(x, meta(*x.shape, dtype=BF16))}), **k)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: call(dict(a, **{rows: x})), (x,), (meta(*x.shape, dtype=BF16),))
    wants = dict(a, **{rows: x.clone().requires_grad_(True)})
    result = call(wants)
    assert result.requires_grad
    with pytest.raises(RuntimeError, match="not implemented"):
        (result * 2).sum().backward()
    with pytest.raises(RuntimeError, match="an argument requires one"):
        call(wants, out=out)
    with torch.no_grad():
        assert call(wants, out=out) is out and not call(wants).requires_grad
    assert not call(a).requires_grad and call(a, out=out) is out


def test_cpu_tensors_are_refused():
    b = ops.KVBlocks.empty(4, 8, 64, "cpu")
    with pytest.raises(NotImplementedError):
        ops.kv_plan(torch.zeros(4, dtype=torch.int32), None, b, 16)
    with pytest.raises(NotImplementedError):
        ops.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
