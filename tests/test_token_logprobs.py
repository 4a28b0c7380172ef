"""Token log-probabilities, entropy, alternatives and their gradient against 64 bits.

Tolerances. A thread adds up to n = vocabulary / 512 (/ 128 in a small one) terms in fp32 and 10 levels of joins follow: (n + 40) 2^-24 relative
for the sum, 2^-20 for the exponentials (2^-22) and their arguments; the logarithm and the differences add 2^-23 of the logits' size. The
entropy's second sum weighs the terms by their distance from the maximum: 30 times that. A gradient is p times what it is multiplied
with, p off by (|log p| + 4) 2^-22, and is rounded once to the logits' type."""
import pytest
import torch

import oneccl_bindings_for_pytorch  # noqa: F401
from torch_ccl_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


def tol(vocab):
    return (vocab / 128 + 40) * 2.0**-24 + 2.0**-20 if vocab <= 4096 else (vocab / 512 + 40) * 2.0**-24 + 2.0**-20


def inputs(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g, device="cuda")


def order(x, top):
    """Ids of the best, equal ones by id, NaN first."""
    key = torch.where(torch.isnan(x), torch.full_like(x, INF), x)
    first = torch.argsort(-key, dim=-1, stable=True)
    nan_first = torch.argsort((~torch.isnan(x)).gather(1, first).to(torch.uint8), dim=-1, stable=True)
    return first.gather(1, nan_first)[:, :top]


def check(x, t, top):
    got = ops.token_logprobs(x, t, top)
    d = x.double()
    ref = torch.log_softmax(d, -1)
    e = tol(x.shape[1])
    size = d.abs().where(torch.isfinite(d), 0).amax(-1) + 20
    rows = torch.arange(x.shape[0], device="cuda")
    lp = ref[rows, t.clamp(0, x.shape[1] - 1)]
    lp = torch.where(t < 0, 0.0, torch.where(t >= x.shape[1], NAN, lp))
    plogp = torch.where(ref.exp() == 0, 0.0, ref.exp() * ref)
    ent = -plogp.sum(-1)

    def near(a, b, bound):
        b32 = b.float()
        same = (torch.isnan(a) & torch.isnan(b32)) | (a == b32)
        return bool((same | ((a.double() - b).abs() <= bound)).all())

    assert near(got.logprob, lp, e + size * 2.0**-22)
    assert near(got.entropy, ent, 30 * e + ent.abs().nan_to_num() * 2.0**-22)
    if top:
        ids = order(x, top)
        assert torch.equal(got.top_ids, ids)
        assert near(got.top_logprobs, ref.gather(1, ids), (e + size * 2.0**-22)[:, None])
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (4, 31), (3, 33), (100, 1024), (2, 2047), (7, 4095), (7, 4097), (3, 4104), (16, 32000), (33, 32003),
                                        (1, 128256), (2, 200001), (700, 5001)])
def test_values(rows, vocab, dtype):
    x, t = inputs(rows, vocab, dtype, rows + vocab)
    for top in {0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}:
        check(x, t, top)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_rows_at_any_offset(dtype, offset):
    for vocab, rows in ((1000, 9), (9001, 5)):
        x, t = inputs(rows, vocab + 13, dtype, offset)
        check(x[:, offset:offset + vocab], t.clamp(max=vocab - 1), 8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [40, 3000, 32003, 100003])
def test_masks_ties_and_what_is_not_finite(dtype, vocab):
    x, t = inputs(14, vocab, dtype, vocab)
    low = torch.finfo(dtype).min
    x[0, 5:] = -INF                     # five left
    x[1, 1:] = low
    x[2] = low                          # all masked with the lowest value: uniform
    x[3] = 1.0                          # all equal
    x[4] = -INF                         # nothing left: NaN, as log_softmax
    x[5, vocab // 2] = NAN
    x[6, vocab // 3] = INF
    x[7] = torch.round(x[7].float()).to(dtype)  # many ties
    x[8, ::2] = -INF
    x[9, : vocab // 2] = low
    x[10] = torch.finfo(dtype).max
    x[11] = 0.0
    x[11, 1::2] = -0.0                  # equal to 0
    x[12, 3:] = -INF
    x[12, :3] = low
    x[13, vocab - 3:] = 40.0
    t[0], t[1], t[8] = 2, vocab - 1, 1
    for top in (0, 1, 20, 32):
        check(x, t, top)


@pytest.mark.parametrize("dtype,mask", [(d, m) for d in (BF16, F32) for m in (-1e4, -1e9, -1e10, -1e20, -1e30, -2.0**100, -1e36, torch.finfo(d).min, -INF)] +
                         [(F16, m) for m in (-1e4, -65504.0, -INF)])
@pytest.mark.parametrize("rows,vocab", [(33, 32000), (33, 1000), (2, 128256)])
def test_masked_ranges_stay_in_the_pass_that_streams(rows, vocab, dtype, mask):
    """Threads that start on masked values, with any value that masks have. The reference that comes with the results is a whole power of two only
    if the row went through that pass; one that was done again, value by value, has one of its logits."""
    x, t = inputs(rows, vocab, dtype, 1)
    x[:, vocab // 8:] = mask
    x[:, : vocab // 16] = mask
    t = t % (vocab // 16) + vocab // 16
    check(x, t, 0)
    check(x, t, 5)
    reference = torch.ops.ccl.token_logprobs(x, t, 0)[2][:, 0].double() * 1.4426950408889634
    # (a few units, rounded to fp32: 2^-20)
    assert ((reference - reference.round()).abs() <= 2.0**-19).all()


def test_the_largest_vocabulary_value_by_value():
    """A row of 2^31 - 1 logits (4 GB) whose maximum is so large that it is done again: a step of that loop from its last element passes 2^31."""
    vocab = 2**31 - 1
    x = torch.zeros(1, vocab, dtype=BF16, device="cuda")
    x[0, vocab - 2] = 2.0**20
    got = ops.token_logprobs(x, torch.tensor([vocab - 2], device="cuda"), 2)
    assert got.logprob.item() == 0 and got.entropy.item() == 0
    assert got.top_ids.tolist() == [[vocab - 2, 0]] and got.top_logprobs.tolist() == [[0.0, -(2.0**20)]]


def test_targets_that_are_none():
    x, t = inputs(6, 5000, F32)
    t[1], t[3], t[4] = -1, -100, 5000
    got = check(x, t, 3)
    assert got.logprob[1] == 0 and got.logprob[3] == 0 and torch.isnan(got.logprob[4])
    none = ops.token_logprobs(x[:0], t[:0], 3)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 3)


def grad_ref(x, t, ids, g_lp, g_ent, g_top):
    d = x.double()
    lp = torch.log_softmax(d, -1)
    p = lp.exp()
    lp = torch.where(p == 0, 0.0, lp)
    ent = -(p * lp).sum(-1, keepdim=True)
    some = ((t >= 0) & (t < x.shape[1])).double()
    g_lp, g_ent = (torch.zeros(x.shape[0], device="cuda") if v is None else v for v in (g_lp, g_ent))
    g_lp = (g_lp.double() * some)[:, None]
    g_ent = g_ent.double()[:, None]
    whole = g_lp + (g_top.double().sum(-1, keepdim=True) if g_top is not None else 0)
    ref = -p * (whole + g_ent * (lp + ent))
    size = p * (whole.abs() + g_ent.abs() * (lp.abs() + ent)) * (lp.abs() + 4) * 2.0**-22 + p * g_ent.abs() * 30 * tol(x.shape[1])
    if g_lp.abs().sum() > 0:
        ref.scatter_add_(1, t.clamp(0, x.shape[1] - 1)[:, None], g_lp)
    if g_top is not None:
        ref.scatter_add_(1, ids, g_top.double())
        size = size + p * g_top.double().abs().sum(-1, keepdim=True) * 2.0**-20 + 2.0**-22 * g_top.double().abs().amax()
    return ref, size + p * (whole.abs() * 4) * tol(x.shape[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 5, 0), (100, 1024, 0), (9, 3001, 32), (5, 8193, 3), (4, 8199, 1), (3, 100003, 20), (33, 32000, 0)])
def test_gradient(rows, vocab, top, dtype):
    x, t = inputs(rows, vocab, dtype, rows + vocab)
    if rows > 4:
        t[2] = -1
        x[1, : vocab // 2] = -INF
    g = torch.Generator(device="cuda").manual_seed(1)
    grads = [torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, top, generator=g, device="cuda")]
    x.requires_grad_(True)
    got = ops.token_logprobs(x, t, top)
    for used in ((0, 1, 2), (0,), (1,), (2,)) if top else ((0, 1), (0,), (1,)):
        outs = [got.logprob, got.entropy] + ([got.top_logprobs] if top else [])
        d, = torch.autograd.grad([outs[i] for i in used], x, [grads[i] for i in used], retain_graph=True)
        xd = x.detach()
        some = [grads[i] if i in used else None for i in range(3)]
        xs = torch.where(torch.isinf(xd), torch.full_like(xd, torch.finfo(dtype).min), xd)
        ref, size = grad_ref(xs, t, got.top_ids, *some)
        assert d.dtype == dtype and d.shape == x.shape
        tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps if dtype == F16 else 2.0**-120
        bound = ref.abs() * torch.finfo(dtype).eps / 2 * 1.001 + size + tiny
        assert ((d.double() - ref).abs() <= bound).all(), float(((d.double() - ref).abs() / bound).max())


def test_gradient_against_differences():
    """Central differences of the 64-bit function: (f(x + h) - f(x - h)) / 2h is off by h^2 / 6 of the third derivative (below 1 here)."""
    x, t = inputs(2, 50, F32, 3, scale=1.0)
    x.requires_grad_(True)
    got = ops.token_logprobs(x, t, 2)
    f = got.logprob.sum() + 0.7 * got.entropy.sum() - 0.3 * got.top_logprobs.sum()
    d, = torch.autograd.grad(f, x)

    def value(z):
        lp = torch.log_softmax(z, -1)
        return lp.gather(1, t[:, None]).sum() - 0.7 * (lp.exp() * lp).sum() - 0.3 * lp.gather(1, got.top_ids).sum()

    h = 1e-4
    for r in range(2):
        for c in range(50):
            a, b = x.detach().double(), x.detach().double()
            a[r, c] += h
            b[r, c] -= h
            assert abs(float(value(a) - value(b)) / (2 * h) - float(d[r, c])) <= 1e-6


def test_gradient_of_broadcast_results_and_of_repeated_ids():
    x, t = inputs(6, 40, F32, 5)
    t[0] = int(x[0].argmax())  # also the best alternative
    x.requires_grad_(True)
    got = ops.token_logprobs(x, t, 4)
    (got.logprob.sum() + got.entropy.mean() + got.top_logprobs[:, 1].sum()).backward()  # expanded and partly empty gradients
    g_top = torch.zeros(6, 4, device="cuda")
    g_top[:, 1] = 1
    ref, size = grad_ref(x.detach(), t, got.top_ids, torch.ones(6, device="cuda"), torch.full((6,), 1 / 6, device="cuda"), g_top)
    assert ((x.grad.double() - ref).abs() <= ref.abs() * 2.0**-23 + size).all()
    x.grad = None
    ops.token_logprobs(x, t, 4).logprob.sum().backward()
    with torch.no_grad():
        assert not ops.token_logprobs(x, t).logprob.requires_grad


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 3), (4, 8), (3, 1)])
def test_gradient_of_strided_rows(dtype, offset, pad):
    for vocab in (333, 9001):
        base, t = inputs(5, offset + vocab + pad, dtype, vocab)
        t = t.clamp(max=vocab - 1)
        base.requires_grad_(True)
        got = ops.token_logprobs(base[:, offset:offset + vocab], t, 2)
        (got.logprob.sum() + got.entropy.sum()).backward()
        x = base.detach()[:, offset:offset + vocab]
        ref, size = grad_ref(x, t, got.top_ids, torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), None)
        d = base.grad[:, offset:offset + vocab].double()
        assert ((d - ref).abs() <= ref.abs() * torch.finfo(dtype).eps / 2 * 1.001 + size + 2.0**-120).all()
        assert (base.grad[:, :offset] == 0).all() and (base.grad[:, offset + vocab:] == 0).all()


@pytest.mark.parametrize("offset", [2.0**7, -(2.0**10), 2.0**14, -(2.0**17), 2.0**20, 2.0**23])
@pytest.mark.parametrize("vocab", [1000, 32003])
def test_a_common_offset_of_a_row_takes_nothing(vocab, offset):
    """Differences of fp32 logits are exact, wherever they lie: the bounds are those of the logits without the offset (of up to 20, and 2^-40 of the
    offset for the two parts that a base-2 reference is turned to natural units with)."""
    x, t = inputs(5, vocab, F32, vocab)
    x = (x + offset).requires_grad_(True)
    got = ops.token_logprobs(x, t, 4)
    ref = torch.log_softmax(x.detach().double(), -1)
    e, far = tol(vocab), abs(offset) * 2.0**-40
    lp = ref.gather(1, t[:, None])[:, 0]
    assert ((got.logprob.double() - lp).abs() <= e + 40 * 2.0**-22 + far).all()
    assert ((got.entropy.double() + (ref.exp() * ref).sum(-1)).abs() <= 31 * e).all()
    assert ((got.top_logprobs.double() - ref.gather(1, got.top_ids)).abs() <= e + 40 * 2.0**-22 + far).all()
    g = torch.randn(5, device="cuda"), torch.randn(5, device="cuda"), torch.randn(5, 4, device="cuda")
    d, = torch.autograd.grad([got.logprob, got.entropy, got.top_logprobs], x, g)
    want, size = grad_ref(x.detach(), t, got.top_ids, *g)
    p = ref.exp()
    assert ((d.double() - want).abs() <= want.abs() * 2.0**-23 + size + p * far * 100).all()
    # two shards of the vocabulary, joined
    half = vocab // 2
    if 2 * half == vocab:
        parts = torch.stack([torch.ops.ccl.token_logprobs_shard(x.detach()[:, i * half:(i + 1) * half], t, 4, i * half, vocab) for i in range(2)])
        joined = torch.ops.ccl.token_logprobs_merge(parts, t, 4, vocab)
        assert ((joined[0].double() - lp).abs() <= 2 * e + 40 * 2.0**-22 + far).all()


@pytest.mark.parametrize("shards,vocab,top", [(2, 500, 5), (4, 40, 32), (8, 4000, 20), (8, 3, 20), (2, 16001, 0), (64, 8, 32)])
def test_shards_of_a_vocabulary(shards, vocab, top):
    """The shards' results, joined, are the whole vocabulary's; so are their gradients."""
    rows, total = 9, shards * vocab
    x, t = inputs(rows, total, F32, shards)
    t[0], t[1], t[2] = 0, total - 1, -1
    x[3, : total // 2] = -INF
    x[4] = 2.0
    t[3] = total - 2
    pieces = [x[:, i * vocab:(i + 1) * vocab] for i in range(shards)]
    parts = torch.stack([torch.ops.ccl.token_logprobs_shard(p, t, top, i * vocab, total) for i, p in enumerate(pieces)])
    lp, ent, lse, top_lp, ids = torch.ops.ccl.token_logprobs_merge(parts, t, top, total)
    want = ops.token_logprobs(x, t, top)
    e = 2 * tol(total) + 40 * 2.0**-22
    assert ((lp - want.logprob).abs() <= e).all() and ((ent - want.entropy).abs() <= 30 * e).all()
    if top:
        # (row 3 may have fewer unmasked ids than alternatives: -inf on both sides)
        assert torch.equal(ids, want.top_ids) and ((top_lp == want.top_logprobs) | ((top_lp - want.top_logprobs).abs() <= e)).all()
    g = [torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda"), torch.randn(rows, top, device="cuda")]
    whole = torch.ops.ccl.token_logprobs_backward(x, t, lse, ent, ids, *g, 0, total)
    for i, p in enumerate(pieces):
        d = torch.ops.ccl.token_logprobs_backward(p, t, lse, ent, ids, *g, i * vocab, total)
        assert torch.equal(d, whole[:, i * vocab:(i + 1) * vocab])


def test_graph_other_stream_and_repeats():
    x, t = inputs(16, 32000, F32)
    want = ops.token_logprobs(x, t, 5)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(x, t, 5), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = ops.token_logprobs(x, t, 5)
    x2, t2 = inputs(16, 32000, F32, 9)
    x.copy_(x2)
    t.copy_(t2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, ops.token_logprobs(x2, t2, 5)))


def test_step_captured_with_its_gradient():
    """Forward and backward in one graph, warmed up on the capture's stream as torch asks."""
    x, t = inputs(64, 2000, BF16)
    x.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.token_logprobs(x, t)
        d, = torch.autograd.grad(got.logprob.sum() - got.entropy.sum(), x)
        want = d.clone()
        del got, d
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = ops.token_logprobs(x, t)
        d, = torch.autograd.grad(got.logprob.sum() - got.entropy.sum(), x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(d, want)


def test_a_captured_gradient_of_a_leaf_that_an_eager_graph_holds_is_refused():
    x, t = inputs(64, 2000, BF16)
    x.requires_grad_(True)
    held = ops.token_logprobs(x, t)  # on the default stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="delete those before"):
        with torch.cuda.graph(graph, stream=s):
            torch.autograd.grad(ops.token_logprobs(x, t).logprob.sum(), x)
    torch.cuda.synchronize()
    want, = torch.autograd.grad(held.logprob.sum(), x)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        d, = torch.autograd.grad(ops.token_logprobs(x, t).logprob.sum(), x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(d, want)


def test_group_of_one_rank():
    import torch.distributed as dist

    dist.init_process_group("ccl", store=dist.HashStore(), rank=0, world_size=1)
    try:
        x, t = inputs(5, 3000, BF16)
        x.requires_grad_(True)
        a, b = ops.token_logprobs(x, t, 6, group=dist.group.WORLD), ops.token_logprobs(x, t, 6)
        for p, q in zip(a, b):
            assert torch.equal(p, q) if p.dtype == torch.int64 else ((p - q).abs() <= 30 * tol(3000)).all()
        da, = torch.autograd.grad(a.logprob.sum(), x)
        db, = torch.autograd.grad(b.logprob.sum(), x)
        assert ((da.double() - db.double()).abs() <= db.double().abs() * 2.0**-7 + 2.0**-18).all()
    finally:
        dist.destroy_process_group()


def test_second_derivatives_are_refused():
    x, t = inputs(3, 40, F32)
    x.requires_grad_(True)
    d, = torch.autograd.grad(ops.token_logprobs(x, t).entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.square().sum(), x)
