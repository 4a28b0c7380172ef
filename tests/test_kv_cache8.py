"""The 8-bit paged cache against its definition in 64 bits: what is written (rotation, tails, codes, scales) and what attention makes of it.

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, to e4m3 by 2^-4 (or half the smallest step, 2^-10, of a scale), to int8
by half a scale; fp32 divisions and products in front of it add a few 2^-24. Attention: weights are rounded to f16 (2^-11 of each), scores and
sums are as good as fp32 (2^-15 of sum |w v| covers scores of up to 2^6 with a few 2^-22 each), the result is rounded to bf16."""
import pytest
import torch

import oneccl_bindings_for_pytorch  # noqa: F401
from torch_ccl_b200 import ops

pytestmark = pytest.mark.gpu
BF16, E4M3, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8
QMAX = {E4M3: 448.0, I8: 127.0}


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables(n, dim):
    inv = 1.0 / (10000.0 ** (torch.arange(0, dim, 2, device="cuda").float() / dim))
    ang = torch.arange(n, device="cuda").float()[:, None] * inv[None]
    return ang.cos().contiguous(), ang.sin().contiguous()


def rope64(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h].double(), x[..., h:].double()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def near_bf16(got, ref):
    """One rounding of `ref`, whose own products and sum were rounded to fp32 (terms are at most |ref| + cancelled parts: 1e-5 here)."""
    return bool(((got.double() - ref).abs() <= ref.abs() * 2.0**-8 + 1e-5).all())


def check_page(codes, scale, values, dtype):
    """One head's page [block, dim] holds the bf16 `values`."""
    x = values.double()
    want = max(float(x.abs().max()) / QMAX[dtype], 2.0**-40)
    assert abs(float(scale) - want) <= want * 2.0**-23
    y = codes.double() * float(scale)
    step = float(scale) / 2 if dtype == I8 else torch.maximum(x.abs() * 2.0**-4, torch.full_like(x, float(scale) * 2.0**-10))
    # the quotient x / scale is rounded to fp32 first: by 2^-24 of up to 127, 2^-17 of a step of int8, so that a value that close to the
    # middle between two codes may go to either: half a step and 2^-17 of one; of e4m3, 2^-24 of the value on top of its 2^-4
    slack = 2.0**-16 if dtype == I8 else 2.0**-20
    assert ((y - x).abs() <= step * (1 + slack) * (1 + 2.0**-40)).all()


class World:
    """Tables, cache and qkv of a batch whose cache is filled with random pages, stale numbers where nothing may be read."""

    def __init__(self, at, kv, group, block, dim, dtype, seed=0, spare=3):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.at, self.kv, self.group, self.block, self.dim, self.dtype = at, kv, group, block, dim, dtype
        B, self.heads = len(at), kv * group
        used = [max(p, 0) // block + 1 for p in at]
        M = max(used) + 1
        P = sum(used) + spare
        order = torch.randperm(P, generator=g, device="cuda").tolist()
        rows, k = [], 0
        for n in used:
            rows.append(order[k:k + n] + [-1] * (M - n))
            k += n
        self.table = i32(rows)
        self.cache = ops.KVCache8.empty(P, kv, block, dim, B, dtype)
        for pool, scale, tail in zip(self.cache[0:2], self.cache[2:4], self.cache[4:6]):
            if dtype == I8:
                pool.copy_(torch.randint(-127, 128, pool.shape, generator=g, device="cuda").to(I8))
            else:
                pool.copy_((torch.randn(pool.shape, generator=g, device="cuda") * 120).clamp(-448, 448).to(E4M3))
            scale.copy_((0.2 + torch.rand(scale.shape, generator=g, device="cuda")) * 3 / QMAX[dtype])
            tail.copy_(torch.randn(tail.shape, generator=g, device="cuda"))
            unused = order[k:]  # and the pages that are not full yet
            unused += [rows[b][n - 1] for b, n in enumerate(used)]
            scale[unused] = float("nan")
            for b, p in enumerate(at):
                tail[b, :, max(p, 0) % block:] = float("nan")
        self.positions = i32(at)
        self.qkv = torch.randn(B, (self.heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16)
        self.cos, self.sin = tables(M * block, dim)

    def reference(self, cache, b):
        """(new k, v, attention output, its sum |w v|, largest |v|) of row b in 64 bits, from the cache's contents before the call."""
        p, D, bs = self.at[b], self.dim, self.block
        x = self.qkv[b].view(-1, D)
        c, s = self.cos[p].double(), self.sin[p].double()
        q, kn, vn = rope64(x[:self.heads], c, s), rope64(x[self.heads:self.heads + self.kv], c, s), x[self.heads + self.kv:]
        full = self.table[b, :p // bs].long()

        def of(pool, scale, tail, new):
            paged = pool[full].double() * scale[full].double()[..., None, None]  # [n, kv, bs, D]
            return torch.cat([paged.transpose(0, 1).reshape(self.kv, -1, D), tail[b, :, :p % bs].double(), new.to(BF16).double()[:, None]], 1).repeat_interleave(self.group, 0)

        k, v = of(cache.k, cache.k_scale, cache.k_tail, kn.to(BF16)), of(cache.v, cache.v_scale, cache.v_tail, vn)
        w = torch.softmax(torch.einsum("hd,htd->ht", q, k) / D**0.5, -1)
        return kn, vn, torch.einsum("ht,htd->hd", w, v), torch.einsum("ht,htd->hd", w, v.abs()), v.abs().amax(1)

    def check(self, run):
        before = ops.KVCache8(*[t.clone() for t in self.cache])
        out = run(self).double().view(len(self.at), self.heads, self.dim)
        written = set()
        for b, p in enumerate(self.at):
            place = p % self.block
            if p < 0:
                assert (out[b] == 0).all()
                for t in (4, 5):
                    assert torch.equal(self.cache[t][b].view(torch.int16), before[t][b].view(torch.int16))
                continue
            kn, vn, ref, mag, vmax = self.reference(before, b)
            assert near_bf16(self.cache.k_tail[b, :, place], kn) and torch.equal(self.cache.v_tail[b, :, place], vn)
            for t in (4, 5):  # the rest of the tail is as it was
                rest = [i for i in range(self.block) if i != place]
                assert torch.equal(self.cache[t][b][:, rest].view(torch.int16), before[t][b][:, rest].view(torch.int16))
            bound = ref.abs() * 2.0**-8 + mag * (2.0**-11 + 2.0**-15) + vmax * 2.0**-20
            assert ((out[b] - ref).abs() <= bound).all(), (b, p, float(((out[b] - ref).abs() / bound).max()))
            if place == self.block - 1:
                page = int(self.table[b, p // self.block])
                written.add(page)
                for h in range(self.kv):
                    check_page(self.cache.k[page, h], self.cache.k_scale[page, h], self.cache.k_tail[b, h], self.dtype)
                    check_page(self.cache.v[page, h], self.cache.v_scale[page, h], self.cache.v_tail[b, h], self.dtype)
        others = [i for i in range(self.cache.k.shape[0]) if i not in written]
        for t in range(4):
            a, c = self.cache[t].view(torch.uint8 if t < 2 else torch.int32), before[t].view(torch.uint8 if t < 2 else torch.int32)
            assert torch.equal(a[others], c[others])


def attend(w, **k):
    return ops.decode_attention_8bit(w.qkv, w.positions, w.table, w.cache, w.cos, w.sin, w.heads, **k)


EDGES = [0, 1, 14, 15, 16, 17, 31, 32, 47, 63, 64, 65, 127, 128, 129, 255, 256, 300, -1]


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_around_every_border(block, dim, dtype):
    World(EDGES, 2, 3, block, dim, dtype, seed=block + dim).check(attend)


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("kv,group", [(1, 1), (3, 2), (2, 7), (1, 8), (2, 9), (1, 16), (1, 17), (2, 32), (1, 71)])
def test_attention_of_any_number_of_heads(kv, group, dtype):
    World([40, 0, 159, 511], kv, group, 16, 128, dtype, seed=group).check(attend)
    World([333, 64], kv, group, 32, 64, dtype, seed=group).check(attend)


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("at,block", [([4096], 16), ([5003], 64), ([8191, 3], 128), ([2047, 2048, 2049, 700, -1, 4500], 32)])
def test_attention_of_long_contexts_in_splits(at, block, dtype):
    """One sequence and one KV head: as many splits as there are, more than 32 units of 16 positions for a warp, ragged ones with fewer."""
    World(at, 1, 4, block, 128, dtype, seed=len(at)).check(attend)
    World(at, 1, 12, block, 64, dtype, seed=len(at)).check(attend)


def test_many_sequences_without_a_split():
    World([(i * 37) % 200 for i in range(700)], 4, 1, 16, 64, E4M3).check(attend)


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch", [74, 111, 148, 200])
def test_attention_in_ctas_of_every_size(batch, dim, dtype):
    """296, 444 and 592 pairs of a sequence and a KV head fill the GPU with CTAs of six, four and three warps; 800 do not fit at once."""
    g = torch.Generator().manual_seed(batch)
    at = EDGES + torch.randint(0, 500, (batch - len(EDGES),), generator=g).tolist()
    World(at, 4, 3, 32, dim, dtype, seed=batch).check(attend)


def test_rows_with_strides_and_a_given_result():
    w = World([100, 31, 5], 2, 4, 32, 128, E4M3)
    wide = torch.full((3, w.qkv.shape[1] + 24), float("nan"), device="cuda", dtype=BF16)
    wide[:, 8:-16] = w.qkv
    w.qkv = wide[:, 8:-16]
    room = torch.full((3, w.heads * 128 + 16), 7.0, device="cuda", dtype=BF16)

    def run(w):
        out = room[:, 8:-8]
        assert attend(w, out=out) is out
        assert (room[:, :8] == 7).all() and (room[:, -8:] == 7).all()
        return out.contiguous()

    w.check(run)
    with pytest.raises(RuntimeError, match="shares memory"):
        attend(w, out=wide[:, 8:8 + w.heads * 128])
    with pytest.raises(RuntimeError, match="multiple of 16 bytes"):
        attend(w, out=room[:, 4:-12])


def test_a_result_in_the_cache_is_refused():
    w = World([100, 31, 5], 2, 4, 32, 128, E4M3)
    plan = ops.kv_plan(i32([0, 0, 0]), i32([1, 1, 1]), ops.KVBlocks.empty(3, 4, w.cache.k.shape[0]), 32, 3)
    for tail in w.cache[4:]:
        rows = tail.view(3, -1)
        with pytest.raises(RuntimeError, match="shares memory"):
            attend(w, out=rows[:, :w.heads * 128])
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.kv_append_8bit(w.qkv, plan, w.cache, w.cos, w.sin, w.heads, out=rows[:, :(w.heads + 2) * 128])


def test_scales_of_every_size():
    """Pages whose V scales differ by 2^40: weights are kept relative to what they contribute."""
    w = World([321, 95], 2, 4, 16, 128, I8)
    for b in range(2):
        for i in range(w.at[b] // 16):
            page = int(w.table[b, i])
            w.cache.v_scale[page] = 2.0 ** (-30 + (i * 7) % 40)
            w.cache.k_scale[page] *= 2.0 ** ((i * 5) % 7 - 5)
    w.check(attend)


def test_large_and_small_queries():
    w = World([200, 77, 16, 31], 1, 4, 16, 128, E4M3)
    for b, f in enumerate([2.0**-60, 30.0, 0.0, 2.0**100]):
        w.qkv[b, :w.heads * 128] *= f
    before = ops.KVCache8(*[t.clone() for t in w.cache])
    out = attend(w).double().view(4, w.heads, 128)
    for b in range(3):  # scores of some hundred: their fp32 roundings are 2^-16 of a weight's logarithm
        _, _, ref, mag, vmax = w.reference(before, b)
        assert ((out[b] - ref).abs() <= ref.abs() * 2.0**-8 + mag * (2.0**-11 + 2.0**-12) + vmax * 2.0**-20).all()
    # scores of 2^100: all the weight on the largest one
    x = w.qkv[3].view(-1, 128)
    q = rope64(x[:4], w.cos[31].double(), w.sin[31].double())
    k = torch.cat([before.k[int(w.table[3, 0]), 0].double() * float(before.k_scale[int(w.table[3, 0]), 0]), w.cache.k_tail[3, 0].double()])
    v = torch.cat([before.v[int(w.table[3, 0]), 0].double() * float(before.v_scale[int(w.table[3, 0]), 0]), w.cache.v_tail[3, 0].double()])
    best = v[(q @ k.T).argmax(-1)]
    assert ((out[3] - best).abs() <= best.abs() * 2.0**-8 + best.abs() * 2.0**-11 + 1e-6).all()


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("dim", [64, 128])
def test_queries_down_to_the_smallest(dim, dtype):
    """Rows whose largest element is anywhere between 2^-100 and the smallest bf16 number: all positions weigh the same."""
    exponents = list(range(-100, -136, -1))
    w = World([40 + i for i in range(len(exponents))], 1, 4, 16, dim, dtype)
    for b, e in enumerate(exponents):
        w.qkv[b, :4 * dim] *= 2.0**e
    w.check(attend)


def test_nan_and_infinity_stay_where_they_are():
    """A page with a NaN spoils its own sequence and KV head, in whatever way, and no other."""
    w = World([100, 100, 100], 2, 2, 16, 128, E4M3)
    clean = World([100, 100, 100], 2, 2, 16, 128, E4M3)
    want = attend(clean).view(3, 2, 2, 128)
    w.cache.k_scale[int(w.table[1, 2]), 0] = float("nan")
    w.cache.v_tail[2, 1, 1, 5] = float("inf")
    out = attend(w).view(3, 2, 2, 128)
    assert torch.isnan(out[1, 0]).all()
    assert torch.isinf(out[2, 1, :, 5]).all()
    for b, h in ((0, 0), (0, 1), (1, 1), (2, 0)):
        assert torch.equal(out[b, h], want[b, h])
    assert torch.equal(out[2, 1, :, :5], want[2, 1, :, :5]) and torch.equal(out[2, 1, :, 6:], want[2, 1, :, 6:])


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("at", [100, 3000, 20000])
def test_what_is_not_finite_is_not_a_number_in_every_split(at, dtype):
    """A page with an infinity has an infinite scale, and 0 * inf in every position: NaN, in one split, a cluster's, or more. So have scores that
    pass fp32. Not the zeros of a page outside the pool."""
    for change in ("k", "v", "score"):
        w = World([at, 40, at], 1, 4, 16, 128, dtype)
        clean = World([at, 40, at], 1, 4, 16, 128, dtype)
        want = attend(clean)
        if change == "score":
            w.qkv[2, :5 * 128] = 2.0**70  # q and the new k: their product is 2^147
        else:
            scale = w.cache.k_scale if change == "k" else w.cache.v_scale
            scale[int(w.table[2, 3])] = float("inf")
        out = attend(w)
        assert torch.isnan(out[2]).all(), change
        assert torch.equal(out[:2], want[:2])


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("at", [100, 3000, 20000])
def test_scores_below_fp32_are_not_a_number_either(at, dtype):
    """Whatever other positions the warp that reads them has: pages of one block, of four and of eight with scores of -2^147."""
    for pages in (1, 4, 8):
        w = World([at, 40], 1, 4, 16, 128, dtype)
        w.cos.fill_(1)
        w.sin.zero_()
        w.qkv[0, :4 * 128] = 2.0**70
        w.qkv[0, 4 * 128:5 * 128] = 0
        w.cache.k_tail[0] = 0
        w.cache.k_scale[w.table[0, :at // 16].long()] = 2.0**-80
        low = w.table[0, :min(pages, at // 16)].long()
        w.cache.k.view(torch.uint8)[low] = torch.full((), -1.0, device="cuda").to(dtype).view(torch.uint8)
        w.cache.k_scale[low] = 2.0**70
        out = attend(w)
        assert torch.isnan(out[0]).all() and not torch.isnan(out[1]).any()


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_an_infinity_in_a_block_that_fills_up(dtype):
    """In the tail it is the new token's own; once the block is a page, everything that reads it is NaN."""
    for part in (0, 1):
        w = World([31, 30], 1, 2, 16, 128, dtype)
        w.cache[4 + part][0, 0, 3, 7] = float("inf")
        attend(w)
        assert torch.isinf(w.cache[2 + part][int(w.table[0, 1]), 0])
        w.at, w.positions = [32, 31], i32([32, 31])
        out = attend(w)
        assert torch.isnan(out[0]).all() and not torch.isnan(out[1]).any()


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_nan_or_an_infinity_spoils_its_page(value, dtype):
    """Whoever quantises it gives it a scale that is not finite, and the heads that read it, and no others, are NaN."""
    for part in (0, 1):
        w = World([31, 31], 2, 2, 16, 128, dtype)  # a token fills the block
        w.cache[4 + part][0, 1, 3, 7] = value
        attend(w)
        w.at, w.positions = [32, 32], i32([32, 32])
        out = attend(w).view(2, 4, 128)
        assert not torch.isfinite(w.cache[2 + part][int(w.table[0, 1]), 1])
        assert torch.isnan(out[0, 2:]).all() and not torch.isnan(out[0, :2]).any() and not torch.isnan(out[1]).any()
        blocks, cache = ops.KVBlocks.empty(2, 3, 6), ops.KVCache8.empty(6, 2, 16, 128, 2, dtype)  # a prompt does
        qkv = torch.randn(64, 8 * 128, generator=w.g, device="cuda").to(BF16)
        qkv[19, (4 + 2 * part + 1) * 128 + 70] = value  # position 19 of the first request, the second KV head
        plan = ops.kv_plan(i32([0, 0]), i32([32, 32]), blocks, 16, 64)
        ops.kv_append_8bit(qkv, plan, cache, w.cos, w.sin, 4)
        assert [bool(torch.isfinite(cache[2 + part][p, h])) for p in blocks.table[0, :2].tolist() for h in range(2)] == [True, True, True, False]
        ops.kv_plan(w.positions, None, blocks, 16)
        out = ops.decode_attention_8bit(w.qkv, w.positions, blocks.table, cache, w.cos, w.sin, 4).view(2, 4, 128)
        assert torch.isnan(out[0, 2:]).all() and not torch.isnan(out[0, :2]).any() and not torch.isnan(out[1]).any()


def test_pages_outside_the_pool():
    """Rows of zeros for a sequence with such a page, in the same split or another, and its token is still appended."""
    at = [100, 100, 3000, 15]
    w = World(at, 1, 4, 16, 128, E4M3)
    clean = World(at, 1, 4, 16, 128, E4M3)
    want = attend(clean)
    w.table[1, 3] = w.cache.k.shape[0]
    w.table[2, 1] = -7
    w.table[3, 0] = 1 << 30  # the page that its full block would go to
    out = attend(w)
    assert (out[1] == 0).all() and (out[2] == 0).all()
    assert torch.equal(out[0], want[0]) and torch.equal(out[3], want[3])
    for t in (4, 5):
        assert torch.equal(w.cache[t].view(torch.int16), clean.cache[t].view(torch.int16))


def test_positions_outside_the_tables():
    w = World([40, 40, 40, 40], 1, 2, 16, 128, E4M3)
    w.positions.copy_(i32([40, w.table.shape[1] * 16, -5, 2**31 - 1]))
    before = [t.clone() for t in w.cache]
    out = attend(w)
    assert (out[1:] == 0).all() and (out[0] != 0).any()
    w.cos, w.sin = w.cos[:40].contiguous(), w.sin[:40].contiguous()  # position 40 has no angle
    assert (attend(w) == 0).all()
    for t in (4, 5):
        assert torch.equal(w.cache[t][1:].view(torch.int16), before[t][1:].view(torch.int16))
    for t in (0, 1):
        assert torch.equal(w.cache[t].view(torch.uint8), before[t].view(torch.uint8))


def test_offsets_past_32_bits():
    """Pages near the end of pools of 6 GB each."""
    P = (6 << 30) // (128 * 128)
    w = World([300, 127, 1000], 1, 4, 128, 128, I8)
    big = ops.KVCache8(*[torch.empty(P, 1, 128, 128, dtype=I8, device="cuda") for _ in range(2)], *[torch.full((P, 1), float("nan"), device="cuda") for _ in range(2)], *w.cache[4:])
    shift = P - w.cache.k.shape[0]
    for t in range(4):
        big[t][shift:] = w.cache[t]
    out = ops.decode_attention_8bit(w.qkv, w.positions, torch.where(w.table >= 0, w.table + shift, -1), big, w.cos, w.sin, w.heads)
    small = ops.KVCache8(*w.cache[:4], w.cache.k_tail.clone(), w.cache.v_tail.clone())
    assert torch.equal(out, ops.decode_attention_8bit(w.qkv, w.positions, w.table, small, w.cos, w.sin, w.heads))
    for t in range(4):
        assert torch.equal(big[t][shift:].view(torch.uint8), small[t].view(torch.uint8))


# ---- append ------------------------------------------------------------------------------------------------------------------------

def admitted(before, new, block, blocks, room=None):
    """A plan for requests that hold `before` tokens already."""
    if any(before):
        ops.kv_plan(i32([0] * len(before)), i32(before), blocks, block, 0)
    return ops.kv_plan(i32(before), i32(new), blocks, block, sum(new) if room is None else room)


def check_append(before, new, kv, heads, block, dim, dtype, room=None, given=False, seed=0, zero=()):
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, N = len(before), sum(new)
    room = N if room is None else room
    width = max(-(-(b + t) // block) for b, t in zip(before, new)) + 1
    blocks = ops.KVBlocks.empty(R, width, R * width + 5)
    cache = ops.KVCache8.empty(R * width + 5, kv, block, dim, R, dtype)
    for t in (4, 5):
        cache[t].copy_(torch.randn(cache[t].shape, generator=g, device="cuda"))
    old = [t.clone() for t in cache]
    plan = admitted(before, new, block, blocks, room)
    cos, sin = tables(width * block, dim)
    qkv = torch.randn(room, (heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16)
    for r in zero:  # a request of zeros
        qkv[int(plan.starts[r]):int(plan.starts[r + 1])] = 0
        cache.k_tail[r] = cache.v_tail[r] = old[4][r] = old[5][r] = 0
    wide = torch.full((room, (heads + kv) * dim + 8), 7.0, device="cuda", dtype=BF16)
    out = ops.kv_append_8bit(qkv, plan, cache, cos, sin, heads, **({"out": wide[:, :-8]} if given else {}))
    rows = qkv.view(room, -1, dim)
    live = plan.positions[:N].long()
    turned = rope64(rows[:N, :heads + kv], cos[live].double()[:, None], sin[live].double()[:, None])
    assert near_bf16(out[:N].reshape(N, -1, dim), turned)
    assert (out[N:] == (7 if given else 0)).all() and (wide[:, -8:] == 7).all()
    keys, values = out[:N].reshape(N, -1, dim)[:, heads:], rows[:N, heads + kv:]
    table, pages = blocks.table.tolist(), set()
    for r in range(R):
        a, e, n = int(plan.starts[r]), int(plan.starts[r + 1]), before[r]
        for pool, scale, tail, was, x in ((cache.k, cache.k_scale, cache.k_tail, old[4], keys), (cache.v, cache.v_scale, cache.v_tail, old[5], values)):
            line = torch.cat([was[r, :, :n % block].transpose(0, 1), x[a:e]])  # from the first touched block on
            for i in range(line.shape[0] // block):
                page = table[r][n // block + i]
                pages.add(page)
                for h in range(kv):
                    check_page(pool[page, h], scale[page, h], line[i * block:(i + 1) * block, h], dtype)
            left = line[line.shape[0] // block * block:].transpose(0, 1)
            want = was[r].clone()
            if e > a:
                want[:, :left.shape[1]] = left
            assert torch.equal(tail[r], want), r
    others = [i for i in range(cache.k.shape[0]) if i not in pages]
    for t in range(4):
        assert torch.equal(cache[t][others].float(), old[t][others].float())


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_around_every_border(block, dim, dtype):
    check_append([0] * 8, [1, block - 1, block, block + 1, 0, 2 * block, 3 * block + 5, 7], 3, 5, block, dim, dtype, seed=block)


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("block", [16, 64, 128])
def test_append_in_the_middle_of_a_block(block, dtype):
    """The old part of the tail joins the first block while the last one goes to the tail."""
    before = [5, block - 1, block, block + 3, 2 * block - 1, 3, 9, 1, block // 2]
    new = [1, 1, 1, block - 3, block + 1, 2 * block, 5 * block + 2, 4 * block - 1, 0]
    check_append(before, new, 2, 3, block, 128, dtype, seed=block)
    check_append(before, new, 5, 0, block, 64, dtype, seed=block)


@pytest.mark.parametrize("given", [False, True])
def test_append_rows_behind_the_last_token(given):
    check_append([0, 3], [40, 21], 2, 4, 16, 128, E4M3, room=200, given=given)


def test_append_of_zeros_and_of_many():
    check_append([0, 0, 0], [50, 40, 16], 1, 1, 16, 128, I8, zero=(1,))
    check_append([0] * 100, [(i * 13) % 70 for i in range(100)], 1, 2, 16, 64, E4M3)
    check_append([3, 0], [1500, 1024], 8, 32, 32, 128, E4M3)


def test_append_skips_what_is_outside():
    """Requests, positions, slots and starts that make no sense: the rows are skipped, the pages not written; the others are as they are alone."""
    cos, sin = tables(64, 128)
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(48, 3 * 128, generator=g, device="cuda").to(BF16)

    def go(requests, positions, slots, starts):
        cache = ops.KVCache8.empty(4, 1, 16, 128, 2)
        out = ops.kv_append_8bit(qkv, ops.KVPlan(i32(starts), i32(requests), i32(positions), i32(slots)), cache, cos, sin, 1)
        return [out] + [t.float() for t in cache]

    pos = list(range(24)) * 2
    good = go([0] * 24 + [1] * 24, pos, list(range(48)), [0, 24, 48])
    for requests, positions, slots, starts in [
            ([0] * 24 + [9] * 24, pos, list(range(48)), [0, 24, 48]), ([0] * 24 + [-3] * 24, pos, list(range(48)), [0, 24, 48]),
            ([0] * 24 + [1] * 24, pos[:24] + [64] * 24, list(range(48)), [0, 24, 48]), ([0] * 24 + [1] * 24, pos[:24] + [2**31 - 1] * 24, list(range(48)), [0, 24, 48])]:
        got = go(requests, positions, slots, starts)
        assert torch.equal(got[0][:24], good[0][:24]) and (got[0][24:] == 0).all()
        for a, b in zip(got[5:], good[5:]):
            assert torch.equal(a[0], b[0]) and (a[1] == 0).all()
    for slots in ([0] * 24 + [64] * 24, [0] * 24 + [-1] * 24, [0] * 24 + [2**31 - 1] * 24):
        got = go([0] * 24 + [1] * 24, pos, slots, [0, 24, 48])
        assert torch.equal(got[0], good[0]) and torch.equal(got[5], good[5]) and (got[1][1:] == 0).all()
    go([0] * 24 + [1] * 24, pos, list(range(48)), [1000, -5, 2**31 - 1])
    torch.cuda.synchronize()


@pytest.mark.parametrize("end", [-2**31, -2**31 + 1, -6, 0, 1, 2**31 - 1])
@pytest.mark.parametrize("first", [3, 15])
def test_append_where_a_request_ends_in_front_of_its_rows(first, end):
    """Nothing is read or written in front of or behind the rows, and another request's are as they are alone."""
    g = torch.Generator(device="cuda").manual_seed(0)
    cos, sin = tables(64, 128)
    qkv = torch.randn(48, 3 * 128, generator=g, device="cuda").to(BF16)

    def go(starts):
        cache = ops.KVCache8.empty(8, 1, 16, 128, 2)
        wide = torch.full((148, 2 * 128), 7.0, device="cuda", dtype=BF16)
        # request 1 has the first 32 rows, request 0 the last 16, so that starts[1] is the end of the one and the beginning of the other
        plan = ops.KVPlan(i32(starts), i32([1] * 32 + [0] * 16), i32(list(range(32)) + [first + i for i in range(16)]), i32(list(range(32)) + [64 + first + i for i in range(16)]))
        ops.kv_append_8bit(qkv, plan, cache, cos, sin, 1, out=wide[50:98])
        assert (wide[:50] == 7).all() and (wide[98:] == 7).all()
        return wide[50:82], [t.float() for t in cache]

    out, cache = go([32, end, 32])
    want, want_cache = go([32, 48, 32])
    assert torch.equal(out, want)
    for a, b in zip(cache[:4], want_cache[:4]):
        assert torch.equal(a[:2], b[:2])
    for a, b in zip(cache[4:], want_cache[4:]):
        assert torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("before", [0, 5, 16, 19])
@pytest.mark.parametrize("angles", [24, 33, 40, 47, 48, 49, 63, 64])
def test_append_up_to_the_end_of_the_rotary_tables(angles, before, dtype):
    """Rows with an angle are what they are in a prompt that ends there, those without one are left alone, wherever the request and the tables end."""
    end, block, kv, heads, dim = 64, 16, 3, 2, 128
    g = torch.Generator(device="cuda").manual_seed(angles + before)
    qkv = torch.randn(end - before, (heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16)
    old = torch.randn(2, 1, kv, block, dim, generator=g, device="cuda").to(BF16)
    cos, sin = tables(end, dim)

    def go(rows, angles):
        blocks, cache = ops.KVBlocks.empty(1, 5, 9), ops.KVCache8.empty(9, kv, block, dim, 1, dtype)
        cache.k_tail.copy_(old[0])
        cache.v_tail.copy_(old[1])
        admitted([before], [end - before], block, blocks)  # the same pages for both
        plan = ops.kv_plan(i32([before]), i32([rows]), blocks, block, rows)
        out = torch.full((rows, (heads + kv) * dim), 7.0, device="cuda", dtype=BF16)
        ops.kv_append_8bit(qkv[:rows], plan, cache, cos[:angles].contiguous(), sin[:angles].contiguous(), heads, out=out)
        return out, cache

    n = angles - before
    out, cache = go(end - before, angles)
    want, want_cache = go(n, end)
    assert torch.equal(out[:n], want) and (out[n:] == 7).all()
    for a, b in zip(cache, want_cache):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- all together --------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,block,dim", [(E4M3, 16, 128), (I8, 32, 64)])
def test_prompts_then_tokens_then_release(dtype, block, dim):
    """Requests of different lengths are admitted, their prompts appended in two pieces, 40 tokens decoded with a graph that takes its own
    pages, and the pages given back; a second group of requests then runs on them. Every step against 64 bits."""
    kv, heads, R = 2, 6, 4
    blocks = ops.KVBlocks.empty(R, 12, 34)
    cache = ops.KVCache8.empty(34, kv, block, dim, R, dtype)
    cos, sin = tables(12 * block, dim)
    g = torch.Generator(device="cuda").manual_seed(1)
    for turn in range(2):
        first, second = [block + 3, 2, 3 * block, 0], [5, block - 2, 7, 2 * block + 1]
        for before, new in (([0] * R, first), (first, second)):
            plan = ops.kv_plan(i32(before), i32(new), blocks, block, sum(new))
            assert blocks.state.tolist()[1] == 0
            ops.kv_append_8bit(torch.randn(sum(new), (heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16), plan, cache, cos, sin, heads)
        w = World.__new__(World)
        w.kv, w.heads, w.group, w.block, w.dim, w.dtype, w.cache, w.table, w.cos, w.sin = kv, heads, heads // kv, block, dim, dtype, cache, blocks.table, cos, sin
        w.positions = i32([a + b for a, b in zip(first, second)])
        w.qkv = torch.zeros(R, (heads + 2 * kv) * dim, device="cuda", dtype=BF16)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.kv_plan(w.positions, None, blocks, block)
            out = attend(w)
        for step in range(40):
            w.at = [int(p) for p in w.positions]
            w.qkv.copy_(torch.randn(w.qkv.shape, generator=g, device="cuda"))

            def run(w):
                graph.replay()
                return out

            ops.kv_plan(w.positions, None, blocks, block)  # (so that the model sees the table that the step uses)
            w.check(run)
            w.positions += 1
        ops.kv_release(torch.ones(R, dtype=torch.bool, device="cuda"), blocks)
        assert int(blocks.state[0]) == 34 and (blocks.table == -1).all()


def test_two_graphs_on_two_streams():
    """Two captured steps over the halves of one cache, replayed at the same time: nothing is shared but the pages."""
    at = [3000, 2500, 1234, 2999]
    w, alone = World(at, 2, 4, 16, 128, E4M3), World(at, 2, 4, 16, 128, E4M3)
    want = attend(alone)
    outs, graphs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        half = slice(2 * i, 2 * i + 2)
        c = w.cache.rows(2 * i, 2 * i + 2)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            for _ in range(20):
                out = ops.decode_attention_8bit(w.qkv[half], w.positions[half], w.table[half], c, w.cos, w.sin, w.heads)
        outs.append(out)
    for _ in range(5):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    # (fewer sequences are split finer: equal within the bound of two bf16 roundings and the weights' f16)
    got = torch.cat(outs).double()
    assert ((got - want.double()).abs() <= want.double().abs() * 2.0**-7 + 2.0**-10).all()


def test_repeats_are_equal():
    w = World([3000, 100, 2047, 31], 2, 4, 32, 128, I8)
    first = attend(w).clone()
    state = [t.clone() for t in w.cache]
    for _ in range(20):
        assert torch.equal(attend(w), first)
    for a, b in zip(state, w.cache):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
