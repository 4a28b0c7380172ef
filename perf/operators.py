"""The operators of serving from an 8-bit paged KV cache, and of token log-probabilities, as timed cases.

Four kinds of call:

  attn    `ops.decode_attention_8bit`: one new token for each of `batch` sequences: rotary embedding, append, attention over the cache
  append  `ops.kv_append_8bit`: rotary embedding of whole prompts and their quantisation into the cache's pages
  plan    `ops.kv_plan` and `ops.kv_release`: requests are admitted (blocks from the pool, a slot for every token) and leave again
  logp    `ops.token_logprobs`: log-probability of given tokens, entropy, the best alternatives; with `backward` the logits' gradient too

The cache. `block` tokens of one KV head share a page: 8-bit codes (e4m3 or int8) and one fp32 scale for K, one for V. The block that a
sequence is still filling is held in bf16 (its "tail") and quantised once, when its last token arrives:
scale = max(amax / qmax, 2^-40), code = round(x / scale). Attention of position p reads the blocks before p // block from their pages and the
rest, the new token included, from the tail.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's operators.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
LEAST_SCALE = 2.0 ** -40
THETA = 10000.0


def listed():
    mha = dict(heads=32, kv_heads=32, dim=128)  # the 7B architecture of the benchmark
    gqa = dict(heads=32, kv_heads=8, dim=128)   # grouped-query heads
    return [
        # one user in a long chat on the 7B model: a launch per layer, nothing but latency
        dict(name="attn_b1", kind="attn", batch=1, context=1000, ragged=False, block=16, codes="e4m3", **mha),
        # the benchmark's decode step: 16 users with prompts of 1024 ids
        dict(name="attn_b16", kind="attn", batch=16, context=1087, ragged=False, block=32, codes="e4m3", **mha),
        # a busy server: many sequences of very different lengths, grouped-query heads
        dict(name="attn_ragged_b33", kind="attn", batch=33, context=2999, ragged=True, block=64, codes="e4m3", **gqa),
        # a few users with documents of 65 thousand ids, eight heads to a KV head
        dict(name="attn_long_b7", kind="attn", batch=7, context=65521, ragged=False, block=128, codes="int8", heads=64, kv_heads=8, dim=128),
        # a few prompts of odd lengths
        dict(name="append_3x777", kind="append", batch=3, tokens=777, before=0, ragged=True, block=16, codes="e4m3", **gqa),
        # the benchmark's prompts: 16 x 1024 ids
        dict(name="append_16x1024", kind="append", batch=16, tokens=1024, before=0, ragged=False, block=32, codes="e4m3", **mha),
        # a handful of short requests arrives
        dict(name="plan_16", kind="plan", requests=16, tokens=40, before=0, block=16, short=False),
        # a server that takes in a thousand requests at once, some of them in the middle of their prompt; its pool is too small for all of them
        dict(name="plan_1000", kind="plan", requests=1000, tokens=262, before=100, block=16, short=True),
        # log-probabilities of the ids that 16 users were just given, with five alternatives
        dict(name="logp_decode_b16", kind="logp", rows=16, vocab=32000, dtype="f32", top=5, backward=False),
        # a small model's training step: fp32 logits, value and gradient
        dict(name="logp_train_100x1024", kind="logp", rows=100, vocab=1024, dtype="f32", top=0, backward=True),
        # scoring a prompt with a large vocabulary of odd size, twenty alternatives
        dict(name="logp_score_777x100003", kind="logp", rows=777, vocab=100003, dtype="bf16", top=20, backward=False),
        # a training step on sequences that the model wrote itself: log-probabilities, entropies and the gradient of both
        dict(name="logp_train_4095x32000", kind="logp", rows=4095, vocab=32000, dtype="bf16", top=0, backward=True),
    ]


# ---- drawn cases -------------------------------------------------------------------------------------

def _log(rng, lo, hi, step=1):
    """A whole number between lo and hi, evenly spread over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _draw(rng, kind):
    if kind in ("attn", "append"):
        kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
        c = dict(kind=kind, block=rng.choice([16, 32, 64, 128]), codes=rng.choice(["e4m3", "e4m3", "int8"]), dim=rng.choice([64, 128, 128]),
                 kv_heads=kv, heads=kv * rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), ragged=rng.random() < 0.6)
        if kind == "attn":
            return dict(c, batch=_log(rng, 1, 256), context=_log(rng, 1, 65536))
        return dict(c, batch=_log(rng, 1, 64), tokens=_log(rng, 1, 8192), before=rng.choice([0, 0, _log(rng, 1, 4096)]))
    if kind == "plan":
        return dict(kind=kind, requests=_log(rng, 1, 4000), tokens=_log(rng, 1, 30000), before=rng.choice([0, _log(rng, 1, 30000)]),
                    block=rng.choice([16, 32, 64, 128]), short=rng.random() < 0.4)
    return dict(kind=kind, rows=_log(rng, 1, 8192), vocab=_log(rng, 500, 200000), dtype=rng.choice(sorted(DTYPES)),
                top=rng.choice([0, 1, 5, 20, 32]), backward=rng.random() < 0.5)


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def draw(rng):
    kind = rng.choice(["attn", "attn", "append", "plan", "logp"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        c = _draw(rng, kind)
        if _cost(c) > most:
            continue
        if kind == "attn" and c["batch"] * (c["context"] + c["block"]) * c["kv_heads"] * c["dim"] > 500 << 20:
            continue  # the padded 32-bit copies of the plain form would not fit the card
        if kind == "append" and c["batch"] * (c["tokens"] + c["before"]) * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] > 400 << 20:
            continue
        if kind == "plan" and c["requests"] * (c["tokens"] + c["before"]) > 400_000:
            continue
        return c


# ---- sizes -------------------------------------------------------------------------------------------

def _spread(n, most, ragged):
    """`n` lengths up to `most`: all of them `most`, or spread between 1 and `most` in no order."""
    if not ragged:
        return [most] * n
    return [max(1, most - (i * 7919 % n) * most // n) for i in range(n)]


def _before(case):
    """Tokens that each sequence of an append or plan case already holds."""
    n = case.get("batch") or case["requests"]
    return [case["before"] * (i % 3) // 2 for i in range(n)]


def _plan_sizes(case):
    """(lengths, new tokens, blocks needed, free blocks, tokens there is room for) of a plan case; other requests hold 1000 blocks more."""
    n, bs = case["requests"], case["block"]
    held = _before(case)
    new = [0 if n > 4 and i % 11 == 10 else v for i, v in enumerate(_spread(n, case["tokens"], n > 1))]  # some slots of the batch are empty
    need = [(h + t + bs - 1) // bs if t else 0 for h, t in zip(held, new)]
    total = sum(need)
    pool = max(1, total * 9 // 10) if case["short"] else total + 7
    return held, new, need, pool, sum(new)


def work(case):
    if case["kind"] == "attn":
        B, H, KV, D, bs = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["block"]
        n = b = 0
        for p in _spread(B, case["context"], case["ragged"]):
            full = p // bs
            n += p + 1
            b += full * (KV * (2 * bs * D + 8) + 4) + (p % bs) * KV * D * 4  # pages and their scales, the tail
        return {"bytes": b + B * ((2 * H + 2 * KV) * D * 2 + KV * D * 4 + 4), "flops": 4 * H * D * n}
    if case["kind"] == "append":
        H, KV, D, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
        n = sum(_spread(case["batch"], case["tokens"], case["ragged"]))
        return {"bytes": n * ((H + 2 * KV) * D * 2 + (H + KV) * D * 2 + 2 * KV * D + 12) + case["batch"] * KV * bs * D * 4, "flops": n * (H + KV) * D * 3}
    if case["kind"] == "plan":
        _, _, need, pool, tokens = _plan_sizes(case)
        blocks = min(sum(need), pool)
        # lengths, new tokens, starts and counts of a request; free list and table entry of a block, taken and given back; three words a token
        return {"bytes": case["requests"] * 24 + blocks * 16 + tokens * 12, "flops": 0}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * DTYPES[case["dtype"]].itemsize * (3 if case["backward"] else 1) + case["rows"] * (16 + 12 * case["top"]), "flops": n * (12 if case["backward"] else 6)}


# ---- inputs ------------------------------------------------------------------------------------------

def _tables(positions, dim):
    inv = 1.0 / (THETA ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float32) / dim))
    ang = torch.arange(positions, device="cuda", dtype=torch.float32)[:, None] * inv[None, :]
    return ang.cos().contiguous(), ang.sin().contiguous()


def _heads_like(g, *shape):
    """Projection rows as a model has them: normal, some channels several times larger than the rest."""
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    loud = torch.rand(shape[-1], generator=g, device="cuda") < 0.02
    return (x * torch.where(loud, 4.0, 1.0)).to(BF16)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return {"attn": _prepare_attn, "append": _prepare_append, "plan": _prepare_plan, "logp": _prepare_logp}[case["kind"]](case, g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_attn(case, g):
    B, H, KV, D, bs, codes = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["block"], case["codes"]
    pos = _spread(B, case["context"], case["ragged"])
    M = max(pos) // bs + 1
    used = [p // bs + 1 for p in pos]
    P = sum(used) + 1  # one page is nobody's
    pages = torch.randperm(P - 1, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, M), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = pages[at:at + n]
        at += n

    def pool():
        if codes == "int8":
            return torch.randint(-127, 128, (P, KV, bs, D), generator=g, device="cuda", dtype=torch.int8)
        x = torch.empty(P, KV, bs, D, device="cuda", dtype=torch.float16).normal_(0, 100, generator=g)
        return x.clamp_(-448, 448).to(CODES[codes])

    def scales():
        return (0.5 + torch.rand(P, KV, generator=g, device="cuda")) * (3.0 / QMAX[codes])

    cos, sin = _tables(M * bs, D)
    return dict(case=case, qkv=_heads_like(g, B, (H + 2 * KV) * D), positions=_i32(pos), table=table,
                cache=(pool(), pool(), scales(), scales(), _heads_like(g, B, KV, bs, D), _heads_like(g, B, KV, bs, D)), cos=cos, sin=sin)


def _prepare_append(case, g):
    B, H, KV, D, bs, codes = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["block"], case["codes"]
    before, new = _before(case), _spread(case["batch"], case["tokens"], case["ragged"])
    first = [h // bs for h in before]
    blocks = [(h + t + bs - 1) // bs - f for h, t, f in zip(before, new, first)]
    P = sum(blocks) + 1  # one page is nobody's
    pages = torch.randperm(P - 1, generator=g, device="cuda").to(torch.int32)
    starts, page_at, N = [0], [], sum(new)
    for t, n in zip(new, blocks):
        starts.append(starts[-1] + t)
        page_at.append(sum(blocks[:len(page_at)]))
    counts = torch.tensor(new, device="cuda")
    requests = torch.repeat_interleave(torch.arange(B, device="cuda"), counts, output_size=N)
    positions = torch.arange(N, device="cuda") - torch.tensor(starts[:-1], device="cuda")[requests] + torch.tensor(before, device="cuda")[requests]
    block = torch.tensor(page_at, device="cuda")[requests] + positions // bs - torch.tensor(first, device="cuda")[requests]
    slots = pages[block].long() * bs + positions % bs

    def pool():
        return torch.zeros(P, KV, bs, D, device="cuda", dtype=torch.uint8).view(CODES[codes])

    cos, sin = _tables(max(h + t for h, t in zip(before, new)), D)
    return dict(case=case, qkv=_heads_like(g, N, (H + 2 * KV) * D), plan=(_i32(starts), requests.to(torch.int32), positions.to(torch.int32), slots.to(torch.int32)),
                cache=(pool(), pool(), torch.zeros(P, KV, device="cuda"), torch.zeros(P, KV, device="cuda"), _heads_like(g, B, KV, bs, D), _heads_like(g, B, KV, bs, D)),
                cos=cos, sin=sin, dense=max(blocks))


def _prepare_plan(case, g):
    held, new, need, pool, tokens = _plan_sizes(case)
    n = case["requests"]
    order = torch.randperm(n, generator=g, device="cuda")
    lengths, new_tokens = _i32(held)[order], _i32(new)[order]
    return dict(case=case, lengths=lengths, new=new_tokens, tokens=tokens, blocks=(
        torch.full((n, max(max(need), 1)), -1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"),
        torch.randperm(pool + 1000, generator=g, device="cuda").to(torch.int32), _i32([pool, 0])), finished=torch.ones(n, dtype=torch.bool, device="cuda"))


def _prepare_logp(case, g):
    n, v = case["rows"], case["vocab"]
    x = torch.randn(n, v, generator=g, device="cuda", dtype=torch.float32)
    x *= 1.0 + 3.0 * torch.rand(n, 1, generator=g, device="cuda")  # flat and peaked rows
    targets = torch.multinomial(torch.softmax(x[:, : min(v, 4096)], -1), 1, generator=g)[:, 0]
    if n > 8:
        targets[n // 2] = -1  # padding
    d = dict(case=case, logits=x.to(DTYPES[case["dtype"]]), targets=targets)
    if case["backward"]:
        d["logits"].requires_grad_(True)
        d["grads"] = tuple(torch.randn(n, generator=g, device="cuda") for _ in range(2)) + ((torch.randn(n, case["top"], generator=g, device="cuda"),) if case["top"] else ())
    return d


# ---- the calls -----------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attn": _own_attn, "append": _own_append, "plan": _own_plan, "logp": _own_logp}[kind](state)
    with torch.no_grad():
        return {"attn": _plain_attn, "append": _plain_append, "plan": _plain_plan, "logp": _plain_logp}[kind](state)


def _held(state, blocks):
    """The cache's pages as outputs: e4m3 codes with their scales, int8 as the values that they stand for (in the pages `blocks`, or all)."""
    k, v, ks, vs = state["cache"][:4]
    if state["case"]["codes"] == "e4m3":
        return [k, v, ks, vs]
    if blocks is None:
        return [(k * ks[:, :, None, None]).to(BF16), (v * vs[:, :, None, None]).to(BF16), ks, vs]
    return [(k[blocks] * ks[blocks][:, :, None, None]).to(BF16), (v[blocks] * vs[blocks][:, :, None, None]).to(BF16), ks, vs]


def _own_attn(s):
    from torch_ccl_b200 import ops

    out = ops.decode_attention_8bit(s["qkv"], s["positions"], s["table"], ops.KVCache8(*s["cache"]), s["cos"], s["sin"], s["case"]["heads"])
    return [out, *s["cache"][4:], *_held(s, s["table"][:, -1] if s["case"]["codes"] == "int8" else None)]


def _own_append(s):
    from torch_ccl_b200 import ops

    rotated = ops.kv_append_8bit(s["qkv"], ops.KVPlan(*s["plan"]), ops.KVCache8(*s["cache"]), s["cos"], s["sin"], s["case"]["heads"])
    return [rotated, *s["cache"][4:], *_held(s, None)]


def _own_plan(s):
    from torch_ccl_b200 import ops

    blocks = ops.KVBlocks(*s["blocks"])
    plan = ops.kv_plan(s["lengths"], s["new"], blocks, s["case"]["block"], s["tokens"])
    ops.kv_release(s["finished"], blocks)
    return [*plan, *s["blocks"]]


def _own_logp(s):
    from torch_ccl_b200 import ops

    got = ops.token_logprobs(s["logits"], s["targets"], top=s["case"]["top"])
    outs = [got.logprob, got.entropy] + ([got.top_logprobs, got.top_ids] if s["case"]["top"] else [])
    if s["case"]["backward"]:
        outs += torch.autograd.grad(outs[:3] if s["case"]["top"] else outs, [s["logits"]], list(s["grads"]))
    return [t.detach() for t in outs]


# ---- the plain forms -------------------------------------------------------------------------------------

def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _quantise(x, codes):
    """Codes (as bytes) and scales of blocks x [..., block, dim]."""
    top = torch.full((), QMAX[codes], device=x.device)
    scale = (x.abs().amax((-2, -1)) / top).clamp(min=LEAST_SCALE)
    y = x / scale[..., None, None]
    y = y.to(torch.float8_e4m3fn) if codes == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)
    return y.view(torch.uint8), scale


def _plain_attn(s):
    c = s["case"]
    B, H, KV, D, bs = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["block"]
    k, v, ks, vs, kt, vt = s["cache"]
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    x = s["qkv"].float()
    q = _rotate(x[:, : H * D].view(B, H, D), cos, sin).view(B, KV, H // KV, D)
    kn = _rotate(x[:, H * D:(H + KV) * D].view(B, KV, D), cos, sin).to(BF16)
    vn = s["qkv"][:, (H + KV) * D:].view(B, KV, D)
    rows = torch.arange(B, device="cuda")
    kt[rows, :, pos % bs] = kn
    vt[rows, :, pos % bs] = vn
    # blocks that are full now go to their pages
    page = s["table"][rows, pos // bs].long()
    full = (pos % bs == bs - 1)[:, None]

    def turn_in(pool, scales, tail):
        codes, scale = _quantise(tail.float(), c["codes"])
        b8 = pool.view(torch.uint8)
        b8[page] = torch.where(full[:, :, None, None], codes, b8[page])
        scales[page] = torch.where(full, scale, scales[page])

    turn_in(k, ks, kt)
    turn_in(v, vs, vt)
    M = s["table"].shape[1]
    pages = s["table"].long().clamp(min=0)

    def gathered(pool, scales, tail):
        y = pool.view(torch.uint8)[pages].view(pool.dtype).float() * scales[pages][..., None, None]  # [B, M, KV, bs, D]
        return torch.cat([y.transpose(1, 2).reshape(B, KV, M * bs, D), tail.float()], dim=2)

    t = torch.arange(M * bs, device="cuda")[None]
    live = torch.cat([t < (pos // bs * bs)[:, None], torch.arange(bs, device="cuda")[None] <= (pos % bs)[:, None]], dim=1)
    score = torch.matmul(q, gathered(k, ks, kt).transpose(-1, -2)) / math.sqrt(D)
    score = torch.where(live[:, None, None], score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    values = gathered(v, vs, vt)
    out = torch.matmul(p, torch.where(live[:, None, :, None], values, 0.0)).reshape(B, H * D).to(BF16)
    return [out, kt, vt, *_held(s, s["table"][:, -1] if c["codes"] == "int8" else None)]


def _plain_append(s):
    c = s["case"]
    B, H, KV, D, bs, nb = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["block"], s["dense"]
    k, v, ks, vs, kt, vt = s["cache"]
    starts, requests, positions, slots = (t.long() for t in s["plan"])
    x = s["qkv"].float()
    N = x.shape[0]
    cos, sin = s["cos"][positions][:, None], s["sin"][positions][:, None]
    rotated = _rotate(x[:, :(H + KV) * D].view(N, H + KV, D), cos, sin).to(BF16)
    before = positions[starts[:-1]]
    end = before + starts[1:] - starts[:-1]
    first = before // bs
    place = positions - first[requests] * bs  # in the request's own row of blocks
    page = torch.full((B, nb), k.shape[0] - 1, dtype=torch.int64, device="cuda")
    page[requests, place // bs] = slots // bs
    block = first[:, None] + torch.arange(nb, device="cuda")
    full = (block + 1) * bs <= end[:, None]
    page = torch.where(full, page, k.shape[0] - 1)
    left = (end % bs)[:, None] > torch.arange(bs, device="cuda")
    last = (end // bs - first).clamp(max=nb - 1)

    def turn_in(pool, scales, tail, new):
        dense = torch.zeros(B, nb * bs, KV, D, dtype=BF16, device="cuda")
        dense[:, :bs] = tail.transpose(1, 2)
        dense[requests, place] = new
        dense = dense.view(B, nb, bs, KV, D).transpose(2, 3)
        codes, scale = _quantise(dense.float(), c["codes"])
        b8 = pool.view(torch.uint8)
        b8[page] = torch.where(full[:, :, None, None, None], codes, b8[page])
        scales[page] = torch.where(full[:, :, None], scale, scales[page])
        # (a request that ends on a block's border leaves its tail as it was)
        tail.copy_(torch.where(left[:, None, :, None], dense[torch.arange(B, device="cuda"), last], tail))

    turn_in(k, ks, kt, rotated[:, H:])
    turn_in(v, vs, vt, s["qkv"][:, (H + KV) * D:].view(N, KV, D))
    return [rotated.reshape(N, (H + KV) * D), kt, vt, *_held(s, None)]


def _plain_plan(s):
    bs, lengths, new, room = s["case"]["block"], s["lengths"].long(), s["new"].long(), s["tokens"]
    table, held, free, state = s["blocks"]
    R, M = table.shape
    has = held.long()
    # blocks, first come, first served
    want = (lengths + new + bs - 1) // bs
    asks = (new > 0) & (lengths >= 0)
    long = want > M
    need = torch.where(asks & ~long, (want - has).clamp(min=0), 0)
    upto = need.cumsum(0)
    given = (need == 0) | (upto <= state[0])
    need = torch.where(given, need, 0)
    upto = need.cumsum(0)
    base = upto - need
    # tokens of the requests that have their blocks
    t = torch.where(asks & ~long & given, new, 0)
    fits = t.cumsum(0) <= room
    t = torch.where(fits, t, 0)
    starts = torch.cat([t.new_zeros(1), t.cumsum(0)])
    refused = (asks & (t == 0)).sum()
    # table entries of the new blocks
    col = torch.arange(M, device="cuda")[None]
    fresh = (col >= has[:, None]) & (col < (has + need)[:, None])
    rank = base[:, None] + col - has[:, None]
    table.copy_(torch.where(fresh, free[(state[0] - 1 - rank).clamp(0, free.numel() - 1).long()], table))
    held.copy_(has + need)
    state[0] -= upto[-1].to(torch.int32)
    state[1] = refused.to(torch.int32)
    # one entry for each token
    i = torch.arange(room, device="cuda")
    r = torch.searchsorted(starts[1:], i, right=True)
    live = r < R
    r = r.clamp(max=R - 1)
    p = lengths[r] + i - starts[r]
    slot = table[r, torch.where(live, p // bs, 0)].long() * bs + p % bs
    outs = [starts.to(torch.int32)] + [torch.where(live, y, -1).to(torch.int32) for y in (r, p, slot)]
    # the requests leave: their blocks go back to where they came from
    n = torch.where(s["finished"], held.long(), 0)
    upto = n.cumsum(0)
    rank = (upto - n)[:, None] + col
    gone = col < n[:, None]
    to = torch.where(gone, state[0] + upto[-1] - 1 - rank, free.numel())
    free.copy_(torch.cat([free, free.new_zeros(1)]).scatter(0, to.flatten(), table.flatten())[:-1])
    table.copy_(torch.where(gone, -1, table))
    state[0] += upto[-1].to(torch.int32)
    held.copy_(torch.where(s["finished"], 0, held))
    return [*outs, table, held, free, state]


def _plain_logp(s):
    x, t, top = s["logits"].float(), s["targets"], s["case"]["top"]
    some = t >= 0
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    logp = x - lse
    at = t.clamp(min=0)[:, None]
    p = e / z
    ent = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    outs = [torch.where(some, logp.gather(1, at)[:, 0], 0.0), ent]
    if top:
        best = torch.sort(x, dim=-1, descending=True, stable=True)
        ids = best.indices[:, :top]
        outs += [best.values[:, :top] - lse, ids]
    if s["case"]["backward"]:
        g_lp, g_ent = torch.where(some, s["grads"][0], 0.0)[:, None], s["grads"][1][:, None]
        whole = g_lp + (s["grads"][2].sum(-1, keepdim=True) if top else 0.0)
        d = -p * (whole + torch.where(p > 0, g_ent * (logp + ent[:, None]), 0.0))
        d.scatter_add_(1, at, g_lp)
        if top:
            d.scatter_add_(1, ids, s["grads"][2])
        outs.append(d.to(s["logits"].dtype))
    return outs


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "append": _exact_append, "plan": _exact_plan, "logp": _exact_logp}[case["kind"]](s)


def _turned(x, angle_cos, angle_sin):
    """Pairs (i, i + D/2) of x as complex numbers, turned."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.complex(angle_cos.double(), angle_sin.double())
    return torch.cat([z.real, z.imag], -1)


def _page(block, codes):
    """(values of the codes, scale) of one block [bs, D] of 64-bit numbers."""
    scale = max(float(block.abs().max()) / QMAX[codes], LEAST_SCALE)
    y = block / scale
    y = y.float().to(torch.float8_e4m3fn).double() if codes == "e4m3" else torch.round(y).clamp(-127, 127)
    return y, scale


def _exact_attn(s):
    c = s["case"]
    H, KV, D, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    k, v, ks, vs, kt, vt = s["cache"]
    out = torch.empty(c["batch"], H, D, dtype=torch.float64, device="cuda")
    table = s["table"].tolist()
    for b, p in enumerate(s["positions"].tolist()):
        row = s["qkv"][b].view(-1, D)
        q = _turned(row[:H], s["cos"][p], s["sin"][p])
        kt[b, :, p % bs] = _turned(row[H:H + KV], s["cos"][p], s["sin"][p]).to(BF16)
        vt[b, :, p % bs] = row[H + KV:]
        full = torch.tensor(table[b][:p // bs], dtype=torch.long, device="cuda")
        for h in range(KV):
            def all_of(pool, scales, tail):
                paged = pool[:, h].view(torch.uint8)[full].view(pool.dtype).double() * scales[full, h].double()[:, None, None]
                return torch.cat([paged.reshape(-1, D), tail[b, h, : p % bs + 1].double()])

            of = slice(h * (H // KV), (h + 1) * (H // KV))
            w = torch.softmax(q[of] @ all_of(k, ks, kt).T * D ** -0.5, dim=-1)
            out[b, of] = w @ all_of(v, vs, vt)
    for b, p in enumerate(s["positions"].tolist()):
        if p % bs == bs - 1:
            for pool, scales, tail in ((k, ks, kt), (v, vs, vt)):
                for h in range(KV):
                    y, scale = _page(tail[b, h].double(), c["codes"])
                    pool.view(torch.uint8)[table[b][p // bs], h] = y.float().to(pool.dtype).view(torch.uint8)
                    scales[table[b][p // bs], h] = scale
    blocks = s["table"][:, -1].long()
    held = [k, v, ks, vs] if c["codes"] == "e4m3" else [k[blocks] * ks[blocks].double()[:, :, None, None], v[blocks] * vs[blocks].double()[:, :, None, None], ks, vs]
    return [out.reshape(c["batch"], H * D), kt, vt, *held]


def _exact_append(s):
    c = s["case"]
    H, KV, D, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    k, v, ks, vs, kt, vt = s["cache"]
    starts, positions, slots = s["plan"][0].tolist(), s["plan"][2], s["plan"][3].tolist()
    if sum(math.ceil((b - a) / bs) for a, b in zip(starts, starts[1:])) > 4000:
        return None
    rows = s["qkv"].view(len(slots), -1, D)
    turned = _turned(rows[:, :H + KV], s["cos"][positions.long()][:, None], s["sin"][positions.long()][:, None])
    keys, values = turned[:, H:].to(BF16), rows[:, H + KV:]
    before = [int(positions[a]) for a in starts[:-1]]
    for r, (a, e) in enumerate(zip(starts, starts[1:])):
        old = before[r] % bs
        for pool, scales, tail, x in ((k, ks, kt, keys), (v, vs, vt, values)):
            line = torch.cat([tail[r, :, :old].transpose(0, 1), x[a:e]]).transpose(0, 1)  # [KV, tokens, D] from the first touched block on
            n = line.shape[1] // bs
            if n:
                at = torch.tensor([slots[a + max(0, i * bs - old)] // bs for i in range(n)], device="cuda")
                blocks = line[:, : n * bs].reshape(KV, n, bs, D).transpose(0, 1).double()
                scale = (blocks.abs().amax((2, 3)) / QMAX[c["codes"]]).clamp(min=LEAST_SCALE)
                y = blocks / scale[:, :, None, None]
                y = y.float() if c["codes"] == "e4m3" else torch.round(y).clamp(-127, 127)
                pool.view(torch.uint8)[at] = y.to(pool.dtype).view(torch.uint8)
                scales[at] = scale.float()
            tail[r, :, : line.shape[1] - n * bs] = line[:, n * bs:]
    held = [k, v, ks, vs] if c["codes"] == "e4m3" else [k.double() * ks[:, :, None, None], v.double() * vs[:, :, None, None], ks, vs]
    return [turned.reshape(len(slots), -1), kt, vt, *held]


def _exact_plan(s):
    """The same rules, one request after the other."""
    bs, room = s["case"]["block"], s["tokens"]
    table, held, free, state = (t.tolist() for t in s["blocks"])
    left, out_of_blocks, out_of_room, refused = state[0], False, False, 0
    starts, requests, positions, slots = [0], [], [], []
    for r, (n, t) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
        served = False
        if n >= 0 and t > 0:
            want = -(-(n + t) // bs)
            short = max(0, want - held[r])
            if want <= len(table[r]):
                out_of_blocks = out_of_blocks or short > left
                if short == 0 or not out_of_blocks:
                    for i in range(short):
                        left -= 1
                        table[r][held[r]] = free[left]
                        held[r] += 1
                    out_of_room = out_of_room or len(slots) + t > room
                    served = not out_of_room
            refused += not served
            if served:
                for p in range(n, n + t):
                    requests.append(r)
                    positions.append(p)
                    slots.append(table[r][p // bs] * bs + p % bs)
        starts.append(len(slots))
    none = [-1] * (room - len(slots))
    # everybody leaves: what was taken last goes back first
    return [torch.tensor(y, dtype=torch.int32) for y in (starts, requests + none, positions + none, slots + none)] + [
        torch.full_like(s["blocks"][0], -1), torch.zeros_like(s["blocks"][1]), s["blocks"][2], torch.tensor([state[0], refused], dtype=torch.int32)]


def _exact_logp(s):
    x, t, top = s["logits"].double(), s["targets"], s["case"]["top"]
    logp = torch.log_softmax(x, dim=-1)
    p = logp.exp()
    rows = torch.arange(x.shape[0], device="cuda")
    some = (t >= 0).double()
    lp = logp[rows, t.clamp(min=0)] * some
    plogp = torch.nan_to_num(p * logp, nan=0.0)
    ent = -plogp.sum(-1)
    outs = [lp, ent]
    if top:
        ids = torch.argsort(-x, dim=-1, stable=True)[:, :top]
        outs += [logp.gather(1, ids), ids]
    if s["case"]["backward"]:
        g = [y.double() for y in s["grads"]]
        d = -plogp * g[1][:, None] - p * (g[1] * ent)[:, None] - p * (g[0] * some)[:, None]
        d[rows, t.clamp(min=0)] += g[0] * some
        if top:
            d -= p * g[2].sum(-1, keepdim=True)
            d.scatter_add_(1, ids, g[2])
        outs.append(d)
    return outs
