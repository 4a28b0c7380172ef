"""The Llama decoder on the 8-bit paged cache, with log-probabilities: prefill, decode steps across block borders (eager and captured), scoring of
prompts, sequences that end, and a pool that is too small. The oracle is the model's plain fp32 step on the same (dequantised) cache; its
tolerance is that of the bf16 cache's tests, since the matrices and their bf16 roundings are the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(kv_cache, batch=4, max_seq=256, kv_heads=2, **k):
    from torch_ccl_b200.models.llama import LlamaConfig, TPLlamaDecoder

    cfg = LlamaConfig(vocab=1024, hidden=512, n_layers=2, n_heads=4, n_kv_heads=kv_heads, inter=1408)
    return TPLlamaDecoder(cfg, max_batch=batch, max_seq=max_seq, seed=3, kv_cache=kv_cache, **k)


def _prompt(B, S, seed=0):
    return torch.randint(0, 1024, (B, S), generator=torch.Generator().manual_seed(seed))


def _check_logprobs(m, B, top):
    ref = torch.log_softmax(m.logits[:B].double(), -1)
    got = m.last_logprobs
    # logits of a few units: sums of 1024 terms and their logarithm in fp32
    assert ((got.logprob.double() - ref.gather(1, m.next_tokens[:B, None])[:, 0]).abs() < 1e-5).all()
    assert ((got.entropy.double() + (ref.exp() * ref).sum(-1)).abs() < 1e-4).all()
    if top:
        assert torch.equal(got.top_ids[:, 0], m.next_tokens[:B]) and ((got.top_logprobs.double() - ref.gather(1, got.top_ids)).abs() < 1e-5).all()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kv_cache,block,kv_heads", [("fp8", 16, 2), ("int8", 32, 4), ("fp8", 64, 1)])
def test_prefill_and_decode(kv_cache, block, kv_heads, captured):
    m = _model(kv_cache, kv_heads=kv_heads, kv_block=block, logprobs=5)
    B = 4
    m.prefill(_prompt(B, 45))
    assert m.positions[:B].tolist() == [45] * B and m.blocks.held.tolist() == [-(-45 // block)] * B
    if captured:
        m.capture(B)
    for step in range(24):
        ref = m.reference_decode_step(B) if step % 5 == 0 or step in (2, 3, 18, 19) else None
        m.decode_step(B)
        torch.cuda.synchronize()
        if ref is not None:
            torch.testing.assert_close(m.logits[:B], ref, rtol=3e-2, atol=3e-2)
        _check_logprobs(m, B, 5)
    assert m.positions[:B].tolist() == [69] * B and m.blocks.held.tolist() == [-(-69 // block)] * B and m.blocks.state.tolist()[1] == 0


def test_ragged_positions_and_unfused_steps():
    m, u = _model("fp8", kv_block=16, logprobs=0), _model("fp8", kv_block=16, fused=False, logprobs=0)
    for x in (m, u):
        x.prefill(_prompt(4, 33))
        for _ in range(3):
            x.decode_step(2)  # the first two sequences alone
        ref = x.reference_decode_step(4)
        x.decode_step(4)
        assert x.positions.tolist() == [37, 37, 34, 34]
        torch.testing.assert_close(x.logits[:4], ref, rtol=3e-2, atol=3e-2)
        _check_logprobs(x, 4, 0)
    assert torch.equal(m.next_tokens, u.next_tokens)


def test_the_cache_holds_what_the_dense_one_holds():
    """After the same prompt, the 8-bit cache's values are the dense cache's within an 8-bit rounding (and the bf16 roundings of the prompt's
    rotation, which the dense path does in bf16: 2^-7 of the largest element for its products and their sum)."""
    d, q = _model("bf16"), _model("int8", kv_block=16)
    for x in (d, q):
        x.prefill(_prompt(4, 50))
    for b in range(4):
        kd, vd = d._cached(d.layers[0], b, 50)
        kq, vq = q._cached(q.layers[0], b, 50)
        for x, y in ((kd, kq), (vd, vq)):
            most = x.abs().amax((1, 2), keepdim=True)
            assert ((x - y).abs() <= most * (0.5 / 127 + 2.0**-7)).all()


def test_capture_leaves_the_sequences_as_they_were():
    """Warm-up steps before a capture append nothing, also where the next position starts a block."""
    a, b = _model("int8", kv_block=16), _model("int8", kv_block=16)
    for x in (a, b):
        x.prefill(_prompt(4, 46))
        x.decode_step(4)  # position 46 was appended; 47 ends the block
    before = [t.clone() for L in b.layers for t in L["cache"]] + [t.clone() for t in b.blocks]
    b.capture(4)
    for x, y in zip(before, [t for L in b.layers for t in L["cache"]] + list(b.blocks)):
        assert torch.equal(x.view(torch.uint8) if x.dtype.itemsize == 1 else x, y.view(torch.uint8) if y.dtype.itemsize == 1 else y)
    for _ in range(20):
        assert torch.equal(a.decode_step(4), b.decode_step(4)) and torch.equal(a.logits, b.logits)


def test_log_probabilities_after_a_capture_are_those_of_the_first_replay():
    m = _model("fp8", kv_block=16, logprobs=2)
    m.prefill(_prompt(4, 20))
    m.capture(4)
    assert m.last_logprobs is None  # nothing has run that could give any
    m.decode_step(4)
    assert torch.equal(m.last_logprobs.top_ids[:, 0], m.next_tokens[:4].long()) and (m.last_logprobs.logprob <= 0).all()


def test_sequences_end_and_others_take_their_pages():
    m = _model("fp8", kv_block=16, kv_blocks=4 * 4 + 2)
    m.prefill(_prompt(4, 60))
    assert int(m.blocks.state[0]) == 2
    m.finish([1, 3])
    assert int(m.blocks.state[0]) == 10 and m.blocks.held.tolist() == [4, 0, 4, 0]
    ref = m.reference_decode_step(1)
    for _ in range(40):
        m.decode_step(4)
    assert m.positions.tolist()[0] == 100 and m.blocks.held.tolist() == [7, 0, 7, 0] and m.blocks.state.tolist() == [4, 0]
    m.prefill(_prompt(4, 60))  # new sequences in all rows
    torch.testing.assert_close(m.reference_decode_step(1), ref, rtol=0, atol=0)
    assert int(m.blocks.state[0]) == 2
    with pytest.raises(RuntimeError, match="too few"):
        m.prefill(_prompt(4, 100))
    m.prefill(_prompt(4, 60))  # and the model is usable after that
    torch.testing.assert_close(m.reference_decode_step(1), ref, rtol=0, atol=0)


def test_a_pool_that_runs_out_says_so():
    m = _model("fp8", batch=2, kv_block=16, kv_blocks=5)
    m.prefill(_prompt(2, 31))
    for step in range(20):
        m.decode_step(2)
    # positions 32 and on need a third page each: the first sequence gets the fifth; the last step's position 50 needs a fourth
    assert m.blocks.held.tolist() == [3, 2] and m.blocks.state.tolist() == [0, 2]


@pytest.mark.parametrize("kv_cache,S", [("bf16", 12), ("fp8", 12), ("int8", 70)])
def test_score(kv_cache, S):
    m = _model(kv_cache, kv_block=16, logprobs=2) if kv_cache != "bf16" else _model(kv_cache, logprobs=2)
    B, prompt = 3, _prompt(3, S)
    got = m.score(prompt, top=4, chunk_seqs=2)
    assert got.logprob.shape == got.entropy.shape == (B, S - 1) and got.top_ids.shape == got.top_logprobs.shape == (B, S - 1, 4)
    first = m.tokens[:B].clone()
    assert (got.top_logprobs[:, :, 0] >= got.logprob).all() and (got.top_logprobs.diff(dim=-1) <= 0).all()
    at = [1, 2, S - 2]
    for t in at:  # the same from the step that takes id t after the first t
        m.prefill(prompt[:, :t])
        m.tokens[:B] = prompt[:, t].cuda()
        ref = torch.log_softmax(m.reference_decode_step(B).double(), -1)
        # logits agree within 3e-2 + 3e-2 of their size (a few units): so do their differences, twice
        want = ref.gather(1, prompt[:, t + 1, None].cuda())[:, 0]
        assert ((got.logprob[:, t].double() - want).abs() <= 2 * (3e-2 + 3e-2 * 4)).all()
        assert ((got.entropy[:, t].double() + (ref.exp() * ref).sum(-1)).abs() <= 0.3).all()
    m.prefill(prompt)
    assert torch.equal(m.tokens[:B], first)


def test_refusals():
    with pytest.raises(AssertionError, match="kv_cache"):
        _model("fp4")
    with pytest.raises(AssertionError, match="logprobs"):
        _model("fp8", logprobs=33)
    with pytest.raises(RuntimeError, match="16, 32, 64 or 128"):
        _model("fp8", kv_block=24).prefill(_prompt(1, 8))
    with pytest.raises(AssertionError, match="does not fit"):
        _model("fp8", max_seq=64).prefill(_prompt(1, 65))


@pytest.mark.parametrize("fused,captured", [(True, False), (True, True), (False, False)])
def test_a_sequence_waits_for_a_page_and_goes_on(fused, captured):
    """Row 1 gets no third page at position 32. It waits there, also past the steps in which its block would have filled up, and once row 0 has ended
    it goes on with the ids and logits that it has alone in a pool that is large enough."""
    m, alone = _model("fp8", batch=2, kv_block=16, kv_blocks=5, fused=fused, logprobs=2), _model("fp8", batch=2, kv_block=16, fused=fused)
    for x in (m, alone):
        x.prefill(_prompt(2, 31))
        if captured:
            x.capture(2)
    want = []
    for _ in range(49):
        ids = alone.decode_step(2)[1].clone()
        want.append((int(ids), alone.logits[1].clone()))
    assert int(m.decode_step(2)[1]) == want[0][0]
    for step in range(1, 22):
        ids = m.decode_step(2)
        assert ids[1] == -1 and m.positions.tolist()[1] == 32 and m.last_logprobs.logprob[1] == 0
        assert (ids[0] == -1) == (step > 16)  # row 0 has pages up to position 47
    assert m.positions.tolist() == [48, 32] and m.blocks.state.tolist() == [0, 2] and m.waits.tolist() == [True, True]
    m.finish([0])
    for ids, logits in want[1:]:
        got = m.decode_step(2)
        assert int(got[1]) == ids and torch.equal(m.logits[1], logits) and m.blocks.state.tolist()[1] == 0
    assert m.positions.tolist()[1] == 80 and m.blocks.held.tolist() == [0, 5]


def test_a_serving_loop_hands_back_what_it_got():
    """Ids go from step to step through the host, -1 among them."""
    m, alone = _model("int8", batch=2, kv_block=16, kv_blocks=5), _model("int8", batch=2, kv_block=16)
    got = []
    for x in (m, alone):
        x.prefill(_prompt(2, 31))
        ids, out, mine = x.tokens.cpu().pin_memory(), torch.zeros(2, dtype=torch.int64).pin_memory(), []
        for step in range(40):
            if x is m and step == 30:
                x.finish([0])
            x.decode_step_host(ids, out)
            ids.copy_(out)
            mine.append(int(out[1]))
        got.append([i for i in mine if i >= 0])
    assert len(got[0]) == 11 and got[0] == got[1][:11]  # the first step, and those from the 31st on


def test_a_sequence_at_the_end_of_its_room_waits():
    for kv_block in (16, 32):  # of 40 positions: three blocks, and two
        m = _model("fp8", batch=1, max_seq=40, kv_block=kv_block)
        m.prefill(_prompt(1, 38))
        ids = [int(m.decode_step(1)[0]) for _ in range(5)]
        assert all(i >= 0 for i in ids[:2]) and ids[2:] == [-1] * 3 and m.positions.tolist() == [40]


def test_a_prompt_that_was_refused_leaves_idle_rows():
    m, alone = _model("fp8", batch=3, kv_block=16, kv_blocks=7), _model("fp8", batch=3, kv_block=16)
    with pytest.raises(RuntimeError, match="too few"):
        m.prefill(_prompt(3, 40))
    assert m.blocks.state.tolist()[0] == 7 and m.blocks.held.tolist() == [0] * 3 and max(m.positions.tolist()) < 0
    before = [t.clone() for L in m.layers for t in L["cache"][4:]]
    for _ in range(3):
        m.decode_step(3)
    assert m.blocks.held.tolist() == [0] * 3 and all(torch.equal(a, b) for a, b in zip(before, [t for L in m.layers for t in L["cache"][4:]]))
    for x in (m, alone):
        x.prefill(_prompt(2, 40))
        for _ in range(6):
            x.decode_step(2)
    assert torch.equal(m.logits[:2], alone.logits[:2])
