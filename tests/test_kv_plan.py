"""Block tables and slot maps against the same rules applied to one request after the other."""
import random

import pytest
import torch

import oneccl_bindings_for_pytorch  # noqa: F401
from torch_ccl_b200 import ops

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Model:
    """The pool, in Python."""

    def __init__(self, requests, width, free):
        self.table, self.held, self.stack, self.width = [[-1] * width for _ in range(requests)], [0] * requests, list(free), width
        self.capacity = len(free)
        self.left, self.refused = len(free), 0

    def plan(self, lengths, new, block, room):
        out_of_blocks = out_of_room = False
        self.refused, starts, tokens = 0, [0], []
        for r, n in enumerate(lengths):
            t = 1 if new is None else new[r]
            served = False
            if n >= 0 and t > 0:
                want = -(-(n + t) // block)
                short = max(0, want - self.held[r])
                if want <= self.width:
                    out_of_blocks = out_of_blocks or short > self.left
                    if not short or not out_of_blocks:
                        for _ in range(short):
                            self.left -= 1
                            self.table[r][self.held[r]] = self.stack[self.left]
                            self.held[r] += 1
                        served = True
                        if room:
                            out_of_room = out_of_room or len(tokens) + t > room
                            served = not out_of_room
                            if served:
                                tokens += [(r, p, self.table[r][p // block] * block + p % block) for p in range(n, n + t)]
                self.refused += not served
            starts.append(len(tokens))
        tokens += [(-1, -1, -1)] * (room - len(tokens))
        return starts, [x[0] for x in tokens], [x[1] for x in tokens], [x[2] for x in tokens]

    def release(self, finished):
        back = [p for r, f in enumerate(finished) if f for p in self.table[r][:self.held[r]]]
        for p in reversed(back):
            self.stack[self.left] = p
            self.left += 1
        for r, f in enumerate(finished):
            if f:
                self.table[r][:self.held[r]] = [-1] * self.held[r]
                self.held[r] = 0

    def check(self, blocks):
        assert blocks.table.tolist() == self.table and blocks.held.tolist() == self.held
        assert blocks.state.tolist() == [self.left, self.refused]
        assert blocks.free.tolist()[:self.left] == self.stack[:self.left]


def pool(requests, width, num_blocks, seed=0):
    free = list(range(num_blocks))
    random.Random(seed).shuffle(free)
    blocks = ops.KVBlocks.empty(requests, width, num_blocks)
    blocks.free.copy_(i32(free))
    return blocks, Model(requests, width, free)


# rooms on both sides of one CTA, one cluster and the two-launch form (4096 and 32768 tokens)
@pytest.mark.parametrize("requests,most,room,num_blocks", [
    (1, 1, 1, 4), (1, 100, 0, 20), (3, 50, 200, 40), (33, 300, 4096, 400), (33, 300, 4097, 400), (40, 700, 32768, 2000), (40, 900, 32769, 2000),
    (1000, 262, 140000, 9000), (1023, 40, 30000, 3000), (1024, 40, 30000, 1000), (1025, 40, 30000, 3000), (5000, 9, 50000, 3000), (16384, 3, 20000, 20000)])
def test_plan_and_release(requests, most, room, num_blocks):
    rng = random.Random(requests * 7 + room)
    block, width = rng.choice([16, 32]), 64
    blocks, model = pool(requests, width, num_blocks, requests)
    lengths = [rng.choice([0, 0, rng.randrange(0, most + 1), -1]) for _ in range(requests)]
    for step in range(4):
        new = [rng.choice([0, 1, rng.randrange(0, most + 1), rng.randrange(0, most + 1)]) for _ in range(requests)]
        if step == 2:
            new[rng.randrange(requests)] = width * block + 1  # longer than the table
        plan = ops.kv_plan(i32(lengths), i32(new), blocks, block, room)
        for got, want in zip(plan, model.plan(lengths, new, block, room)):
            assert got.tolist() == want
        model.check(blocks)
        # the same plan again takes nothing
        again = ops.kv_plan(i32(lengths), i32(new), blocks, block, room)
        want = model.plan(lengths, new, block, room)
        for got, w in zip(again, want):
            assert got.tolist() == w
        model.check(blocks)
        lengths = [n + t if n >= 0 and 0 < n + t <= width * block and h * block >= n + t else n for n, t, h in zip(lengths, new, model.held)]
        finished = [rng.random() < 0.3 for _ in range(requests)]
        ops.kv_release(torch.tensor(finished, device="cuda"), blocks)
        model.release(finished)
        model.check(blocks)
        lengths = [0 if f else n for n, f in zip(lengths, finished)]


def test_one_token_each_without_a_list():
    blocks, model = pool(20, 8, 30)
    lengths = [i * 5 - 1 for i in range(20)]  # the first one: no request in that row
    for _ in range(40):
        plan = ops.kv_plan(i32(lengths), None, blocks, 16)
        assert plan.slots.numel() == 0 and plan.starts.tolist() == [0] * 21
        model.plan(lengths, None, 16, 0)
        model.check(blocks)
        lengths = [n + 1 if n >= 0 else n for n in lengths]


def test_a_list_with_room_for_two_billion():
    """The last entries of a list that is as long as one may be: a step of the loop behind them passes 2^31. (26 GB)"""
    room = 2**31 - 2
    blocks, _ = pool(2, 4, 8)
    plan = ops.kv_plan(i32([0, 3]), i32([20, 30]), blocks, 16, room)
    assert plan.starts.tolist() == [0, 20, 50] and blocks.state.tolist() == [3, 0]
    assert plan.positions[:50].tolist() == list(range(20)) + list(range(3, 33))
    for t in plan[1:]:
        assert t.shape == (room,)
        for piece in t[50:].split(1 << 28):
            assert int(piece.amin()) == int(piece.amax()) == -1


def test_what_was_planned_last_comes_back_to_its_place():
    blocks, _ = pool(50, 64, 500)
    before = [t.clone() for t in blocks]
    ops.kv_plan(i32([0] * 50), i32(list(range(50))), blocks, 16, 2000)
    ops.kv_release(torch.ones(50, dtype=torch.bool, device="cuda"), blocks)
    assert all(torch.equal(a, b) for a, b in zip(before, blocks))


def test_nothing_to_do():
    blocks, model = pool(3, 4, 0)
    plan = ops.kv_plan(i32([0, 5, -1]), i32([1, 0, 1]), blocks, 16, 10)
    assert plan.starts.tolist() == [0, 0, 0, 0] and plan.slots.tolist() == [-1] * 10 and blocks.state.tolist() == [0, 1]
    none = ops.KVBlocks.empty(0, 4, 7)
    plan = ops.kv_plan(i32([]), None, none, 16, 5)
    assert plan.starts.tolist() == [0] and plan.requests.tolist() == [-1] * 5 and none.state.tolist() == [7, 0]
    ops.kv_release(torch.ones(0, dtype=torch.bool, device="cuda"), none)
    # an empty pool's finished requests, and a second release of the same ones
    ops.kv_release(torch.ones(3, dtype=torch.bool, device="cuda"), blocks)
    assert blocks.state.tolist() == [0, 1] and blocks.table.tolist() == [[-1] * 4] * 3


def test_words_that_make_no_sense_stay_inside_the_arrays():
    blocks, _ = pool(4, 8, 10)
    blocks.state[0] = 1 << 30  # more free pages than the stack has
    plan = ops.kv_plan(i32([0, 2**31 - 5, 0, 0]), i32([40, 100, 2**31 - 1, 40]), blocks, 16, 1000)
    assert plan.requests.tolist() == [0] * 40 + [3] * 40 + [-1] * 920 and blocks.state.tolist() == [4, 2]
    blocks.held.copy_(i32([1000, -5, 0, 3]))
    ops.kv_release(torch.ones(4, dtype=torch.bool, device="cuda"), blocks)
    assert 0 <= int(blocks.state[0]) <= 10 and blocks.held.tolist() == [0] * 4
    torch.cuda.synchronize()


def test_counts_that_add_up_to_two_billion_stay_inside_the_stack():
    """A release of 16384 requests that claim all of the widest table that they may have, in a pool of a few pages. (9 GB)"""
    R, width, pages = 16384, 131071, 1000
    blocks = ops.KVBlocks.empty(R, width, pages)
    guarded = torch.full((pages + 2000,), 77, dtype=torch.int32, device="cuda")
    guarded[1000:2000] = blocks.free
    blocks = blocks._replace(free=guarded[1000:2000])
    blocks.held.fill_(2**31 - 1)
    ops.kv_release(torch.ones(R, dtype=torch.bool, device="cuda"), blocks)
    assert int(blocks.state[0]) == pages and not blocks.held.any()
    assert (guarded[:1000] == 77).all() and (guarded[2000:] == 77).all()


def test_rows_of_a_pool_and_a_graph_on_another_stream():
    blocks, model = pool(12, 16, 100)
    lengths, new = i32([7] * 12), i32([1] * 12)
    some = blocks.rows(4, 10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.kv_plan(lengths[4:10], new[4:10], some, 16, 6)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            plan = ops.kv_plan(lengths[4:10], new[4:10], some, 16, 6)
            lengths += new
        for _ in range(60):
            graph.replay()
    stream.synchronize()
    assert lengths.tolist() == [67] * 12
    assert blocks.held.tolist() == [0] * 4 + [5] * 6 + [0] * 2  # positions 0 .. 66
    assert plan.positions.tolist() == [66] * 6
    taken = [p for row in blocks.table.tolist() for p in row if p >= 0]
    assert len(set(taken)) == 30 and int(blocks.state[0]) == 70
    assert plan.slots.tolist() == [row[4] * 16 + 2 for row in blocks.table.tolist()[4:10]]
