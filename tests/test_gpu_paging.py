"""Page plans and releases against their restatement in whole numbers."""
import random

import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from gpu_util import graph_replay

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


class Server:
    """A block table with its stack, on the device and restated on the host."""

    def __init__(self, ctx, rows, max_pages, page, pages, seed=0):
        r = random.Random(seed)
        self.page, self.ids = page, list(range(pages))
        r.shuffle(self.ids)
        self.host = dict(lengths=[0] * rows, table=[[-1] * max_pages for _ in range(rows)], stack=list(self.ids), free=pages)
        self.lengths, self.table = ints([0] * rows), ints(self.host["table"])
        self.stack, self.free = ints(self.ids), ints([pages])
        self.op = tk.PagePlanOp(ctx, page)
        self.ctx = ctx

    def step(self, rows, new, capacity=None, named=True):
        h = self.host
        want = ref.plan(self.page, rows, new, h["lengths"], h["table"], h["stack"], h["free"])
        total = sum(n for n in new if n > 0)
        capacity = capacity or max(total, 1)
        if want is not None and total > capacity:
            want = None
        starts, kv = ints([-5] * (len(rows) + 1)), ints([-5] * len(rows))
        positions, slots = ints([-5] * capacity), ints([-5] * capacity, torch.int64)
        self.op.launch(None, len(rows), ints(rows) if named else None, ints(new), self.lengths, self.lengths, self.table,
                       self.stack, self.free, self.free, starts, kv, positions, slots)
        status = self.ctx.device_status()
        if want is None:
            assert status == 8
            assert starts.tolist() == [0] * (len(rows) + 1) and kv.tolist() == [0] * len(rows)
            assert slots.tolist() == [-1] * capacity
        else:
            assert status == 0
            pad = capacity - total
            assert starts.tolist() == want["starts"] and kv.tolist() == want["kv_lengths"]
            assert positions.tolist() == want["positions"] + [0] * pad and slots.tolist() == want["slots"] + [-1] * pad
            h.update(lengths=want["lengths"], table=want["table"], free=want["free"])
        self.same()
        return want

    def release(self, rows):
        h = self.host
        for row in rows:
            for k in range(-(-h["lengths"][row] // self.page)):
                h["stack"][h["free"]] = h["table"][row][k]
                h["free"] += 1
            h["lengths"][row] = 0
        self.op.release(None, len(rows), ints(rows), self.lengths, self.lengths, self.table, self.stack, self.free, self.free)
        assert self.ctx.device_status() == 0
        self.same()

    def same(self):
        h = self.host
        assert self.lengths.tolist() == h["lengths"] and self.free.tolist() == [h["free"]]
        assert self.table.tolist() == h["table"] and self.stack.tolist() == h["stack"]


@pytest.mark.parametrize("rows,page,most_new", [(1, 16, 40), (8, 64, 300), (40, 16, 90), (700, 32, 20)])
def test_a_server_over_many_steps(ctx, rows, page, most_new):
    r = random.Random(rows)
    server = Server(ctx, rows, 60, page, rows * 40, rows)
    for _ in range(8):
        chosen = r.sample(range(rows), r.randint(1, rows))
        # prompts, decodes, requests without new tokens; none beyond its row's pages
        new = [min(r.choice([0, 1, 1, r.randint(1, most_new)]), 60 * page - server.host["lengths"][row]) for row in chosen]
        server.step(chosen, new, capacity=max(sum(new), 1) + r.randint(0, 70))
        ended = [row for row in r.sample(range(rows), max(1, rows // 5))]
        server.release(ended)
    held = [i for row, n in enumerate(server.host["lengths"]) for i in server.host["table"][row][:-(-n // page)]]
    assert sorted(held + server.host["stack"][:server.host["free"]]) == sorted(server.ids), "a page was lost or is held twice"


def test_most_requests_and_tokens(ctx):
    server = Server(ctx, 4096, 3, 16, 4096 * 3)
    server.step(list(range(4096)), [i % 40 for i in range(4096)], named=False)
    server.step(list(range(4095, -1, -1)), [1 + (i % 3 == 0) for i in range(4096)])
    wide = Server(ctx, 2, 2000, 64, 4000)
    wide.step([1, 0], [100000, 27])


@pytest.mark.parametrize("rows,new,capacity", [([0, 0], [1, 1], 8), ([0, 4], [1, 1], 8), ([0, -1], [1, 1], 8), ([0, 1], [1, -1], 8),
                                               ([0, 1], [5, 4], 8), ([0], [16 * 5 + 1], 200), ([0, 1, 2], [80, 80, 1], 200),
                                               ([0, 1], [2 ** 31 - 1, 2 ** 31 - 1], 8)])
def test_steps_that_do_not_fit_change_nothing(ctx, rows, new, capacity):
    server = Server(ctx, 4, 5, 16, 10)
    server.step([3], [0], capacity=4)
    assert server.step(rows, new, capacity) is None
    server.step([1, 0], [16, 17])  # and the next one runs


def test_releases_that_do_not_fit_change_nothing(ctx):
    server = Server(ctx, 4, 5, 16, 10)
    server.step([0, 1], [33, 20])
    for rows in ([0, 0], [4], [-1]):
        server.op.release(None, len(rows), ints(rows), server.lengths, server.lengths, server.table, server.stack, server.free, server.free)
        assert ctx.device_status() == 8
        server.same()
    full = ints([10])
    server.op.release(None, 1, ints([0]), server.lengths, server.lengths, server.table, server.stack, full, full)
    assert ctx.device_status() == 8 and full.tolist() == [10]


def test_outputs_of_their_own_and_replay(ctx):
    """With other planes for the new values a step can be planned again; in place, replays go on from one another."""
    server = Server(ctx, 3, 8, 16, 24)
    server.step([0, 2], [20, 5])
    lengths, free = server.lengths.clone(), server.free.clone()
    starts, kv, positions, slots = ints([0] * 4), ints([0] * 3), ints([0] * 6), ints([0] * 6, torch.int64)
    new = ints([1, 1, 1])
    for _ in range(2):
        server.op.launch(None, 3, None, new, server.lengths, lengths, server.table, server.stack, server.free, free, starts, kv,
                         positions, slots)
        assert kv.tolist() == [21, 1, 6] and positions.tolist() == [20, 0, 5, 0, 0, 0] and lengths.tolist() == [21, 1, 6]
        assert server.lengths.tolist() == [20, 0, 5] and slots[3:].tolist() == [-1] * 3

    def step():
        server.op.launch(None, 3, None, new, lengths, lengths, server.table, server.stack, free, free, starts, kv, positions, slots)

    graph = graph_replay(step)  # one run before the capture
    for i in range(40):
        graph.replay()
    assert lengths.tolist() == [62, 42, 47]
    held = [server.table[r, :-(-n // 16)].tolist() for r, n in enumerate(lengths.tolist())]
    assert len({i for row in held for i in row}) == sum(len(row) for row in held) == 10 == 24 - int(free)
    for r, n in enumerate(lengths.tolist()):
        assert int(slots[r]) == held[r][(n - 1) // 16] * 16 + (n - 1) % 16


def test_refusals(ctx):
    server = Server(ctx, 2, 4, 16, 8)
    base = dict(requests=1, request_rows=None, new_tokens=ints([1]), lengths=server.lengths, lengths_output=server.lengths,
                block_table=server.table, free_pages=server.stack, free_count=server.free, free_count_output=server.free,
                starts=ints([0, 0]), kv_lengths=ints([0]), positions=ints([0]), slots=ints([0], torch.int64))

    def refused(text, operator=server.op, **change):
        with pytest.raises(tk.GpuError, match=text):
            operator.launch(None, **{**base, **change})

    refused("request count", requests=0)
    refused("request count", requests=4097, new_tokens=ints([0] * 4097), starts=ints([0] * 4098), kv_lengths=ints([0] * 4097))
    refused("new tokens", new_tokens=ints([1], torch.int64))
    refused("new tokens", requests=2, starts=ints([0, 0, 0]), kv_lengths=ints([0, 0]))
    refused("starts", starts=ints([0]))
    refused("slots", slots=ints([0]))
    refused("positions", slots=ints([0, 0], torch.int64))
    refused("block table", block_table=server.table.view(-1))
    refused("lengths", lengths=server.lengths[:1])
    refused("free count", free_count=torch.tensor([8], dtype=torch.int32))
    refused("power of two", operator=tk.PagePlanOp(ctx, 24))
    refused("power of two", operator=tk.PagePlanOp(ctx, 8))
