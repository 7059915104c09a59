"""Page ids that name no page: reported where they are met."""
import pytest
import torch

import tuiskollm_b200 as tk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def plan(ctx, new, lengths, table, stack, free, capacity):
    starts, kv = ints([0] * (len(new) + 1)), ints([0] * len(new))
    positions, slots = ints([-5] * capacity), ints([-5] * capacity, torch.int64)
    count = ints([free])
    tk.PagePlanOp(ctx, 16).launch(None, len(new), None, ints(new), lengths, lengths, table, ints(stack), count, count, starts, kv,
                                  positions, slots)
    return kv.tolist(), positions.tolist(), slots.tolist()


def test_a_held_page_that_is_none(ctx):
    table, lengths = ints([[4, -1, -1], [2, 3, -1]]), ints([20, 20])
    kv, positions, slots = plan(ctx, [2, 2], lengths, table, [0, 1], 2, 5)
    assert ctx.device_status() == 8, "its tokens would be taken for padding, and dropped"
    assert kv == [22, 22] and positions == [20, 21, 20, 21, 0] and slots == [-1, -1, 52, 53, -1]
    # pages behind the tokens of this step are not looked at
    table, lengths = ints([[-1, 5, -1]]), ints([20])
    assert plan(ctx, [2], lengths, table, [0, 1], 2, 2)[2] == [84, 85]
    assert ctx.device_status() == 0


def test_a_free_page_that_is_none(ctx):
    table, lengths = ints([[-1, -1], [-1, -1]]), ints([0, 0])
    assert plan(ctx, [1, 1], lengths, table, [7, -3, 6], 3, 2)[2] == [96, -1]
    assert ctx.device_status() == 8


def test_a_page_given_back_that_is_none(ctx):
    table, lengths, stack, count = ints([[4, -1, 9]]), ints([20]), ints([0, 0, 0]), ints([0])
    tk.PagePlanOp(ctx, 16).release(None, 1, None, lengths, lengths, table, stack, count, count)
    assert ctx.device_status() == 8 and count.tolist() == [2] and stack.tolist() == [4, -1, 0] and lengths.tolist() == [0]
    table, lengths, count = ints([[4, 9, -1]]), ints([32]), ints([0])
    tk.PagePlanOp(ctx, 16).release(None, 1, None, lengths, lengths, table, stack, count, count)
    assert ctx.device_status() == 0 and stack.tolist() == [4, 9, 0]
