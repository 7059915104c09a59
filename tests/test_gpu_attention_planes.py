"""Planes that the full-attention operators take, and those that they refuse: shapes, overlaps, positions."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def zeros(*shape):
    return torch.zeros(*shape, dtype=BF16, device="cuda")


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


class Calls:
    """One call of each operator that writes rows of heads, whose planes can be replaced."""

    def __init__(self, ctx, tokens=5, q_heads=6, kv_heads=2, dim=128):
        self.cache = ref.Paged([40], kv_heads, dim, 16, 3)
        self.query = normal(1, tokens, q_heads, dim)
        self.key, self.value = normal(2, tokens, kv_heads, dim), normal(3, tokens, kv_heads, dim)
        self.q_out, self.k_out = zeros(tokens, q_heads, dim), zeros(tokens, kv_heads, dim)
        self.paged_op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim)
        self.prompt_op = tk.PromptAttentionOp(ctx, q_heads, kv_heads, dim)
        self.rotary_op = tk.RotaryCacheOp(ctx, q_heads, kv_heads, dim, tk.rotary_frequencies(64, 1e4))
        self.work, self.starts = self.paged_op.workspace(), ints([0, tokens])
        self.paged_base = dict(sequences=1, starts=self.starts, kv_lengths=ints([40]), query=self.query, gate=None,
                               key_cache=self.cache.key, value_cache=self.cache.value, block_table=self.cache.table,
                               request_rows=None, workspace=self.work, output=self.q_out)
        self.prompt_base = dict(sequences=1, starts=self.starts, query=self.query, gate=None, key=self.key, value=self.value,
                                workspace=self.work, output=self.q_out)
        self.rotary_base = dict(tokens=tokens, positions=torch.arange(tokens, dtype=torch.int32, device="cuda"),
                                query=self.query, key=self.key, value=self.value, query_norm=None, key_norm=None,
                                query_output=self.q_out, key_output=self.k_out, key_cache=zeros(2, 16, kv_heads, dim),
                                value_cache=zeros(2, 16, kv_heads, dim), slots=torch.arange(tokens, device="cuda"))

    def paged(self, **change):
        self.paged_op.launch(None, **{**self.paged_base, **change})

    def prompt(self, **change):
        self.prompt_op.launch(None, **{**self.prompt_base, **change})

    def rotary(self, **change):
        self.rotary_op.launch(None, **{**self.rotary_base, **change})


@pytest.fixture(scope="module")
def calls(ctx):
    return Calls(ctx)


def test_outputs_of_another_order_are_refused(ctx, calls):
    """An output whose heads do not lie behind one another in a token's row would be filled in another order."""
    for other in (zeros(6, 5, 128), zeros(128, 6, 5), zeros(768, 5), zeros(6, 640)):
        for call, name in ((calls.paged, "output"), (calls.prompt, "output"), (calls.rotary, "query_output")):
            with pytest.raises(tk.GpuError, match=name.replace("_", " ")):
                call(**{name: other})
    with pytest.raises(tk.GpuError, match="key output"):
        calls.rotary(key_output=zeros(2, 5, 128))
    assert ctx.device_status() == 0


def test_outputs_in_rows_of_any_shape(ctx, calls):
    """Planes with the rows' order: flat, a row a token, heads in groups, more rows than tokens."""
    for call, name in ((calls.paged, "output"), (calls.prompt, "output"), (calls.rotary, "query_output")):
        first = zeros(5, 6, 128)
        call(**{name: first})
        assert float(first.float().abs().sum()) > 0
        for shape in ((5, 768), (5 * 768,), (30, 128), (1, 5, 6, 128), (5, 1, 768), (5, 2, 3, 128), (7, 6, 128)):
            out = zeros(*shape)
            call(**{name: out})
            assert torch.equal(out.view(-1)[:5 * 768], first.view(-1)), (name, shape)
            assert float(out.view(-1)[5 * 768:].float().abs().sum()) == 0
    assert ctx.device_status() == 0


def test_positions_are_axes_by_tokens(ctx, calls):
    query = ref.f64(calls.query)
    positions = torch.arange(5, dtype=torch.int32, device="cuda") * 7
    expected = ref.rotate(query, positions[None], calls.rotary_op.frequencies, None)
    for shape in ((5,), (1, 5), (1, 1, 5)):
        calls.rotary(positions=positions.view(shape))
        assert bool(((ref.f64(calls.q_out) - expected).abs() <= 2.0 ** -8 * expected.abs() + 16 * 2.0 ** -18).all())
    op = tk.RotaryCacheOp(ctx, 6, 2, 128, tk.rotary_frequencies(64, 1e4), torch.tensor([0, 1, 2, 1] * 8, dtype=torch.uint8).cuda())
    axes = torch.stack([positions, positions * 2, positions + 3])
    expected = ref.rotate(query, axes, op.frequencies, op.pair_axes)
    for shape in ((3, 5), (3, 1, 5)):
        op.launch(None, **{**calls.rotary_base, "positions": axes.view(shape)})
        assert bool(((ref.f64(calls.q_out) - expected).abs() <= 2.0 ** -8 * expected.abs() + 16 * 2.0 ** -18).all())
    assert ctx.device_status() == 0
    for other in (axes.view(1, 3, 5), axes[:2].view(1, 2, 5), axes.t().contiguous(), torch.tensor(3, dtype=torch.int32, device="cuda"),
                  torch.zeros(0, 5, dtype=torch.int32, device="cuda")):
        with pytest.raises(tk.GpuError, match="position"):
            op.launch(None, **{**calls.rotary_base, "positions": other})


def test_what_is_no_tensor_is_refused(ctx, calls):
    """With the operators' error, whichever plane it is."""
    for change in (dict(block_table=None), dict(block_table=7), dict(output=None), dict(query=None), dict(key_cache=None),
                   dict(starts=None), dict(workspace=None), dict(kv_lengths=[40])):
        with pytest.raises(tk.GpuError):
            calls.paged(**change)
    for change in (dict(positions=None), dict(positions=[0, 1, 2, 3, 4]), dict(slots=3), dict(query_output=None), dict(key=None)):
        with pytest.raises(tk.GpuError):
            calls.rotary(**change)
    for change in (dict(frequencies=None), dict(frequencies=[1.0] * 32)):
        with pytest.raises(tk.GpuError, match="frequencies"):
            tk.RotaryCacheOp(ctx, 6, 2, 128, **change)
    plan = dict(requests=1, request_rows=None, new_tokens=ints([1]), lengths=ints([0]), lengths_output=ints([0]),
                block_table=ints([[0, 0]]), free_pages=ints([0, 1]), free_count=ints([2]), free_count_output=ints([0]),
                starts=ints([0, 0]), kv_lengths=ints([0]), positions=ints([0]), slots=ints([0], torch.int64))
    op = tk.PagePlanOp(ctx, 16)
    for name in plan:
        if name in ("requests", "request_rows"):
            continue
        for other in (None, 3, [0, 0]):
            with pytest.raises(tk.GpuError):
                op.launch(None, **{**plan, name: other})
    op.launch(None, **plan)
    assert ctx.device_status() == 0


def test_overlaps_are_refused(ctx, calls):
    def refused(call, text, **change):
        with pytest.raises(tk.GpuError, match=text):
            call(**change)

    # caches over rows that other CTAs still read, or over the outputs
    pool = zeros(2 * 16 * 2 * 128 + 5 * 768)
    cache, rows = pool[:2 * 16 * 2 * 128].view(2, 16, 2, 128), pool[2 * 16 * 2 * 128 - 512:][:5 * 768].view(5, 6, 128)
    kv_rows = pool[512:][:5 * 256].view(5, 2, 128)
    for name in ("key_cache", "value_cache"):
        refused(calls.rotary, "cache overlaps the queries", query=rows, **{name: cache})
        refused(calls.rotary, "cache overlaps the query output", query_output=rows, **{name: cache})
        refused(calls.rotary, "cache overlaps the keys", key=kv_rows, **{name: cache})
        refused(calls.rotary, "cache overlaps the values", value=kv_rows, **{name: cache})
        refused(calls.rotary, "cache overlaps the key output", key_output=kv_rows, **{name: cache})
        apart = dict(key_cache=zeros(2, 16, 2, 128), value_cache=zeros(2, 16, 2, 128))
        refused(calls.paged, "output overlaps the key or value cache", output=rows, **{**apart, name: cache})
    # one plane for both caches, and planes that share some of their values
    refused(calls.rotary, "key cache overlaps the value cache", key_cache=cache, value_cache=cache)
    both = zeros(2, 16, 2, 192)
    refused(calls.rotary, "key cache overlaps the value cache", key_cache=both[..., :128], value_cache=both[..., 64:])
    shifted = zeros(3, 16, 2, 128)
    refused(calls.rotary, "key cache overlaps the value cache", key_cache=shifted[:2], value_cache=shifted[1:])
    assert ctx.device_status() == 0


@pytest.mark.parametrize("order", ["heads", "tokens", "pages", "page heads"])
def test_caches_in_one_plane_are_taken(ctx, calls, order):
    """Keys and values in turn: next to each other in a head, a token or a page, and in a page of [heads, tokens]."""
    both = {"heads": zeros(2, 16, 2, 2, 128), "tokens": zeros(2, 16, 2, 2, 128), "pages": zeros(2, 2, 16, 2, 128),
            "page heads": zeros(2, 2, 2, 16, 128)}[order]
    pick = {"heads": lambda i: both[:, :, :, i], "tokens": lambda i: both[:, :, i], "pages": lambda i: both[:, i],
            "page heads": lambda i: both[:, i].transpose(1, 2)}[order]
    calls.rotary(key_cache=pick(0), value_cache=pick(1))
    assert ctx.device_status() == 0
    assert torch.equal(pick(0)[0, :5], calls.k_out) and torch.equal(pick(1)[0, :5], calls.value)
    assert int(both.count_nonzero()) == int(calls.k_out.count_nonzero()) + int(calls.value.count_nonzero())


def test_a_value_that_is_no_number_reaches_its_tile_at_most(ctx):
    """It reaches the tokens that see it, and no token more than 2 * floor(128 / queries of a key/value head) - 1 in front
    of it; a key that is none no token in front of it at all."""
    for q_heads, reach in ((1, 255), (6, 41)):
        tokens, at = 700, 511
        query, key, value = normal(1, tokens, q_heads, 128), normal(2, tokens, 1, 128), normal(3, tokens, 1, 128)
        op = tk.PromptAttentionOp(ctx, q_heads, 1, 128)
        clean, out, work = torch.zeros_like(query), torch.zeros_like(query), op.workspace()
        op.launch(None, 1, ints([0, tokens]), query, None, key, value, work, clean)
        broken = value.clone()
        broken[at] = float("nan")
        op.launch(None, 1, ints([0, tokens]), query, None, key, broken, work, out)
        assert bool(out[at:].isnan().all()) and torch.equal(out[:at - reach], clean[:at - reach])
        broken = key.clone()
        broken[at] = float("nan")
        op.launch(None, 1, ints([0, tokens]), query, None, broken, value, work, out)
        assert bool(out[at:].isnan().all()) and torch.equal(out[:at], clean[:at])
    assert ctx.device_status() == 0
