"""Rotary positions, head norms and cache stores against their 64-bit form."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from gpu_util import SENTINEL, graph_replay, sentinel_plane

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def planes(tokens, q_heads, kv_heads, dim, gated, seed):
    """Views of a fused projection's rows: queries (each with its gate behind it), keys, values."""
    g = torch.Generator().manual_seed(seed)
    wide = 2 * dim if gated else dim
    plane = torch.randn(tokens, q_heads * wide + 2 * kv_heads * dim, generator=g).bfloat16().cuda()
    split = q_heads * wide
    return (plane[:, :split].view(tokens, q_heads, wide)[..., :dim],
            plane[:, split:split + kv_heads * dim].view(tokens, kv_heads, dim),
            plane[:, split + kv_heads * dim:].view(tokens, kv_heads, dim))


def check(actual, expected):
    """One rounding to BF16 (2^-8 of the value).  Before it fp32: the angle's remainder, sine and cosine are within
    2^-22, a norm's factor within 2^-20, two products and a sum add 2^-23 of their size: 2^-18 of the pair's size,
    which is below 16 in these planes (a normal value's 5.5, times sqrt 2, times a norm weight's 1.5)."""
    error = (ref.f64(actual) - expected).abs()
    assert bool((error <= 2.0 ** -8 * expected.abs() + 16 * 2.0 ** -18).all()), float(error.max())


@pytest.mark.parametrize("tokens", [1, 2, 7, 130])
@pytest.mark.parametrize("heads,rotary,axes", [((24, 4, 256), 64, 1), ((24, 4, 256), 256, 3), ((32, 8, 128), 128, 1),
                                               ((3, 1, 128), 16, 4), ((1, 1, 256), 48, 2), ((16, 16, 128), 64, 3)])
@pytest.mark.parametrize("norm,gated", [(False, False), (True, True)])
def test_rotation_and_store(ctx, tokens, heads, rotary, axes, norm, gated):
    q_heads, kv_heads, dim = heads
    query, key, value = planes(tokens, q_heads, kv_heads, dim, gated, tokens)
    g = torch.Generator().manual_seed(9)
    positions = torch.randint(0, 1 << 20, (axes, tokens), generator=g, dtype=torch.int32).cuda()
    frequencies = tk.rotary_frequencies(rotary, 1e7)
    pair_axes = (torch.arange(rotary // 2) % axes).to(torch.uint8).cuda() if axes > 1 else None
    weights = [torch.randn(dim, generator=g).mul(0.1).bfloat16().cuda() if norm else None for _ in range(2)]
    page, pages = 16, tokens // 16 + 3
    slots = torch.randperm(page * pages, generator=g)[:tokens].cuda()
    if tokens > 4:
        slots[3] = -1
    caches = [sentinel_plane((pages, page, kv_heads, dim), torch.bfloat16) for _ in range(2)]
    q_out, k_out = (sentinel_plane((tokens + 1, h, dim), torch.bfloat16) for h in (q_heads, kv_heads))
    op = tk.RotaryCacheOp(ctx, q_heads, kv_heads, dim, frequencies, pair_axes)
    op.launch(None, tokens, positions, query, key, value, *weights, q_out, k_out, *caches, slots)
    assert ctx.device_status() == 0
    check(q_out[:tokens], ref.rotate(query, positions, frequencies, pair_axes, weights[0]))
    check(k_out[:tokens], ref.rotate(key, positions, frequencies, pair_axes, weights[1]))
    for t in (q_out, k_out):
        assert bool((t[tokens:].view(torch.uint8) == SENTINEL).all())
    stored = slots >= 0
    flat = [c.view(-1, kv_heads, dim) for c in caches]
    assert torch.equal(flat[0][slots[stored]], k_out[:tokens][stored]) and torch.equal(flat[1][slots[stored]], value[stored])
    others = torch.ones(page * pages, dtype=torch.bool, device="cuda")
    others[slots[stored]] = False
    for c in flat:
        assert bool((c[others].view(torch.uint8) == SENTINEL).all()), "slots of no token were written"


@pytest.mark.parametrize("order", ["head", "pair"])
def test_cache_orders_without_key_output(ctx, order):
    q_heads, kv_heads, dim, page, pages, tokens = 6, 2, 128, 32, 4, 50
    query, key, value = planes(tokens, q_heads, kv_heads, dim, False, 1)
    if order == "head":
        caches = [torch.zeros(pages, kv_heads, page, dim, dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3) for _ in range(2)]
    else:
        both = torch.zeros(pages, page, kv_heads, 2, dim, dtype=torch.bfloat16, device="cuda")
        caches = [both[:, :, :, 0], both[:, :, :, 1]]
    slots = torch.randperm(page * pages)[:tokens].cuda()
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    frequencies = tk.rotary_frequencies(dim, 1e4)
    q_out = torch.zeros(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.RotaryCacheOp(ctx, q_heads, kv_heads, dim, frequencies)
    op.launch(None, tokens, positions, query, key, value, None, None, q_out, None, *caches, slots)
    got = [c[slots // page, slots % page] for c in caches]
    check(got[0], ref.rotate(key, positions[None], frequencies, None))
    assert torch.equal(got[1], value)
    assert float(caches[0].float().abs().sum((2, 3)).count_nonzero()) == tokens


@pytest.mark.parametrize("position", [0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1])
def test_far_positions(ctx, position):
    """The turns position * frequency / 2 pi are formed in double: below 2^29 turns 2^-24 of a turn are kept."""
    query, key, value = planes(1, 2, 1, 128, False, 3)
    positions = torch.tensor([position], dtype=torch.int32, device="cuda")
    frequencies = tk.rotary_frequencies(128, 1e4)
    q_out, k_out = (torch.zeros(1, h, 128, dtype=torch.bfloat16, device="cuda") for h in (2, 1))
    tk.RotaryCacheOp(ctx, 2, 1, 128, frequencies).launch(None, 1, positions, query, key, None, None, None, q_out, k_out,
                                                         None, None, None)
    check(q_out, ref.rotate(query, positions[None], frequencies, None))
    check(k_out, ref.rotate(key, positions[None], frequencies, None))


def test_in_place_and_replay(ctx):
    tokens, dim = 33, 256
    g = torch.Generator().manual_seed(2)
    query, key = (torch.randn(tokens, h, dim, generator=g).bfloat16().cuda() for h in (6, 2))
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    frequencies = tk.rotary_frequencies(64, 1e7)
    op = tk.RotaryCacheOp(ctx, 6, 2, dim, frequencies)
    expected = [ref.rotate(t, positions[None], frequencies, None) for t in (query, key)]
    fresh = [torch.zeros_like(t) for t in (query, key)]

    def step():
        op.launch(None, tokens, positions, query, key, None, None, None, fresh[0], fresh[1], None, None, None)

    graph = graph_replay(step)
    for t in fresh:
        t.zero_()
    graph.replay()
    op.launch(None, tokens, positions, query, key, None, None, None, query, key, None, None, None)
    for t, o, e in zip((query, key), fresh, expected):
        check(o, e)
        assert torch.equal(t, o)


def test_values_that_are_no_numbers_stay_in_their_pair(ctx):
    query, key, _ = planes(1, 1, 1, 128, False, 4)
    query = query.clone()
    query[0, 0, 100] = float("nan")
    query[0, 0, 5] = float("inf")
    positions = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out, k_out = (torch.zeros(1, 1, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tk.RotaryCacheOp(ctx, 1, 1, 128, tk.rotary_frequencies(32, 1e4)).launch(
        None, 1, positions, query, key, None, None, None, q_out, k_out, None, None, None)
    bad = ~torch.isfinite(q_out[0, 0])
    assert bad.nonzero().flatten().tolist() == [5, 21, 100]


def test_pair_axes_layouts():
    assert tk.rotary_pair_axes((3, 2, 2), device="cpu").tolist() == [0, 0, 0, 1, 1, 2, 2]
    assert tk.rotary_pair_axes((4, 2, 2), True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    with pytest.raises(ValueError):
        tk.rotary_pair_axes((1, 5, 1), True, device="cpu")


def test_refusals_and_reports(ctx):
    tokens, dim = 4, 128
    query, key, value = planes(tokens, 2, 1, dim, False, 5)
    cache = [torch.zeros(2, 16, 1, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    frequencies = tk.rotary_frequencies(64, 1e4)
    q_out = torch.zeros(tokens, 2, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.RotaryCacheOp(ctx, 2, 1, dim, frequencies)
    base = dict(tokens=tokens, positions=torch.arange(tokens, dtype=torch.int32, device="cuda"), query=query, key=key,
                value=value, query_norm=None, key_norm=None, query_output=q_out, key_output=None, key_cache=cache[0],
                value_cache=cache[1], slots=torch.arange(tokens, device="cuda"))

    def refused(text, operator=op, **change):
        with pytest.raises(tk.GpuError, match=text):
            operator.launch(None, **{**base, **change})

    refused("token count", tokens=0, positions=base["positions"][:0])
    refused("fewer than", tokens=5, positions=torch.zeros(5, dtype=torch.int32, device="cuda"))
    refused("positions", positions=base["positions"][:3])
    refused("positions", positions=base["positions"].long())
    refused("go together", slots=None)
    refused("go together", value_cache=None)
    refused("nowhere", key_cache=None, value_cache=None)
    refused("slots", slots=base["slots"].int())
    refused("query output", query_output=q_out[:3])
    refused("query output overlaps the queries", query_output=query.as_strided((tokens, 2, dim), (2 * dim, dim, 1)))
    refused("query norm", query_norm=torch.zeros(64, dtype=torch.bfloat16, device="cuda"))
    refused("different strides", value=value.contiguous())
    refused("rotated values", operator=tk.RotaryCacheOp(ctx, 2, 1, dim, tk.rotary_frequencies(24, 1e4)))
    refused("rotated values", operator=tk.RotaryCacheOp(ctx, 2, 1, dim, tk.rotary_frequencies(256, 1e4)))
    refused("axis count", positions=torch.zeros(9, tokens, dtype=torch.int32, device="cuda"))
    # reported, not fatal: a slot behind the last page, an axis without positions
    op.launch(None, **{**base, "slots": torch.tensor([0, 1, 2, 32], device="cuda")})
    assert ctx.device_status() == 8
    far = tk.RotaryCacheOp(ctx, 2, 1, dim, frequencies, torch.full((32,), 3, dtype=torch.uint8, device="cuda"))
    far.launch(None, **base)
    assert ctx.device_status() == 8
    op.launch(None, **base)
    assert ctx.device_status() == 0
