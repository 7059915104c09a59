"""Attention over paged caches and packed prompts against its 64-bit form."""
import pytest
import torch

import tuiskollm_b200 as tk
import attention_ref as ref
from gpu_util import graph_replay, sentinel_plane, SENTINEL

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def queries(tokens, heads, dim, seed, gated=False):
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(tokens, heads, 2 * dim if gated else dim, generator=g).bfloat16().cuda()
    return wide[..., :dim], wide[..., dim:] if gated else None


def check(output, expected, size, gated=False):
    error = (ref.f64(output) - expected).abs()
    bad = ~(error <= ref.attention_tolerance(expected, size, gated))
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(error[bad].max()), bad.nonzero()[:4].tolist())


def run_paged(ctx, new, cached, heads=(24, 4, 256), page=64, gated=False, order="token", tail=3, seed=0, scale=None):
    q_heads, kv_heads, dim = heads
    kv = [max(0, a + b) for a, b in zip(new, cached)]
    cache = ref.Paged(kv, kv_heads, dim, page, seed, order=order)
    total, starts = sum(new), ref.starts_of(new)
    query, gate = queries(total + tail, q_heads, dim, seed + 1, gated)
    output = sentinel_plane((total + tail, q_heads, dim), torch.bfloat16)
    op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim, scale)
    work = op.workspace()
    op.launch(None, len(new), ints(starts), ints(kv), query, gate, cache.key, cache.value, cache.table, None, work, output)
    assert ctx.device_status() == 0
    expected, size = ref.attention(query[:total], cache.keys, cache.values, starts, op.scale,
                                   None if gate is None else gate[:total])
    check(output[:total], expected, size, gated)
    assert bool((output[total:].view(torch.uint8) == SENTINEL).all()), "rows behind the last sequence were written"
    assert int(work[:4096].view(torch.int32).abs().sum()) == 0, "tickets were left behind"
    return output[:total]


@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 255, 257, 1000])
def test_one_token_over_a_cache(ctx, kv):
    run_paged(ctx, [1], [kv - 1])


@pytest.mark.parametrize("heads", [(24, 4, 256), (32, 8, 128), (16, 16, 128), (8, 1, 256), (1, 1, 128), (5, 5, 256),
                                   (128, 1, 128), (48, 1, 256)])
def test_head_layouts(ctx, heads):
    run_paged(ctx, [1, 5, 40], [300, 129, 0], heads)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128)])
def test_page_sizes(ctx, heads, page):
    run_paged(ctx, [1, 3, 150], [500, 17, 77], heads, page)


@pytest.mark.parametrize("order", ["head", "pair"])
@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128)])
def test_cache_orders(ctx, heads, order):
    run_paged(ctx, [1, 30, 2], [500, 17, 126], heads, 32, order=order)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("new,cached", [([300], [0]), ([300], [1000]), ([1] * 32, list(range(0, 3200, 100))),
                                        ([7, 1, 64, 1, 22, 21, 43], [0, 4000, 100, 0, 64, 2000, 1])])
def test_chunks(ctx, new, cached, gated):
    run_paged(ctx, new, cached, gated=gated)


def test_sequences_without_tokens_or_keys(ctx):
    # no new tokens; more new tokens than keys (the first see nothing); no keys at all
    run_paged(ctx, [0, 3, 0, 40, 2, 0], [100, 64, 0, -30, -2, 5])


def test_many_sequences(ctx):
    new = [1 if i % 3 else i % 7 for i in range(700)]
    run_paged(ctx, new, [i % 50 for i in range(700)], (2, 1, 128), 16)


@pytest.mark.parametrize("scale", [1e-6, 0.0625, 0.5])
def test_scales(ctx, scale):
    """(At 0.5 the bound on a score's error is 128 * 2^-24 * 128 * 0.64 * 0.5 = 3.1e-4, within the tolerance's 2^-10.)"""
    run_paged(ctx, [20, 1], [313, 1000], (6, 2, 128), 32, scale=scale)


@pytest.mark.parametrize("rising", [False, True])
def test_growing_maxima(ctx, rising):
    """Scores that rise (or fall) over hundreds of units: every step moves the reference maximum, and weights of early
    keys vanish.  Keys are +-k * direction with one query along it: scores are exact in fp32 up to 2^-24 of 300, so
    the tolerance holds."""
    dim, n = 256, 1500
    cache = ref.Paged([n], 1, dim, 64, 7)
    ramp = torch.linspace(0, 300, n).bfloat16().float()
    if not rising:
        ramp = ramp.flip(0)
    key = torch.zeros(n, 1, dim)
    key[:, 0, 0] = ramp
    cache.keys[0] = key
    flat = cache.key.float().cpu()
    for j in range(cache.table.shape[1]):
        part = key[64 * j:64 * j + 64]
        flat[int(cache.table[0, j]), :part.shape[0]] = part
    cache.key = flat.bfloat16().cuda()
    query = torch.zeros(40, 3, dim, dtype=torch.bfloat16, device="cuda")
    query[..., 0] = 1.0
    output = torch.zeros(40, 3, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.PagedAttentionOp(ctx, 3, 1, dim, 1.0)
    op.launch(None, 1, ints([0, 40]), ints([n]), query, None, cache.key, cache.value, cache.table, None, op.workspace(), output)
    check(output, *ref.attention(query, cache.keys, cache.values, [0, 40], 1.0))


def run_prompt(ctx, lengths, heads=(24, 4, 256), gated=False, plane=False, seed=0, tail=2):
    q_heads, kv_heads, dim = heads
    total, starts = sum(lengths), ref.starts_of(lengths)
    query, gate = queries(total + tail, q_heads, dim, seed, gated)
    g = torch.Generator().manual_seed(seed + 1)
    both = torch.randn(total + tail, 2, kv_heads, dim, generator=g).bfloat16().cuda()
    key, value = (both[:, 0], both[:, 1]) if plane else (both[:, 0].contiguous(), both[:, 1].contiguous())
    output = sentinel_plane((total + tail, q_heads, dim), torch.bfloat16)
    op = tk.PromptAttentionOp(ctx, q_heads, kv_heads, dim)
    op.launch(None, len(lengths), ints(starts), query, gate, key, value, op.workspace(), output)
    assert ctx.device_status() == 0
    split = [(starts[i], starts[i + 1]) for i in range(len(lengths))]
    expected, size = ref.attention(query[:total], [key[a:b] for a, b in split], [value[a:b] for a, b in split], starts,
                                   op.scale, None if gate is None else gate[:total])
    check(output[:total], expected, size, gated)
    assert bool((output[total:].view(torch.uint8) == SENTINEL).all())


@pytest.mark.parametrize("length", [1, 2, 20, 21, 22, 42, 43, 127, 128, 129, 301])
def test_one_prompt(ctx, length):
    run_prompt(ctx, [length])


@pytest.mark.parametrize("heads", [(24, 4, 256), (32, 8, 128), (3, 3, 128), (64, 1, 256)])
@pytest.mark.parametrize("gated,plane", [(False, False), (True, True)])
def test_packed_prompts(ctx, heads, gated, plane):
    run_prompt(ctx, [3, 0, 130, 1, 257, 64], heads, gated, plane)


def test_launches_repeat_bit_for_bit_and_replay(ctx):
    """Split tiles are joined in the order of their keys whoever is last, and lengths are read from the device: a
    captured launch follows them."""
    q_heads, kv_heads, dim, page = 24, 4, 256, 64
    cache = ref.Paged([3000, 700, 90], kv_heads, dim, page, 3)
    query, _ = queries(3, q_heads, dim, 4)
    output = torch.zeros(3, q_heads, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim)
    work, kv, starts = op.workspace(), ints([3000, 700, 90]), ints([0, 1, 2, 3])

    def step():
        op.launch(None, 3, starts, kv, query, None, cache.key, cache.value, cache.table, None, work, output)

    step()
    first = output.clone()
    for _ in range(20):
        output.zero_()
        step()
        assert torch.equal(output, first)
    graph = graph_replay(step)
    output.zero_()
    graph.replay()
    assert torch.equal(output, first)
    kv.copy_(ints([1500, 699, 2]))
    graph.replay()
    step_keys = [cache.keys[0][:1500], cache.keys[1][:699], cache.keys[2][:2]]
    step_values = [cache.values[0][:1500], cache.values[1][:699], cache.values[2][:2]]
    check(output, *ref.attention(query, step_keys, step_values, [0, 1, 2, 3], op.scale))


def test_request_rows_and_bad_pages(ctx):
    q_heads, kv_heads, dim, page = 6, 2, 128, 16
    cache = ref.Paged([100, 60, 80], kv_heads, dim, page, 3)
    query, _ = queries(2, q_heads, dim, 4)
    output = torch.zeros(2, q_heads, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim)
    work = op.workspace()
    op.launch(None, 2, ints([0, 1, 2]), ints([80, 100]), query, None, cache.key, cache.value, cache.table, ints([2, 0]), work, output)
    assert ctx.device_status() == 0
    check(output, *ref.attention(query, [cache.keys[2], cache.keys[0]], [cache.values[2], cache.values[0]], [0, 1, 2], op.scale))
    # pages outside the cache, a row outside the table and lengths beyond it read as zeros or are cut, and are reported
    table = cache.table.clone()
    table[0, 2] = 10 ** 6
    keys, values = cache.keys[0].clone(), cache.values[0].clone()
    keys[32:48], values[32:48] = 0, 0
    op.launch(None, 1, ints([0, 1]), ints([100]), query, None, cache.key, cache.value, table, None, work, output)
    assert ctx.device_status() == 8
    check(output[:1], *ref.attention(query[:1], [keys], [values], [0, 1], op.scale))
    op.launch(None, 1, ints([0, 1]), ints([100]), query, None, cache.key, cache.value, cache.table, ints([5]), work, output)
    assert ctx.device_status() == 8 and float(output[0].abs().max()) == 0.0
    op.launch(None, 1, ints([0, 5]), ints([10 ** 9]), query, None, cache.key, cache.value, cache.table, None, work, output)
    assert ctx.device_status() == 8


def test_refusals(ctx):
    q_heads, kv_heads, dim, page = 6, 2, 128, 16
    cache = ref.Paged([40], kv_heads, dim, page, 3)
    query, _ = queries(1, q_heads, dim, 4)
    output = torch.zeros(1, q_heads, dim, dtype=torch.bfloat16, device="cuda")
    op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim)
    base = dict(sequences=1, starts=ints([0, 1]), kv_lengths=ints([40]), query=query, gate=None, key_cache=cache.key,
                value_cache=cache.value, block_table=cache.table, request_rows=None, workspace=op.workspace(), output=output)

    def refused(text, operator=op, **change):
        with pytest.raises(tk.GpuError, match=text):
            operator.launch(None, **{**base, **change})

    refused("sequence count", sequences=0)
    refused("fewer rows", sequences=2, starts=ints([0, 1, 1]), kv_lengths=ints([40, 0]))
    refused("starts", starts=ints([0]))
    refused("starts", starts=ints([0, 1], torch.int64))
    refused("key lengths", kv_lengths=torch.tensor([40], dtype=torch.int32))
    refused("query", query=query.half())
    refused("query", query=query[:, :5])
    refused("next to each other", query=query.transpose(1, 2).contiguous().transpose(1, 2))
    refused("gate", gate=query[:, :, :64])
    refused("different strides", value_cache=cache.value.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    refused("power of two", key_cache=cache.key[:, :12], value_cache=cache.value[:, :12])
    refused("multiple of 8", key_cache=torch.zeros(2, 16, 2, 129, dtype=torch.bfloat16, device="cuda")[..., :128],
            value_cache=torch.zeros(2, 16, 2, 129, dtype=torch.bfloat16, device="cuda")[..., :128])
    refused("aligned", query=torch.zeros(6 * 128 + 8, dtype=torch.bfloat16, device="cuda")[4:6 * 128 + 4].view(1, 6, 128))
    refused("overlaps", output=query)
    refused("workspace", workspace=base["workspace"][:4096])
    refused("block table", block_table=cache.table[0])
    refused("scale", operator=tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim, -1.0))
    refused("scale", operator=tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim, float("nan")))
    wide = dict(key_cache=torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), query=query[..., :64].contiguous(),
                output=output[..., :64].contiguous())
    refused("64 values", operator=tk.PagedAttentionOp(ctx, q_heads, kv_heads, 64), value_cache=wide["key_cache"], **wide)
    uneven = tk.PagedAttentionOp(ctx, 6, 4, dim)
    refused("evenly", operator=uneven, key_cache=torch.zeros(2, 16, 4, dim, dtype=torch.bfloat16, device="cuda"),
            value_cache=torch.zeros(2, 16, 4, dim, dtype=torch.bfloat16, device="cuda"))
    op.launch(None, **base)
    assert ctx.device_status() == 0
