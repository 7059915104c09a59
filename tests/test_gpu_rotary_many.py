"""Rotary positions of thousands of tokens, where a CTA may have four of them, against their 64-bit form."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from gpu_util import SENTINEL, graph_replay, sentinel_plane
from test_gpu_rotary import check, planes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


# Up to 2047 tokens a CTA has one; from then on four (whole CTAs, one to three tokens in the last) where the heads of
# queries, keys and values are one round of a CTA's at most, 64 of 128 values or 32 of 256, with norms half of one.
@pytest.mark.parametrize("tokens", [1027, 2047, 2048, 2049, 2050, 2051])
@pytest.mark.parametrize("heads,rotary,axes", [((24, 4, 256), 64, 3), ((48, 8, 128), 128, 1), ((56, 8, 128), 64, 1), ((3, 1, 128), 48, 2),
                                               ((12, 2, 256), 128, 3), ((16, 8, 128), 16, 1), ((40, 2, 256), 256, 1)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_and_store(ctx, tokens, heads, rotary, axes, norm):
    q_heads, kv_heads, dim = heads
    query, key, value = planes(tokens, q_heads, kv_heads, dim, norm, tokens)
    g = torch.Generator().manual_seed(9)
    positions = torch.randint(0, 1 << 20, (axes, tokens), generator=g, dtype=torch.int32).cuda()
    frequencies = tk.rotary_frequencies(rotary, 1e7)
    pair_axes = (torch.arange(rotary // 2) % axes).to(torch.uint8).cuda() if axes > 1 else None
    weights = [torch.randn(dim, generator=g).mul(0.1).bfloat16().cuda() if norm else None for _ in range(2)]
    page, pages = 64, tokens // 64 + 3
    slots = torch.randperm(page * pages, generator=g)[:tokens].cuda()
    slots[5], slots[tokens - 1], slots[tokens - 3] = -1, -1, -1
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


@pytest.mark.parametrize("heads", [(6, 2, 256), (30, 2, 128), (72, 2, 128)])
def test_in_place_and_replay(ctx, heads):
    q_heads, kv_heads, dim = heads
    tokens = 2501
    g = torch.Generator().manual_seed(2)
    query, key = (torch.randn(tokens, h, dim, generator=g).bfloat16().cuda() for h in (q_heads, kv_heads))
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda")
    frequencies = tk.rotary_frequencies(64, 1e7)
    op = tk.RotaryCacheOp(ctx, q_heads, kv_heads, dim, frequencies)
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


def test_one_and_four_tokens_a_cta_agree(ctx):
    """A token's result does not depend on how many others are rotated with it."""
    tokens, heads, dim = 2060, (14, 2), 256
    query, key, value = planes(tokens, *heads, dim, True, 4)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") * 177
    op = tk.RotaryCacheOp(ctx, *heads, dim, tk.rotary_frequencies(64, 1e7))
    weights = [torch.randn(dim, generator=torch.Generator().manual_seed(s)).mul(0.1).bfloat16().cuda() for s in (1, 2)]
    whole = [torch.zeros(tokens, h, dim, dtype=torch.bfloat16, device="cuda") for h in heads]
    op.launch(None, tokens, positions, query, key, None, *weights, *whole, None, None, None)
    part = [torch.zeros_like(t) for t in whole]
    for a in range(0, tokens, 515):
        op.launch(None, 515, positions[a:a + 515], query[a:a + 515], key[a:a + 515], None, *weights, part[0][a:a + 515],
                  part[1][a:a + 515], None, None, None)
    assert torch.equal(whole[0], part[0]) and torch.equal(whole[1], part[1])
