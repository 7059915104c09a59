"""Tiles that many pairs of CTAs share, against the 64-bit form: what the parts leave, and their join."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from test_gpu_attention import run_paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128), (6, 1, 256), (1, 1, 128)])
@pytest.mark.parametrize("keys", [1500, 4097, 16001])
def test_one_token(ctx, keys, heads, gated):
    """Six rows and fewer in 12 to 74 parts."""
    run_paged(ctx, [1], [keys - 1], heads, gated=gated)


@pytest.mark.parametrize("heads,keys", [((24, 4, 256), 16001), ((6, 1, 256), 8001), ((8, 2, 128), 9000), ((64, 1, 128), 12000)])
@pytest.mark.parametrize("new", [9, 21, 32, 64])
def test_short_chunks_over_long_caches(ctx, new, heads, keys):
    """Tiles of 36 rows to 128 in each CTA of a pair, in five parts to sixty-one."""
    run_paged(ctx, [new], [keys - new], heads, gated=new == 32)


@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128)])
def test_long_sequences_among_many(ctx, heads):
    """More sequences than a warp has lanes, a few of them split, in front, between and behind the short ones."""
    new = [1] * 20 + [50] + [1] * 20 + [0, 3, 1]
    cached = [9000] + [5 * i for i in range(19)] + [7000] + [100 + i for i in range(20)] + [10, 4, 12000]
    run_paged(ctx, new, cached, heads)
    run_paged(ctx, [1] * 600 + [30], [i % 9 for i in range(600)] + [20000], heads, 16)


def test_parts_are_joined_in_one_order(ctx):
    """The same bits whoever joins: twenty launches of a step with tiles in many parts, of few rows and of many."""
    for new, keys in (([1, 1], [16000, 3000]), ([32], [16001])):
        cache = ref.Paged(keys, 4, 256, 64, 3)
        query = torch.randn(sum(new), 24, 256, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
        op = tk.PagedAttentionOp(ctx, 24, 4, 256)
        work, first = op.workspace(), None
        starts, kv = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (ref.starts_of(new), keys))
        for _ in range(20):
            out = torch.zeros_like(query)
            op.launch(None, len(new), starts, kv, query, None, cache.key, cache.value, cache.table, None, work, out)
            first = out if first is None else first
            assert torch.equal(out, first)
        expected, size = ref.attention(query, cache.keys, cache.values, ref.starts_of(new), op.scale)
        assert bool(((ref.f64(first) - expected).abs() <= ref.attention_tolerance(expected, size)).all())
    assert ctx.device_status() == 0
