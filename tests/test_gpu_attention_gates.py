"""Gated attention rows of every magnitude, and gates that lie where the projection left them."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk

pytestmark = pytest.mark.gpu

HEADS = [(24, 4, 256), (8, 2, 128)]


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def tolerance(out, size, keys):
    """The weights are rounded to BF16 (2^-8 of `size`), the result is (2^-8 of it), a row that waits for its gate to FP16
    (2^-11 of the result); what fp32 does to scores and sums stays below 2^-10 of `size` (as in attention_ref).  All of it is
    relative to the value itself, whatever the row's others are.  A product or a sum below the smallest normal number,
    2^-126, may count as zero: one a key, and the result."""
    return (2.0 ** -8 + 2.0 ** -10) * size + (2.0 ** -8 + 2.0 ** -11) * out.abs() + (keys + 2) * 2.0 ** -126


def set_values(cache, values, page):
    """Gives the cache's only sequence other values, in the plane too."""
    cache.values[0] = values.bfloat16().float()
    plane = cache.value.cpu()
    for j in range(cache.table.shape[1]):
        part = cache.values[0][j * page:(j + 1) * page].bfloat16()
        plane[int(cache.table[0, j]), :part.shape[0]] = part
    cache.value = plane.cuda()


def run_values(ctx, new, keys, heads, sizes, special=None):
    """`sizes` [dim]: what a normal value of each place is multiplied by."""
    q_heads, kv_heads, dim = heads
    cache = ref.Paged([keys], kv_heads, dim, 64, 5)
    values = cache.values[0] * sizes
    if special is not None:
        values[0, :, 9] = special
    set_values(cache, values, 64)
    g = torch.Generator().manual_seed(6)
    query = torch.randn(new, q_heads, dim, generator=g).bfloat16().cuda()
    gate = (2.0 * torch.randn(new, q_heads, dim, generator=g)).bfloat16().cuda()
    gate[:, :, 3] = 0.0
    output = torch.zeros_like(query)
    op = tk.PagedAttentionOp(ctx, q_heads, kv_heads, dim)
    op.launch(None, 1, ints([0, new]), ints([keys]), query, gate, cache.key, cache.value, cache.table, None, op.workspace(),
              output)
    assert ctx.device_status() == 0
    expected, size = ref.attention(query, cache.keys, cache.values, [0, new], op.scale, gate)
    got, finite = ref.f64(output), torch.isfinite(expected)
    bad = ~((got - expected).abs() <= tolerance(expected, size, keys)) & finite
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], expected[bad][:4])
    assert torch.equal(got[~finite], expected[~finite])
    return finite


# one key; a tile that no cut falls into; a tile that is split over many pairs
@pytest.mark.parametrize("new,keys", [(1, 1), (1, 17), (40, 60), (1, 3000)])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("largest", [1e35, 1e30, 1.0, 1e-34])
def test_rows_of_every_size(ctx, new, keys, heads, largest):
    # weights reach 2^8 in front of the division by their sum: 3000 keys of 5.5e35 would leave fp32
    if keys > 100:
        largest = min(largest, 1e30)
    run_values(ctx, new, keys, heads, torch.full((heads[2],), largest))


@pytest.mark.parametrize("new,keys", [(1, 1), (1, 17), (40, 60), (1, 3000)])
@pytest.mark.parametrize("heads", HEADS)
def test_rows_with_values_of_many_sizes(ctx, new, keys, heads):
    """A row's small values keep their digits next to its large ones."""
    run_values(ctx, new, keys, heads, 10.0 ** torch.linspace(-30, 30, heads[2]))


@pytest.mark.parametrize("special", [float("inf"), float("-inf")])
@pytest.mark.parametrize("new,keys", [(1, 1), (40, 60), (1, 3000)])
@pytest.mark.parametrize("heads", HEADS)
def test_rows_with_an_infinity(ctx, new, keys, heads, special):
    finite = run_values(ctx, new, keys, heads, torch.ones(heads[2]), special)
    assert (~finite).nonzero()[:, 2].unique().tolist() == [9]


def test_a_row_without_a_number_gates_the_others(ctx):
    """A NaN reaches its place of the rows that see it, and no other."""
    heads, new, keys = (24, 4, 256), 3, 20
    cache = ref.Paged([keys], heads[1], heads[2], 64, 5)
    values = cache.values[0].clone()
    values[0, 1, 100] = float("nan")
    set_values(cache, values, 64)
    g = torch.Generator().manual_seed(6)
    query, gate = (torch.randn(new, heads[0], heads[2], generator=g).bfloat16().cuda() for _ in range(2))
    output = torch.zeros_like(query)
    op = tk.PagedAttentionOp(ctx, *heads)
    op.launch(None, 1, ints([0, new]), ints([keys]), query, gate, cache.key, cache.value, cache.table, None, op.workspace(),
              output)
    expected, size = ref.attention(query, cache.keys, cache.values, [0, new], op.scale, gate)
    good = torch.isfinite(expected)
    assert torch.equal(good, torch.isfinite(ref.f64(output)))
    error = (ref.f64(output) - expected).abs()[good]
    assert bool((error <= tolerance(expected, size, keys)[good]).all())
