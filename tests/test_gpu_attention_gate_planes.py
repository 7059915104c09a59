"""Gates with strides of their own: where the projection left them, next to queries rotated into a dense plane."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from gpu_util import graph_replay
from test_gpu_full_attention_step import HIDDEN, VALUE_WIDTH, Layer, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return tk.Context()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def wide_plane(tokens, heads, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    plane = torch.randn(tokens, heads * 2 * dim + 64, generator=g).bfloat16().cuda()
    both = plane[:, :heads * 2 * dim].view(tokens, heads, 2 * dim)
    return both[..., :dim], both[..., dim:]


@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128), (1, 1, 128)])
@pytest.mark.parametrize("new,cached", [([1], [0]), ([1], [3000]), ([1, 0, 70], [129, 5, 300])])
def test_paged(ctx, heads, new, cached):
    q_heads, kv_heads, dim = heads
    kv = [a + b for a, b in zip(new, cached)]
    cache, tokens = ref.Paged(kv, kv_heads, dim, 64, 1), sum(new)
    query, gate = wide_plane(tokens, q_heads, dim)
    op = tk.PagedAttentionOp(ctx, *heads)
    work, results = op.workspace(), []
    # both dense; the queries dense; the gate dense; both in the plane
    for q, g in ((query.contiguous(), gate.contiguous()), (query.contiguous(), gate), (query, gate.contiguous()), (query, gate)):
        out = torch.zeros(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda")
        op.launch(None, len(new), ints(ref.starts_of(new)), ints(kv), q, g, cache.key, cache.value, cache.table, None, work, out)
        results.append(out)
    assert ctx.device_status() == 0
    expected, size = ref.attention(query, cache.keys, cache.values, ref.starts_of(new), op.scale, gate)
    assert bool(((ref.f64(results[0]) - expected).abs() <= ref.attention_tolerance(expected, size, gated=True)).all())
    for out in results[1:]:
        assert torch.equal(out, results[0])


@pytest.mark.parametrize("heads", [(24, 4, 256), (8, 2, 128)])
def test_prompt(ctx, heads):
    q_heads, kv_heads, dim = heads
    lengths = [3, 130, 1, 200]
    tokens, starts = sum(lengths), ref.starts_of(lengths)
    query, gate = wide_plane(tokens, q_heads, dim, 2)
    g = torch.Generator().manual_seed(3)
    key, value = (torch.randn(tokens, kv_heads, dim, generator=g).bfloat16().cuda() for _ in range(2))
    op = tk.PromptAttentionOp(ctx, *heads)
    work, results = op.workspace(), []
    for q, o in ((query.contiguous(), gate.contiguous()), (query.contiguous(), gate)):
        out = torch.zeros(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda")
        op.launch(None, len(lengths), ints(starts), q, o, key, value, work, out)
        results.append(out)
    split = [(starts[i], starts[i + 1]) for i in range(len(lengths))]
    expected, size = ref.attention(query, [key[a:b] for a, b in split], [value[a:b] for a, b in split], starts, op.scale, gate)
    assert bool(((ref.f64(results[0]) - expected).abs() <= ref.attention_tolerance(expected, size, gated=True)).all())
    assert torch.equal(results[1], results[0]) and ctx.device_status() == 0


class ChainedLayer(Layer):
    """The layer with nothing between its operators: the gate is read in the projection's plane."""

    def step(self, requests, new):
        t = self.tokens
        self.plan.launch(None, requests, None, new, self.lengths, self.lengths, self.table, self.stack, self.free,
                         self.free, self.starts, self.kv, self.positions, self.slots)
        self.qkv.launch(None, t, self.x, self.codes, self.scales, self.qkv_w, self.qkv_s, self.plane)
        self.rotary.launch(None, t, self.positions, self.query, self.key, self.value, *self.norms, self.rotated, None,
                           self.keys, self.values, self.slots)
        self.attention.launch(None, requests, self.starts, self.kv, self.rotated, self.gate, self.keys, self.values,
                              self.table, None, self.workspace, self.attended)
        self.out.launch(None, t, HIDDEN, VALUE_WIDTH, self.attended.view(t, VALUE_WIDTH), self.codes2, self.scales2,
                        self.out_w, self.out_s, self.y)


def test_a_layer_without_a_copy_of_the_gate():
    """A prompt, then decode steps as replays of one captured graph that holds the library's launches alone."""
    ctx = tk.Context()
    layer = ChainedLayer(ctx, 50, 1, 4)
    layer.step(1, ints([50]))
    assert ctx.device_status() == 0
    plane = layer.plane.clone().cpu()
    close(layer, 50, [(plane, 50)])
    decode = ChainedLayer(ctx, 1, 1, 4)
    for name in ("qkv_w", "qkv_s", "out_w", "out_s", "norms", "keys", "values", "table", "lengths", "free", "stack"):
        setattr(decode, name, getattr(layer, name))
    one = ints([1])
    graph = graph_replay(lambda: decode.step(1, one))  # runs one step in front of the capture
    g = torch.Generator().manual_seed(9)
    for step in range(3):
        if step > 0:
            decode.x.copy_(torch.randn(1, HIDDEN, generator=g).bfloat16())
            graph.replay()
        assert ctx.device_status() == 0
        plane = torch.cat([plane, decode.plane.cpu()])
        close(decode, 1, [(plane, 1)])


def test_refusals(ctx):
    cache = ref.Paged([40], 2, 128, 16, 3)
    query, gate = wide_plane(5, 6, 128)
    op = tk.PagedAttentionOp(ctx, 6, 2, 128)
    out = torch.zeros(5, 6, 128, dtype=torch.bfloat16, device="cuda")
    work = op.workspace()

    def refused(text, gate, output=out):
        with pytest.raises(tk.GpuError, match=text):
            op.launch(None, 1, ints([0, 5]), ints([40]), query, gate, cache.key, cache.value, cache.table, None, work, output)

    plane = torch.zeros(5 * 6 * 256, dtype=torch.bfloat16, device="cuda")
    refused("gate head stride 132", plane[:5 * 6 * 132].view(5, 6, 132)[..., :128])
    refused("gate token stride 780", plane[:5 * 780].view(5, 780)[:, :768].view(5, 6, 128))
    refused("gate plane is not 16-byte aligned", plane[4:4 + 5 * 768].view(5, 6, 128))
    refused("gate", gate[:3])
    refused("gate", plane[:1].view(1, 1, 1).expand(5, 6, 128))
    # the gate's last rows lie in the output, where rows of the queries' strides would not
    refused("overlaps the gate", plane.view(5, 6, 256)[..., :128], plane[5 * 768:].view(5, 6, 128))
    op.launch(None, 1, ints([0, 5]), ints([40]), query.contiguous(), gate, cache.key, cache.value, cache.table, None, work, out)
    assert ctx.device_status() == 0
