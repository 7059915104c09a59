"""The operators of a full-attention layer as a step uses them, one behind the other: FP8 QKV projection, page plan,
head norms with rotary positions and cache stores, attention, output projection."""
import pytest
import torch

import attention_ref as ref
import tuiskollm_b200 as tk
from gpu_util import graph_replay

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, DIM, PAGE = 5120, 24, 4, 256, 64
QKV_ROWS = Q_HEADS * 2 * DIM + 2 * KV_HEADS * DIM  # 14336: each query head with its gate, keys, values
VALUE_WIDTH = Q_HEADS * DIM


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


class Layer:
    """One layer's weights, planes and cache for up to `tokens` rows and `rows` requests."""

    def __init__(self, ctx, tokens, rows, pages, seed=0):
        from tuiskollm_b200 import synth

        g = torch.Generator().manual_seed(seed)
        self.ctx, self.tokens = ctx, tokens
        self.qkv_w, self.qkv_s = synth.torch_fp8_weights(seed + 1, 1, QKV_ROWS, HIDDEN, "cuda")
        self.out_w, self.out_s = synth.torch_fp8_weights(seed + 1, 2, HIDDEN, VALUE_WIDTH, "cuda")
        self.norms = [torch.randn(DIM, generator=g).mul(0.1).bfloat16().cuda() for _ in range(2)]
        bf16 = dict(dtype=torch.bfloat16, device="cuda")
        self.x = torch.randn(tokens, HIDDEN, generator=g).bfloat16().cuda()
        self.codes = torch.zeros(tokens, HIDDEN, dtype=torch.uint8, device="cuda")
        self.scales = torch.zeros(tokens, dtype=torch.float32, device="cuda")
        self.codes2 = torch.zeros(tokens, VALUE_WIDTH, dtype=torch.uint8, device="cuda")
        self.scales2 = torch.zeros(tokens, dtype=torch.float32, device="cuda")
        self.plane = torch.zeros(tokens, QKV_ROWS, **bf16)
        wide = self.plane[:, :Q_HEADS * 2 * DIM].view(tokens, Q_HEADS, 2 * DIM)
        self.query, self.gate = wide[..., :DIM], wide[..., DIM:]
        self.key = self.plane[:, Q_HEADS * 2 * DIM:-KV_HEADS * DIM].view(tokens, KV_HEADS, DIM)
        self.value = self.plane[:, -KV_HEADS * DIM:].view(tokens, KV_HEADS, DIM)
        # the gate's strides are the projection's, so the rotated queries take their place in the plane
        self.rotated = torch.zeros(tokens, Q_HEADS, DIM, **bf16)
        self.keys, self.values = (torch.full((pages, PAGE, KV_HEADS, DIM), float("nan"), **bf16) for _ in range(2))
        self.attended = torch.zeros(tokens, Q_HEADS, DIM, **bf16)
        self.y = torch.zeros(tokens, HIDDEN, **bf16)
        self.table = torch.full((rows, 16), -1, dtype=torch.int32, device="cuda")
        self.lengths, self.free = ints([0] * rows), ints([pages])
        self.stack = ints(torch.randperm(pages, generator=g).tolist())
        self.starts, self.kv = ints([0] * (rows + 1)), ints([0] * rows)
        self.positions, self.slots = ints([0] * tokens), ints([0] * tokens, torch.int64)
        self.frequencies = tk.rotary_frequencies(64, 1e7)
        self.plan = tk.PagePlanOp(ctx, PAGE)
        self.qkv = tk.FullAttentionQkvOp(ctx, QKV_ROWS)
        self.rotary = tk.RotaryCacheOp(ctx, Q_HEADS, KV_HEADS, DIM, self.frequencies)
        self.attention = tk.PagedAttentionOp(ctx, Q_HEADS, KV_HEADS, DIM)
        self.workspace = self.attention.workspace()
        self.out = tk.Fp8ProjectionOp(ctx)

    def step(self, requests, new):
        """`new` new tokens of requests 0 .. requests - 1, with what lies behind them in the planes padded."""
        t = self.tokens
        self.plan.launch(None, requests, None, new, self.lengths, self.lengths, self.table, self.stack, self.free,
                         self.free, self.starts, self.kv, self.positions, self.slots)
        self.qkv.launch(None, t, self.x, self.codes, self.scales, self.qkv_w, self.qkv_s, self.plane)
        self.rotary.launch(None, t, self.positions, self.query, self.key, self.value, *self.norms, self.rotated, None,
                           self.keys, self.values, self.slots)
        # queries rotated into a plane of their own: the gate goes with them as one of the same strides
        gate = self.gate.contiguous()
        self.attention.launch(None, requests, self.starts, self.kv, self.rotated, gate, self.keys, self.values, self.table,
                              None, self.workspace, self.attended)
        self.out.launch(None, t, HIDDEN, VALUE_WIDTH, self.attended.view(t, VALUE_WIDTH), self.codes2, self.scales2,
                        self.out_w, self.out_s, self.y)


def expected(layer, history):
    """Attention of the last step from the projection's rows of all steps: one [tokens, QKV_ROWS] plane per request."""
    outs, sizes = [], []
    for rows, new in history:
        t = rows.shape[0]
        wide = rows[:, :Q_HEADS * 2 * DIM].reshape(t, Q_HEADS, 2 * DIM)
        at = torch.arange(t)[None]
        # what the operators pass on is BF16: the rotated queries and keys, the values
        query = ref.rotate(wide[..., :DIM], at, layer.frequencies, None, layer.norms[0]).bfloat16()
        key = ref.rotate(rows[:, Q_HEADS * 2 * DIM:-KV_HEADS * DIM].reshape(t, KV_HEADS, DIM), at, layer.frequencies, None,
                         layer.norms[1]).bfloat16()
        value = rows[:, -KV_HEADS * DIM:].reshape(t, KV_HEADS, DIM)
        out, size = ref.attention(query[t - new:], [key], [value], [0, new], DIM ** -0.5, wide[t - new:, :, DIM:])
        outs.append(out)
        sizes.append(size)
    return torch.cat(outs), torch.cat(sizes)


def close(layer, tokens, history):
    """Beyond the attention's own tolerance: a rotated query or key that lies at a rounding border may be rounded the
    other way than the 64-bit one, one unit of 2^-8 of it.  Such a value moves a score by 2^-8 |q k| / 16 of one of 256
    products, below 2^-8 * 5.5^2 * 1.5^2 / 16 = 0.017 for normal planes with norm weights up to 1.5; a few dozen of them
    in a row of 256 add up to at most 0.1 in the exponent, a tenth of the weights' size."""
    out, size = expected(layer, history)
    error = (ref.f64(layer.attended[:tokens]) - out).abs()
    assert bool((error <= ref.attention_tolerance(out, size, gated=True) + 0.1 * size).all()), float(error.max())
    # and as a whole: rounding errors of 2^-9 of independent signs, three of them, far below 1 %
    assert float(error.norm() / out.norm()) < 0.01


def test_prompts_then_decode_steps():
    """Two prompts of different lengths in one step, then decode steps as replays of one captured graph."""
    ctx = tk.Context()
    layer = Layer(ctx, 77 + 40, 2, 12)
    layer.step(2, ints([77, 40]))
    assert ctx.device_status() == 0
    planes = [layer.plane[:77].clone().cpu(), layer.plane[77:117].clone().cpu()]
    close(layer, 117, [(planes[0], 77), (planes[1], 40)])
    # the output projection of the same rows
    weights = ref.f64(layer.out_s.view(torch.bfloat16))[:, None] * ref.f64(layer.out_w.view(torch.float8_e4m3fn).float())
    rows = ref.f64(layer.attended.view(117, VALUE_WIDTH))
    error = ref.f64(layer.y) - rows @ weights.t()
    # e4m3 activations: 2^-4 of each product at most, of independent signs
    assert float(error.norm()) < 2.0 ** -4 * float((rows @ weights.t()).norm())

    decode = Layer(ctx, 4, 2, 12)  # two requests in planes padded to four rows
    for name in ("qkv_w", "qkv_s", "out_w", "out_s", "norms", "keys", "values", "table", "lengths", "free", "stack"):
        setattr(decode, name, getattr(layer, name))
    one = ints([1, 1])
    decode.attended.fill_(7.0)
    graph = graph_replay(lambda: decode.step(2, one))  # runs one step in front of the capture
    g = torch.Generator().manual_seed(9)
    for step in range(4):
        if step > 0:
            decode.x.copy_(torch.randn(4, HIDDEN, generator=g).bfloat16())
            graph.replay()
        assert ctx.device_status() == 0
        for r in range(2):
            planes[r] = torch.cat([planes[r], decode.plane[r:r + 1].cpu()])
        close(decode, 2, [(planes[0], 1), (planes[1], 1)])
        assert bool((decode.attended[2:] == 7.0).all()), "padded rows were written"
    assert decode.lengths.tolist() == [81, 44]


def test_a_prompt_in_chunks_is_the_prompt_at_once():
    """Paged chunks of a prompt against packed attention over it, and against one chunk."""
    ctx = tk.Context()
    tokens, chunks = 300, [1, 128, 43, 128]
    g = torch.Generator().manual_seed(3)
    query, key, value = (torch.randn(tokens, h, DIM, generator=g).bfloat16().cuda() for h in (Q_HEADS, KV_HEADS, KV_HEADS))
    whole = torch.zeros_like(query)
    prompt = tk.PromptAttentionOp(ctx, Q_HEADS, KV_HEADS, DIM)
    work = prompt.workspace()
    prompt.launch(None, 1, ints([0, tokens]), query, None, key, value, work, whole)
    pages = -(-tokens // PAGE)
    keys, values = (torch.zeros(pages, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    keys.view(-1, KV_HEADS, DIM)[:tokens], values.view(-1, KV_HEADS, DIM)[:tokens] = key, value
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    paged = tk.PagedAttentionOp(ctx, Q_HEADS, KV_HEADS, DIM)
    at = 0
    expected_out, size = ref.attention(query, [key], [value], [0, tokens], paged.scale)
    for n in chunks:
        out = torch.zeros(n, Q_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        paged.launch(None, 1, ints([0, n]), ints([at + n]), query[at:at + n], None, keys, values, table, None, work, out)
        for o in (out, whole[at:at + n]):
            error = (ref.f64(o) - expected_out[at:at + n]).abs()
            assert bool((error <= ref.attention_tolerance(expected_out[at:at + n], size[at:at + n])).all())
        at += n
    assert ctx.device_status() == 0


def test_two_streams_with_a_workspace_each():
    """Launches that overlap, eager and captured, with a workspace each give what they give alone."""
    ctx = tk.Context()
    op = tk.PagedAttentionOp(ctx, Q_HEADS, KV_HEADS, DIM)
    jobs = []
    for seed, (new, cached) in enumerate([([1, 1, 1], [3000, 900, 40]), ([60, 1], [700, 2500])]):
        kv = [a + b for a, b in zip(new, cached)]
        cache = ref.Paged(kv, KV_HEADS, DIM, PAGE, seed)
        g = torch.Generator().manual_seed(seed)
        query = torch.randn(sum(new), Q_HEADS, DIM, generator=g).bfloat16().cuda()
        out, work, stream = torch.zeros_like(query), op.workspace(), torch.cuda.Stream()
        starts, kv = ints(ref.starts_of(new)), ints(kv)

        def launch(stream=None, new=new, starts=starts, kv=kv, query=query, cache=cache, work=work, out=out):
            op.launch(stream, len(new), starts, kv, query, None, cache.key, cache.value, cache.table, None, work, out)

        launch()
        torch.cuda.synchronize()
        jobs.append((launch, out, out.clone(), stream, graph_replay(launch)))
    for _ in range(30):
        for launch, out, alone, stream, graph in jobs:
            with torch.cuda.stream(stream):
                out.zero_()
                launch(stream)
                launch(stream.cuda_stream)
                graph.replay()
    torch.cuda.synchronize()
    for launch, out, alone, stream, graph in jobs:
        assert torch.equal(out, alone)
    assert ctx.device_status() == 0
