"""Plain 64-bit forms of the full-attention step's operators, on the CPU, and builders of their planes."""
import numpy as np
import torch


def f64(t):
    return t.detach().cpu().double()


def attention(query, keys, values, starts, scale, gate=None):
    """Causal attention of packed queries [tokens, heads, dim]; keys/values: one [k, kv heads, dim] per sequence.
    Returns (output, magnitude): magnitude = sum of softmax * |v|, what a relative error of the weights scales."""
    query = f64(query)
    out, size = torch.zeros_like(query), torch.zeros_like(query)
    group = query.shape[1] // keys[0].shape[1]
    for s, (key, value) in enumerate(zip(keys, values)):
        key, value = f64(key), f64(value)
        a, b = starts[s], starts[s + 1]
        new, kv = b - a, key.shape[0]
        seen = torch.arange(kv)[None, :] <= kv - new + torch.arange(new)[:, None]
        for h in range(query.shape[1]):
            score = query[a:b, h] @ key[:, h // group].t() * scale
            score = score.masked_fill(~seen, float("-inf"))
            for i in range(new):
                n = int(seen[i].sum())
                if n == 0:
                    continue
                weight = torch.softmax(score[i, :n], -1)
                out[a + i, h] = weight @ value[:n, h // group]
                size[a + i, h] = weight @ value[:n, h // group].abs()
    if gate is not None:
        open_ = torch.sigmoid(f64(gate))
        out, size = out * open_, size * open_
    return out, size


def attention_tolerance(out, size, gated=False):
    """The weights are rounded to BF16 (2^-8 of each, so 2^-8 of `size`), the result is (2^-8 of it).  Scores and
    sums are fp32: the exponent's error, up to dim * 2^-24 * sum |q k| * scale, is below 2^-11 for the normal planes
    of these tests (256 * 2^-24 * 256 * 0.64 / 16 = 1.6e-4), and ex2 and the sums add less; 2^-10 covers them.  A gated row is rounded
    to FP16 in front of its gate: 2^-11 more of the result, and 2^-25 of the row's largest value, which lies far below
    2^-10 of `size`; a row that holds a value that is not finite to BF16, 2^-8."""
    return (2.0 ** -8 + 2.0 ** -10) * size + (2.0 ** -8 + 2.0 ** -11 if gated else 2.0 ** -8) * out.abs() + 1e-30


def rotate(x, positions, frequencies, pair_axes, weight=None, epsilon=1e-6):
    """x [tokens, heads, dim] in 64 bits; positions [axes, tokens]."""
    x = f64(x)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon) * (1.0 + f64(weight))
    half = frequencies.numel()
    axes = torch.zeros(half, dtype=torch.long) if pair_axes is None else pair_axes.cpu().long()
    angle = positions.cpu().double()[axes].t() * f64(frequencies)  # [tokens, half]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def plan(page, rows, new, lengths, table, stack, free):
    """Python integers: the step's outputs, or None where it does not fit."""
    lengths, table = list(lengths), [list(r) for r in table]
    if len(set(rows)) != len(rows) or any(r < 0 or r >= len(lengths) for r in rows) or any(n < 0 for n in new):
        return None
    starts, kv, positions, slots, top = [0], [], [], [], free
    for row, n in zip(rows, new):
        old = lengths[row]
        if old + n > len(table[row]) * page:
            return None
        for k in range(-(-old // page), -(-(old + n) // page)):
            top -= 1
            if top < 0:
                return None
            table[row][k] = stack[top]
        for p in range(old, old + n):
            positions.append(p)
            slots.append(table[row][p // page] * page + p % page)
        lengths[row] = old + n
        kv.append(old + n)
        starts.append(starts[-1] + n)
    return dict(lengths=lengths, table=table, free=top, starts=starts, kv_lengths=kv, positions=positions, slots=slots)


class Paged:
    """A paged cache with sequences of given lengths in it; what no sequence holds is `filler`."""

    def __init__(self, lengths, kv_heads, dim, page, seed=0, filler=float("nan"), order="token", spare=2):
        g = torch.Generator().manual_seed(seed)
        held = [-(-n // page) for n in lengths]
        pages, most = sum(held) + spare, max(max(held), 1)
        ids = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lengths), most), -7, dtype=torch.int32)
        self.keys, self.values = [], []
        shape = (pages, page, kv_heads, dim)
        key, value = torch.full(shape, filler), torch.full(shape, filler)
        at = 0
        for s, n in enumerate(lengths):
            k = torch.randn(n, kv_heads, dim, generator=g).bfloat16().float()
            v = torch.randn(n, kv_heads, dim, generator=g).bfloat16().float()
            self.keys.append(k)
            self.values.append(v)
            for j in range(held[s]):
                self.table[s, j] = ids[at]
                part = k[j * page:(j + 1) * page]
                key[ids[at], :part.shape[0]] = part
                value[ids[at], :part.shape[0]] = v[j * page:(j + 1) * page]
                at += 1
        self.key, self.value = (self._lay(t, order) for t in (key, value))
        if order == "pair":  # one plane, keys and values of a token next to each other
            both = torch.stack([key, value], 3).bfloat16().cuda()
            self.key, self.value = both[:, :, :, 0], both[:, :, :, 1]
        self.table = self.table.cuda()

    @staticmethod
    def _lay(t, order):
        t = t.bfloat16()
        if order == "head":  # [pages, heads, tokens, dim] in memory
            return t.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
        return t.cuda()


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
