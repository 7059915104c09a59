"""The operators around the attention of a full-attention layer, as measurable cases.

Between the fused QKV projection and the output projection a serving program builds the block tables
and slot maps of its key/value cache (``page_plan``), normalises and rotates queries and keys and
stores keys and values (``rotary``), and attends: over the paged cache for decode steps and for chunks
of new tokens (``paged``), over the packed rows of whole prompts (``prompt``).

A case is one pass through one of them.  With ``own`` false it is computed in elementary torch
operations, with ``own`` true by the package's operators.  ``exact`` restates the definitions in 64 bits.

Geometry: 24 query heads over 4 key/value heads of 256 values (the 8192-row projection; 14336 rows where
a gate lies behind each query head), and generic layouts with heads of 128.
"""
from __future__ import annotations

import math
import zlib

import torch

own = False

HEADS = {  # layout -> (query heads, key/value heads, values per head)
    "24x4x256": (24, 4, 256),
    "32x8x128": (32, 8, 128),
    "16x16x128": (16, 16, 128),
    "8x1x256": (8, 1, 256),
}
EPSILON = 1e-6
THETA = 1e7


def listed():
    return [
        # Block tables and slots of a decode step of eight requests: the smallest plan, all latency.
        {"name": "plan_decode_8", "kind": "page_plan", "requests": 8, "most_new": 1, "most_cached": 4096, "page": 64, "finished": 0},
        # A step of a busy server: prompt chunks next to decodes, some requests just ended.
        {"name": "plan_mixed_301", "kind": "page_plan", "requests": 301, "most_new": 512, "most_cached": 8192, "page": 16, "finished": 37},
        # One decoded token, gated layout with head norms: rotate, store.
        {"name": "rotary_1", "kind": "rotary", "tokens": 1, "heads": "24x4x256", "rotary": 64, "axes": 1, "gated": True, "norm": True, "page": 64},
        # An odd chunk of an image's tokens: three position axes, far positions.
        {"name": "rotary_777_axes", "kind": "rotary", "tokens": 777, "heads": "24x4x256", "rotary": 64, "axes": 3, "gated": True, "norm": True, "page": 64},
        # A large prompt batch in the generic layout, every value rotated.
        {"name": "rotary_8192", "kind": "rotary", "tokens": 8192, "heads": "32x8x128", "rotary": 128, "axes": 1, "gated": False, "norm": False, "page": 128},
        # One decoded token over a 4096-token context: latency.
        {"name": "decode_1", "kind": "paged", "requests": 1, "most_new": 1, "most_cached": 4096, "ragged": False, "heads": "24x4x256", "page": 64, "gated": True},
        # A decode batch of ragged contexts: cache bandwidth.
        {"name": "decode_32", "kind": "paged", "requests": 32, "most_new": 1, "most_cached": 16384, "ragged": True, "heads": "24x4x256", "page": 64, "gated": True},
        # A chunk of 512 new tokens over 16000 cached ones, small pages.
        {"name": "chunk_512", "kind": "paged", "requests": 1, "most_new": 512, "most_cached": 16000, "ragged": False, "heads": "24x4x256", "page": 16, "gated": False},
        # Chunks of different lengths, some of one token, in the generic layout.
        {"name": "chunks_mixed_9", "kind": "paged", "requests": 9, "most_new": 300, "most_cached": 5000, "ragged": True, "heads": "32x8x128", "page": 32, "gated": False},
        # A short odd prompt.
        {"name": "prompt_301", "kind": "prompt", "sequences": 1, "longest": 301, "heads": "24x4x256", "gated": False},
        # Packed prompts of different lengths, heads of 128.
        {"name": "prompt_packed_7", "kind": "prompt", "sequences": 7, "longest": 1777, "heads": "32x8x128", "gated": False},
        # One long prompt: the largest contraction.
        {"name": "prompt_8192", "kind": "prompt", "sequences": 1, "longest": 8192, "heads": "24x4x256", "gated": True},
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["page_plan", "rotary", "rotary", "paged", "paged", "paged", "prompt", "prompt"])
    case = {"kind": kind}
    if kind == "page_plan":
        requests = _log(rng, 1, 512)
        case.update(requests=requests, most_new=_log(rng, 1, 512), most_cached=_log(rng, 16, 8192),
                    page=rng.choice([16, 32, 64, 128]), finished=rng.randint(0, requests // 4))
        return case
    heads = rng.choice(sorted(HEADS))
    if kind == "rotary":
        dim = HEADS[heads][2]
        case.update(tokens=_log(rng, 1, 8192), heads=heads, rotary=rng.choice([64, dim // 2, dim]),
                    axes=rng.choice([1, 1, 3]), gated=rng.random() < 0.5, norm=rng.random() < 0.5,
                    page=rng.choice([16, 64, 256]))
    elif kind == "paged":
        decode = rng.random() < 0.5
        requests = _log(rng, 1, 64) if decode else _log(rng, 1, 8)
        most_cached = _log(rng, 64, 16384 if requests <= 16 else 4096)
        # the queries times keys of a chunk stay below the long prompt's
        most_new = 1 if decode else _log(rng, 2, max(2, min(1024, 16 * 1024 * 1024 // (requests * (most_cached + 1024)))))
        case.update(requests=requests, most_new=most_new, most_cached=most_cached, ragged=rng.random() < 0.7,
                    heads=heads, page=rng.choice([16, 32, 64, 128]), gated=rng.random() < 0.5)
    else:
        sequences = _log(rng, 1, 16)
        case.update(sequences=sequences, longest=_log(rng, 2, int(6000 / math.sqrt(sequences))), heads=heads,
                    gated=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------------------- inputs

def _lengths(case, what, count, low, high, ragged=True):
    """`count` whole numbers in [low, high], the first of them `high`; they belong to the case, not to the seed."""
    numbers = sorted((k, v) for k, v in case.items() if k != "name")
    g = torch.Generator().manual_seed(zlib.crc32(repr((what, numbers)).encode()))
    if not ragged:
        return [high] * count
    u = torch.rand(count, generator=g, dtype=torch.float64)
    out = [int(round(low * (high / low) ** float(x))) for x in u]
    out[0] = high
    return out


def _query_chunks(case):
    """(new tokens, cached tokens before them) of every request of a paged case."""
    cached = _lengths(case, "cached", case["requests"], max(1, case["most_cached"] // 16), case["most_cached"], case["ragged"])
    new = _lengths(case, "new", case["requests"], 1, case["most_new"], case["ragged"])
    return new, cached


def _page_case(case):
    """New tokens, cached tokens and finished requests of a plan, on the host."""
    n = case["requests"]
    cached = _lengths(case, "cached", n, 1, case["most_cached"])
    new = _lengths(case, "new", n, 1, case["most_new"])
    cached[-1] = 0 if n > 1 else cached[-1]  # a request that starts
    return new, cached


def _prompt_lengths(case):
    return _lengths(case, "new", case["sequences"], max(1, case["longest"] // 12), case["longest"])


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(lengths):
    total = [0]
    total.extend(torch.tensor(lengths, dtype=torch.int64).cumsum(0).tolist())
    return total


def _frequencies(rotary):
    return THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)


def _pair_axes(rotary, axes):
    """The axis whose position turns each pair: the axes in turn, the first takes what is left over."""
    pairs = rotary // 2
    if axes == 1:
        return torch.zeros(pairs, dtype=torch.uint8)
    turn = torch.arange(pairs, dtype=torch.int64)
    return torch.where(turn < pairs // axes * axes, turn % axes, 0).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def bf16(*shape, std=1.0):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, std, generator=g)

    def order(count):
        return torch.randperm(count, generator=g, device="cuda").to(torch.int32)

    kind = case["kind"]
    state = {"case": case, "kind": kind}
    if kind == "page_plan":
        n, page = case["requests"], case["page"]
        new, cached = _page_case(case)
        finished = case["finished"]
        rows = n + finished
        most_pages = -(-(case["most_cached"] + case["most_new"]) // page)
        held = [-(-c // page) for c in cached] + [most_pages] * finished
        slots_of_rows = order(rows)  # the row of the table that each request has
        free = sum(-(-(c + t) // page) - -(-c // page) for c, t in zip(cached, new)) + 64
        pages = sum(held) + free
        ids = order(pages)
        at = torch.arange(most_pages, device="cuda")[None, :]
        first = _ints(_starts(held)[:-1], torch.int64)[:, None]
        mine = at < _ints(held, torch.int64)[:, None]
        table = torch.full((rows, most_pages), -1, dtype=torch.int32, device="cuda")
        table[slots_of_rows.long()] = torch.where(mine, ids[(first + at).clamp(max=pages - 1)], -1)
        lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")
        lengths[slots_of_rows.long()] = _ints(cached + [most_pages * page] * finished)
        stack = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        stack[:free] = ids[sum(held):]
        total = sum(new)
        state.update(requests=n, finished=finished, page=page, rows=slots_of_rows[:n].contiguous(),
                     ended=slots_of_rows[n:].contiguous(), new=_ints(new), lengths=lengths,
                     lengths_out=lengths.clone(), table=table, stack=stack, free=_ints([free]), free_mid=_ints([0]),
                     free_out=_ints([0]), starts=_ints([0] * (n + 1)), kv_lengths=_ints([0] * n),
                     positions=_ints([0] * total), slots=_ints([0] * total, torch.int64), total=total, pages=pages)
        if own:
            import tuiskollm_b200 as tk

            state["op"] = tk.PagePlanOp(tk.Context(), page_tokens=page)
        return state

    q_heads, kv_heads, dim = HEADS[case["heads"]]
    state.update(q_heads=q_heads, kv_heads=kv_heads, dim=dim)
    if kind == "rotary":
        t, page, axes, rotary = case["tokens"], case["page"], case["axes"], case["rotary"]
        wide = 2 * dim if case["gated"] else dim
        plane = bf16(t, q_heads * wide + 2 * kv_heads * dim)  # what the QKV projection left
        query = plane[:, :q_heads * wide].view(t, q_heads, wide)[:, :, :dim]
        key = plane[:, q_heads * wide:q_heads * wide + kv_heads * dim].view(t, kv_heads, dim)
        value = plane[:, q_heads * wide + kv_heads * dim:].view(t, kv_heads, dim)
        pages = -(-t // page) + 3
        first = int(torch.randint(0, 200000, (1,), generator=g, device="cuda"))
        steps = torch.arange(t, device="cuda")
        scan = [steps, steps // 40, steps % 40][:axes] if axes > 1 else [steps]
        positions = (first + torch.stack(scan)).to(torch.int32).contiguous()
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].contiguous()
        state.update(
            tokens=t, query=query, key=key, value=value, positions=positions, slots=slots, rotary=rotary,
            frequencies=_frequencies(rotary).cuda(), pair_axes=_pair_axes(rotary, axes).cuda(),
            query_norm=bf16(dim, std=0.1) if case["norm"] else None,
            key_norm=bf16(dim, std=0.1) if case["norm"] else None,
            key_cache=torch.zeros((pages, page, kv_heads, dim), dtype=torch.bfloat16, device="cuda"),
            value_cache=torch.zeros((pages, page, kv_heads, dim), dtype=torch.bfloat16, device="cuda"),
            query_out=torch.zeros((t, q_heads, dim), dtype=torch.bfloat16, device="cuda"))
        if own:
            import tuiskollm_b200 as tk

            state["op"] = tk.RotaryCacheOp(tk.Context(), q_heads, kv_heads, dim, state["frequencies"],
                                           state["pair_axes"])
        return state

    state["scale"] = 1.0 / math.sqrt(dim)
    if kind == "paged":
        n, page = case["requests"], case["page"]
        new, cached = _query_chunks(case)
        total, kv = sum(new), [a + b for a, b in zip(new, cached)]
        held = [-(-k // page) for k in kv]
        pages, most_pages = sum(held) + 3, max(held)
        ids = order(pages)
        at = torch.arange(most_pages, device="cuda")[None, :]
        first = _ints(_starts(held)[:-1], torch.int64)[:, None]
        table = torch.where(at < _ints(held, torch.int64)[:, None], ids[(first + at).clamp(max=pages - 1)], -1)
        state.update(table=table.to(torch.int32).contiguous(), page=page,
                     key_cache=bf16(pages, page, kv_heads, dim), value_cache=bf16(pages, page, kv_heads, dim))
    else:
        new = _prompt_lengths(case)
        total, kv, n = sum(new), new, len(new)
        state.update(key=bf16(total, kv_heads, dim), value=bf16(total, kv_heads, dim))
    gated = case["gated"]
    wide = bf16(total, q_heads, 2 * dim if gated else dim)
    state.update(sequences=n, tokens=total, query=wide[:, :, :dim], gate=wide[:, :, dim:] if gated else None,
                 starts=_ints(_starts(new)), kv_lengths=_ints(kv), longest_new=max(new), longest_kv=max(kv),
                 output=torch.zeros((total, q_heads, dim), dtype=torch.bfloat16, device="cuda"))
    if own:
        import tuiskollm_b200 as tk

        kinds = {"paged": tk.PagedAttentionOp, "prompt": tk.PromptAttentionOp}
        state["op"] = kinds[kind](tk.Context(), q_heads, kv_heads, dim)
        state["workspace"] = state["op"].workspace()
    return state


# ---------------------------------------------------------------------------- plain forms

def _plain_plan(s):
    """Released pages go on the stack in order, new ones come off its top in order."""
    page, table, rows = s["page"], s["table"], s["rows"].long()
    lengths, stack, free = s["lengths"].clone(), s["stack"].clone(), s["free"].long()
    columns = torch.arange(table.shape[1], device="cuda")[None, :]
    if s["finished"]:
        ended = s["ended"].long()
        count = (lengths[ended].long() + page - 1) // page
        place = (count.cumsum(0) - count)[:, None] + columns
        gives = columns < count[:, None]
        stack[(free + place)[gives]] = table[ended][gives]
        lengths[ended] = 0
        free = free + count.sum()
    old = lengths[rows].long()
    length = old + s["new"].long()
    held = (old + page - 1) // page
    need = (length + page - 1) // page - held
    rank = (need.cumsum(0) - need)[:, None] + columns - held[:, None]
    fresh = (columns >= held[:, None]) & (columns < (held + need)[:, None])
    mine = torch.where(fresh, stack[(free - 1 - rank).clamp(0, stack.numel() - 1)], table[rows])
    table = table.clone()
    table[rows] = mine
    lengths[rows] = length.to(torch.int32)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), s["new"].long().cumsum(0)])
    token = torch.arange(s["total"], device="cuda")
    request = torch.searchsorted(starts[1:], token, right=True)
    position = old[request] + token - starts[request]
    slots = mine[request, position // page].long() * page + position % page
    return {"lengths": lengths, "table": table, "stack": stack, "free": (free - need.sum()).to(torch.int32),
            "starts": starts.to(torch.int32), "kv_lengths": length.to(torch.int32),
            "positions": position.to(torch.int32), "slots": slots}


def _plain_norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON) * (1.0 + weight.float())


def _plain_rotary(s):
    """Pair (i, i + rotary / 2) of a head turns by position[axis of i] * frequency[i]; the rest passes."""
    half = s["rotary"] // 2
    angle = s["positions"].double()[s["pair_axes"].long()].t() * s["frequencies"]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turned(x):
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).to(torch.bfloat16)

    keys, values = s["key_cache"].clone(), s["value_cache"].clone()
    keys.view(-1, s["kv_heads"], s["dim"])[s["slots"]] = turned(_plain_norm(s["key"], s["key_norm"]))
    values.view(-1, s["kv_heads"], s["dim"])[s["slots"]] = s["value"]
    return {"query": turned(_plain_norm(s["query"], s["query_norm"])), "key_cache": keys, "value_cache": values}


def _plain_attention(s):
    """Token i of a sequence of q new tokens over k keys sees keys 0 .. k - q + i; sequences padded to the longest."""
    n, dim, q_heads, kv_heads = s["sequences"], s["dim"], s["q_heads"], s["kv_heads"]
    starts, kv = s["starts"].long(), s["kv_lengths"].long()
    new = starts[1:] - starts[:-1]
    row, column = torch.arange(s["longest_new"], device="cuda"), torch.arange(s["longest_kv"], device="cuda")
    live = row[None, :] < new[:, None]
    token = torch.where(live, starts[:-1, None] + row, 0)
    there = column[None, :] < kv[:, None]
    if s["kind"] == "paged":
        page = s["page"]
        place = s["table"].long()[:, column // page].clamp(min=0) * page + column % page
        flat_k, flat_v = s["key_cache"].view(-1, kv_heads, dim), s["value_cache"].view(-1, kv_heads, dim)
    else:
        place = torch.where(there, starts[:-1, None] + column, 0)
        flat_k, flat_v = s["key"], s["value"]
    key, value = flat_k[place].float(), flat_v[place].float().masked_fill_(~there[:, :, None, None], 0.0)
    query = s["query"][token].float().view(n, -1, kv_heads, q_heads // kv_heads, dim)
    score = torch.einsum("nqhgd,nkhd->nhgqk", query, key).mul_(s["scale"])
    seen = column[None, None, :] <= (kv - new)[:, None, None] + row[None, :, None]
    score.masked_fill_(~(seen & there[:, None, :])[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1)
    out = torch.einsum("nhgqk,nkhd->nhgqd", score, value) / total[..., None]
    out = out.permute(0, 3, 1, 2, 4).reshape(n, -1, q_heads, dim)[live]
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return {"output": out.to(torch.bfloat16)}


# ----------------------------------------------------------------------------------- run

def run(s):
    kind = s["kind"]
    if not own:
        return _plain_plan(s) if kind == "page_plan" else _plain_rotary(s) if kind == "rotary" else _plain_attention(s)
    op = s["op"]
    if kind == "page_plan":
        free = s["free"]
        if s["finished"]:
            op.release(None, s["finished"], s["ended"], s["lengths"], s["lengths_out"], s["table"], s["stack"],
                       s["free"], s["free_mid"])
            free = s["free_mid"]
        op.launch(None, s["requests"], s["rows"], s["new"], s["lengths"], s["lengths_out"], s["table"], s["stack"],
                  free, s["free_out"], s["starts"], s["kv_lengths"], s["positions"], s["slots"])
        return {"lengths": s["lengths_out"], "table": s["table"], "stack": s["stack"], "free": s["free_out"],
                "starts": s["starts"], "kv_lengths": s["kv_lengths"], "positions": s["positions"], "slots": s["slots"]}
    if kind == "rotary":
        op.launch(None, s["tokens"], s["positions"], s["query"], s["key"], s["value"], s["query_norm"], s["key_norm"],
                  s["query_out"], None, s["key_cache"], s["value_cache"], s["slots"])
        return {"query": s["query_out"], "key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    if kind == "paged":
        op.launch(None, s["sequences"], s["starts"], s["kv_lengths"], s["query"], s["gate"], s["key_cache"],
                  s["value_cache"], s["table"], None, s["workspace"], s["output"])
    else:
        op.launch(None, s["sequences"], s["starts"], s["query"], s["gate"], s["key"], s["value"], s["workspace"],
                  s["output"])
    return {"output": s["output"]}


# ---------------------------------------------------------------------------------- work

def _visible(new, kv):
    """Query-key pairs of a sequence: token i of `new` sees kv - new + i + 1 keys."""
    return new * (kv - new) + new * (new + 1) // 2


def work(case):
    kind = case["kind"]
    if kind == "page_plan":
        new, cached = _page_case(case)
        page, total = case["page"], sum(new)
        fresh = sum(-(-(c + t) // page) - -(-c // page) for c, t in zip(cached, new))
        held = sum(-(-c // page) for c in cached)
        ended = case["finished"] * -(-(case["most_cached"] + case["most_new"]) // page)
        touched = sum(1 for c in cached if c % page)  # last pages that new tokens go on in
        return {"bytes": 12 * total + 8 * fresh + 24 * case["requests"] + 4 * min(held, touched) + 8 * ended, "flops": 0}
    q_heads, kv_heads, dim = HEADS[case["heads"]]
    if kind == "rotary":
        t = case["tokens"]
        moved = 2 * t * (q_heads + 2 * kv_heads) * dim * 2 + t * (8 + 4 * case["axes"])
        return {"bytes": moved, "flops": t * (q_heads + kv_heads) * (3 * case["rotary"] + (4 * dim if case["norm"] else 0))}
    if kind == "paged":
        new, cached = _query_chunks(case)
        kv = [a + b for a, b in zip(new, cached)]
    else:
        new = kv = _prompt_lengths(case)
    rows = sum(new) * q_heads * dim * 2 * (3 if case["gated"] else 2)
    pairs = sum(_visible(a, b) for a, b in zip(new, kv))
    return {"bytes": rows + sum(kv) * kv_heads * dim * 2 * 2, "flops": 4 * pairs * q_heads * dim}


# --------------------------------------------------------------------------------- exact

def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "page_plan":
        page = s["page"]
        lengths, table, stack = s["lengths"].tolist(), s["table"].tolist(), s["stack"].tolist()
        free = int(s["free"])
        for row in s["ended"].tolist():
            for k in range(-(-lengths[row] // page)):
                stack[free] = table[row][k]
                free += 1
            lengths[row] = 0
        top, starts, kv, positions, slots = free, [0], [], [], []
        for row, new in zip(s["rows"].tolist(), s["new"].tolist()):
            old = lengths[row]
            for k in range(-(-old // page), -(-(old + new) // page)):
                top -= 1
                table[row][k] = stack[top]
            for p in range(old, old + new):
                positions.append(p)
                slots.append(table[row][p // page] * page + p % page)
            lengths[row] = old + new
            kv.append(old + new)
            starts.append(starts[-1] + new)
        return {"lengths": _ints(lengths), "table": _ints(table), "stack": _ints(stack), "free": _ints([top]),
                "starts": _ints(starts), "kv_lengths": _ints(kv), "positions": _ints(positions),
                "slots": _ints(slots, torch.int64)}
    if kind == "rotary":
        out, r = {}, s["rotary"]
        for name in ("query", "key"):
            x, w = s[name].double(), s[name + "_norm"]
            if w is not None:
                x = x / (x.pow(2).sum(-1, keepdim=True) / s["dim"] + EPSILON).sqrt() * (w.double() + 1.0)
            y = x.clone()
            for pair in range(r // 2):
                turn = s["positions"][int(s["pair_axes"][pair])].double() * float(s["frequencies"][pair])
                z = torch.complex(x[..., pair], x[..., pair + r // 2]) * torch.polar(torch.ones_like(turn), turn)[:, None]
                y[..., pair], y[..., pair + r // 2] = z.real, z.imag
            out[name] = y
        keys, values = s["key_cache"].double(), s["value_cache"].double()
        keys.view(-1, s["kv_heads"], s["dim"]).index_copy_(0, s["slots"], out["key"])
        values.view(-1, s["kv_heads"], s["dim"]).index_copy_(0, s["slots"], s["value"].double())
        return {"query": out["query"], "key_cache": keys, "value_cache": values}
    result = torch.zeros((s["tokens"], s["q_heads"], s["dim"]), dtype=torch.float64, device="cuda")
    group = s["q_heads"] // s["kv_heads"]
    starts, kv = s["starts"].tolist(), s["kv_lengths"].tolist()
    for i in range(s["sequences"]):
        a, b = starts[i], starts[i + 1]
        hidden = torch.ones((b - a, kv[i]), dtype=torch.bool, device="cuda").triu(kv[i] - (b - a) + 1)
        if kind == "paged":
            where = s["table"][i, :-(-kv[i] // s["page"])].long()
            key, value = (s[c][where].flatten(0, 1)[:kv[i]] for c in ("key_cache", "value_cache"))
        else:
            key, value = s["key"][a:b], s["value"][a:b]
        for h in range(s["q_heads"]):
            score = s["query"][a:b, h].double() @ key[:, h // group].double().t() * s["scale"]
            weight = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
            result[a:b, h] = weight @ value[:, h // group].double()
    if s["gate"] is not None:
        result = result * torch.sigmoid(s["gate"].double())
    return {"output": result}
