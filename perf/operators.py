"""The paged cache's operators, as cases to measure: append (with the position rotation on the way), attention over
pages of 16-bit or 4-bit rows, and reading rows back.

A slot is one KV head of one sequence: index sequence * heads + head.  Its rows lie in pages of `page` rows, which a page
table names in any order.  A 4-bit row holds, per group of `group` channels, a float16 scale and offset, and a code of
0..15 per channel that stands for offset + scale * (code - 8).

Cases: "op" is append, attend or read; `sequences` sequences with between `low` and `high` rows in each slot (spread, as
evictions leave them), between 1 and `tokens` new tokens each (all `tokens` where `even`).
"""
import math

import torch

own = False

CODE_LEVELS = 15
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    head8 = {"heads": 8, "groups": 4, "dim": 128}  # the 32-layer, 8-KV-head shape of the benchmark
    return [
        # One decode step of one request: three rows a head and the step's queries rotated.  Latency.
        {"name": "append16_step", "op": "append", "bits": 16, "group": 0, "page": 64, "dtype": "bf16", **head8,
         "sequences": 1, "tokens": 1, "even": True, "low": 2000, "high": 2000, "rotary": 128, "interleaved": False, "fused": True},
        # A prompt of mixed requests going into 16-bit pages (the static batch's prompts are 1,024 to 16,384 long).
        {"name": "append16_prompts", "op": "append", "bits": 16, "group": 0, "page": 64, "dtype": "bf16", **head8,
         "sequences": 8, "tokens": 4096, "even": False, "low": 0, "high": 0, "rotary": 128, "interleaved": False, "fused": True},
        # A decode step of a batch into 4-bit pages, small heads, rotation of half the channels in neighbouring pairs.
        {"name": "append4_batch", "op": "append", "bits": 4, "group": 32, "page": 32, "dtype": "f16", "heads": 8, "groups": 4, "dim": 64,
         "sequences": 61, "tokens": 1, "even": True, "low": 100, "high": 4096, "rotary": 32, "interleaved": True, "fused": False},
        # A whole 32,768-token prompt quantised into 4-bit pages.
        {"name": "append4_prompt", "op": "append", "bits": 4, "group": 64, "page": 64, "dtype": "bf16", **head8,
         "sequences": 1, "tokens": 32768, "even": True, "low": 0, "high": 0, "rotary": 128, "interleaved": False, "fused": True},
        # One request's decode step over its evicted budget of about 2,000 rows a head.  Latency.
        {"name": "attend4_step", "op": "attend", "bits": 4, "group": 64, "page": 64, "dtype": "bf16", **head8,
         "sequences": 1, "tokens": 1, "even": True, "low": 1900, "high": 2100},
        # The static batch of 8 requests, slots as ragged as evictions leave them.
        {"name": "attend4_ragged", "op": "attend", "bits": 4, "group": 64, "page": 64, "dtype": "bf16", **head8,
         "sequences": 8, "tokens": 1, "even": True, "low": 1024, "high": 18384},
        # The large serving shape: 32 requests of 32,768 rows a head, 8 query heads a KV head.
        {"name": "attend4_long", "op": "attend", "bits": 4, "group": 128, "page": 128, "dtype": "bf16", "heads": 8, "groups": 8, "dim": 128,
         "sequences": 32, "tokens": 1, "even": True, "low": 32768, "high": 34768},
        # Checking up to 7 drafted tokens a sequence, small heads, pages smaller than a tile, odd group count.
        {"name": "attend4_verify", "op": "attend", "bits": 4, "group": 32, "page": 16, "dtype": "f16", "heads": 5, "groups": 3, "dim": 64,
         "sequences": 24, "tokens": 7, "even": False, "low": 7, "high": 9001},
        # The audit window: 250 queries over a prompt of 34,768 rows.
        {"name": "attend4_window", "op": "attend", "bits": 4, "group": 64, "page": 64, "dtype": "bf16", **head8,
         "sequences": 1, "tokens": 250, "even": True, "low": 34768, "high": 34768},
        # The static batch in 16-bit pages.
        {"name": "attend16_ragged", "op": "attend", "bits": 16, "group": 0, "page": 64, "dtype": "f16", **head8,
         "sequences": 8, "tokens": 1, "even": True, "low": 1024, "high": 18384},
        # One layer of the benchmark's request back in the packed layout, for the audit.
        {"name": "read4_layer", "op": "read", "bits": 4, "group": 64, "page": 64, "dtype": "bf16", **head8,
         "sequences": 1, "tokens": 1, "even": True, "low": 33000, "high": 36000},
        # A few short slots, 32-channel groups: latency.
        {"name": "read4_short", "op": "read", "bits": 4, "group": 32, "page": 16, "dtype": "f16", "heads": 3, "groups": 1, "dim": 64,
         "sequences": 2, "tokens": 1, "even": True, "low": 1, "high": 700},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "read"])
    dim = rng.choice([64, 128])
    bits = rng.choice([4, 4, 16]) if op != "read" else 4
    case = {"op": op, "bits": bits, "group": rng.choice([g for g in (32, 64, 128) if g <= dim]) if bits == 4 else 0,
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "f16"]), "heads": rng.choice([1, 2, 3, 4, 5, 8, 8]),
            "groups": rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), "dim": dim, "sequences": _spread(rng, 1, 64)}
    heads = case["heads"]
    if op == "append":
        most = 32768 * 8 * 6 // (heads * (case["groups"] + 2))  # no more than the largest prompt above
        case["tokens"] = min(_spread(rng, 1, 32768), max(1, most // case["sequences"]))
        case["even"] = rng.random() < 0.5
        case["low"] = rng.choice([0, 0, 1, 500])
        case["high"] = case["low"] + rng.choice([0, 1, 37, 2000])
        case["rotary"] = rng.choice([dim, dim, dim // 2, 16])
        case["interleaved"] = rng.random() < 0.3
        case["fused"] = rng.random() < 0.5
        return case
    case["tokens"], case["even"] = 1, True
    if op == "attend" and rng.random() < 0.5:
        case["tokens"], case["even"] = _spread(rng, 2, 256), rng.random() < 0.5
    byte = {4: 1, 16: 4}[bits]
    # Bytes within the long case's, and products within the window's.
    rows = 32 * 8 * 33768 // (byte * 4 * heads * case["sequences"])
    if op == "attend":
        rows = min(rows, 34768 * 250 * 4 * 8 // (heads * case["sequences"] * case["tokens"] * case["groups"]))
    else:
        rows = min(rows, 34768 * 8 // (heads * case["sequences"]))
    case["high"] = _spread(rng, 1, max(1, min(rows, 131072)))
    case["low"] = max(1, int(case["high"] * rng.choice([0.05, 0.5, 0.9, 1.0])))
    return case


# ------------------------------------------------------------------ inputs

def _layout(case, seed):
    """New tokens a sequence, rows before and rows after, on the host.  What an output's shape goes by is the case's alone."""
    g = torch.Generator().manual_seed(seed * 2 + 1 if case["op"] == "attend" else 1)
    S, H, T = case["sequences"], case["heads"], case["tokens"]
    low, high = case["low"], case["high"]
    counts = torch.full((S,), T) if case["even"] else torch.randint(1, T + 1, (S,), generator=torch.Generator().manual_seed(2))
    rows = torch.randint(low, high + 1, (S * H,), generator=g)
    new = counts.repeat_interleave(H)
    lengths = rows + new if case["op"] == "append" else rows
    return counts, rows, lengths


def _normal(shape, generator, dtype, spread=None):
    x = torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32)
    return (x if spread is None else x * spread).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, D, H, P = DTYPES[case["dtype"]], case["dim"], case["heads"], case["page"]
    S, Q = case["sequences"], case["heads"] * case["groups"]
    counts, before, lengths = _layout(case, seed)
    starts = torch.zeros(S + 1, dtype=torch.int32)
    starts[1:] = counts.cumsum(0)
    total = int(starts[-1])
    need = (lengths + P - 1) // P
    wide = int(need.max()) + 1
    pages = int(need.sum()) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(S * H, wide, dtype=torch.int64)
    at = torch.arange(wide)[None, :] + (need.cumsum(0) - need)[:, None]
    used = torch.arange(wide)[None, :] < need[:, None]
    table[used] = order[at[used]]
    state = {"case": dict(case), "table": table.to(torch.int32).cuda(), "lengths": lengths.to(torch.int32).cuda(),
             "starts": starts.cuda(), "longest": int(lengths.max()), "total": total}
    channel = torch.exp(0.5 * torch.randn(D, generator=g, device="cuda"))  # some channels are larger than others
    filled = case["op"] != "append"
    if case["bits"] == 16:
        make = (lambda spread: _normal((pages, P, D), g, dtype, spread)) if filled else (lambda spread: torch.zeros(pages, P, D, dtype=dtype, device="cuda"))
        state |= {"keys": make(channel), "values": make(None), "key_scales": None, "value_scales": None}
    else:
        for name, spread in (("key", channel), ("value", None)):
            codes = torch.zeros(pages, P, D // 2, dtype=torch.uint8, device="cuda")
            scales = torch.zeros(pages, P, D // case["group"], 2, dtype=torch.float16, device="cuda")
            if filled:
                some = 1 << 14  # pages at a time, so that the float32 rows stay small
                for a in range(0, pages, some):
                    codes[a:a + some], scales[a:a + some] = _quantise(_normal((min(some, pages - a), P, D), g, torch.float32, spread), case["group"])
            state |= {name + "s": codes, name + "_scales": scales}
    state["positions"] = torch.zeros(pages, P, dtype=torch.float32, device="cuda")
    if case["op"] == "append":
        if case["fused"]:  # a model's joint projection, split into views
            joint = _normal((total, Q + 2 * H, D), g, dtype)
            joint[:, Q:Q + H] *= channel.to(dtype)
            state |= {"queries": joint[:, :Q], "new_keys": joint[:, Q:Q + H], "new_values": joint[:, Q + H:]}
        else:
            state |= {"queries": _normal((total, Q, D), g, dtype), "new_keys": _normal((total, H, D), g, dtype, channel),
                      "new_values": _normal((total, H, D), g, dtype)}
        sequence = torch.arange(S).repeat_interleave(counts)
        first = before.view(S, H).amax(1) + torch.randint(0, 1000, (S,), generator=torch.Generator().manual_seed(seed))
        state["new_positions"] = (first[sequence] + torch.arange(total) - starts[:-1].long()[sequence]).cuda()
        R = case["rotary"]
        angle = torch.arange(int(state["new_positions"].max()) + 1, dtype=torch.float64, device="cuda")[:, None] * (
            500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R))
        state["rotary"] = torch.cat((angle.cos(), angle.sin()), 1).float()  # [positions, R]: cosines, then sines
        new = counts.repeat_interleave(H)
        state["first_rows"] = (lengths - new).to(torch.int32).cuda()
        row_starts = torch.zeros(S * H + 1, dtype=torch.int32)
        row_starts[1:] = new.cumsum(0)
        state["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    elif case["op"] == "attend":
        state["queries"] = _normal((total, Q, D), g, dtype)
        state["workspace"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")  # kept, as a program keeps it
        state["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        state["positions"] = torch.randint(0, 50000, (pages, P), generator=g, device="cuda").float()
        state["first_rows"] = torch.zeros(S * H, dtype=torch.int32, device="cuda")
        row_starts = torch.zeros(S * H + 1, dtype=torch.int32)
        row_starts[1:] = lengths.cumsum(0)
        state["flag"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] != "attend":
        state["row_starts"], state["rows"] = row_starts.cuda(), int(row_starts[-1])
    return state


# ------------------------------------------------------------ plain forms

def _quantise(x, group):
    """Codes uint8 [..., D / 2] (even channel in the low bits) and float16 [..., D / group, 2] (scale, offset)."""
    x = x.unflatten(-1, (-1, group))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) * (1.0 / CODE_LEVELS)).half()
    offset = (low + 8 * scale.float()).half()
    fine = torch.isfinite(scale) & torch.isfinite(offset)
    inverse = torch.where(scale > 0, scale.float().reciprocal(), 0)[..., None]
    code = (((x - offset.float()[..., None]) * inverse).round() + 8).clamp(0, 15)
    code = torch.where(fine[..., None], code, 0).to(torch.uint8).flatten(-2)
    nan = torch.full_like(scale, float("nan"))
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack((torch.where(fine, scale, nan), torch.where(fine, offset, nan)), -1)


def _values(codes, scales):
    """The float32 rows that codes and scales stand for."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    n = n.unflatten(-1, (scales.shape[-2], -1))
    return (scales[..., 1:].float() + scales[..., :1].float() * n).flatten(-2)


def _rotate(x, table, interleaved):
    """x [tokens, heads, D] in float32, its first table.shape[1] channels rotated by each token's cosines and sines."""
    x = x.float()
    R = table.shape[1]
    cos, sin = table[:, None, :R // 2], table[:, None, R // 2:]
    head, rest = x[..., :R], x[..., R:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :R // 2], head[..., R // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((head, rest), -1)


def _tokens(starts, total):
    """Each token's sequence, its place in it, and the sequence's new tokens."""
    token = torch.arange(total, device=starts.device)
    sequence = torch.searchsorted(starts, token, right=True) - 1
    return sequence, token - starts[sequence], (starts[1:] - starts[:-1])[sequence]


def _append(s, case):
    H, P = case["heads"], case["page"]
    sequence, place, count = _tokens(s["starts"], s["total"])
    slot = sequence[:, None] * H + torch.arange(H, device=sequence.device)
    row = s["lengths"][slot] - count[:, None] + place[:, None]
    page, line = s["table"][slot, row // P].long(), row % P
    cs = s["rotary"][s["new_positions"]]
    keys = _rotate(s["new_keys"], cs, case["interleaved"])
    if case["bits"] == 16:
        s["keys"][page, line] = keys.to(s["keys"].dtype)
        s["values"][page, line] = s["new_values"]
    else:
        s["keys"][page, line], s["key_scales"][page, line] = _quantise(keys, case["group"])
        s["values"][page, line], s["value_scales"][page, line] = _quantise(s["new_values"].float(), case["group"])
    s["positions"][page, line] = s["new_positions"].float()[:, None].expand(-1, H)
    return _rotate(s["queries"], cs, case["interleaved"]).to(s["queries"].dtype)


def _read(s, case):
    slot = torch.searchsorted(s["row_starts"], torch.arange(s["rows"], device="cuda"), right=True) - 1
    row = torch.arange(s["rows"], device="cuda") - s["row_starts"][slot] + s["first_rows"][slot]
    page, line = s["table"][slot, row // case["page"]].long(), row % case["page"]
    dtype = DTYPES[case["dtype"]]
    return (_values(s["keys"][page, line], s["key_scales"][page, line]).to(dtype),
            _values(s["values"][page, line], s["value_scales"][page, line]).to(dtype), s["positions"][page, line])


def _attend(s, case):
    H, G, D, P, T, S = (case[k] for k in ("heads", "groups", "dim", "page", "tokens", "sequences"))
    pages = s["table"][:, :-(-s["longest"] // P)].long()
    if case["bits"] == 16:
        keys, values = s["keys"][pages].float(), s["values"][pages].float()
    else:
        keys, values = _values(s["keys"][pages], s["key_scales"][pages]), _values(s["values"][pages], s["value_scales"][pages])
    keys, values = keys.flatten(1, 2), values.flatten(1, 2)
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    index = (s["starts"][:-1, None].long() + torch.arange(T, device="cuda")).clamp(max=s["total"] - 1)
    q = s["queries"].float()[index].view(S, T, H, G, D).transpose(1, 2).reshape(S * H, T * G, D)
    scores = torch.bmm(q, keys.transpose(1, 2)) * (D ** -0.5)
    del keys
    last = s["lengths"].view(S, H, 1) - counts[:, None, None] + torch.arange(T, device="cuda")  # a query's last row
    seen = torch.arange(scores.shape[-1], device="cuda") <= last.view(S * H, T, 1)
    scores = scores.view(S * H, T, G, -1).masked_fill_(~seen[:, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp_(scores.sub_(torch.where(torch.isfinite(top), top, 0))).flatten(1, 2)
    norm = weight.sum(-1, keepdim=True)
    # Rows that no page holds (beyond a slot's length) weigh zero; what lies there may be anything finite.
    out = torch.bmm(weight, values) / torch.where(norm > 0, norm, 1)
    lse = top.flatten(1) + norm.flatten(1).log()
    sequence, place, _ = _tokens(s["starts"], s["total"])
    out = out.view(S, H, T, G, D).transpose(1, 2)[sequence, place].reshape(-1, H * G, D)
    lse = lse.view(S, H, T, G).transpose(1, 2)[sequence, place].reshape(-1, H * G)
    return out.to(s["queries"].dtype), lse


def run(state):
    s, case = state, state["case"]
    if own:
        from code_for_iclr27_b200.paged import Pages, paged_append, paged_attention, paged_read

        pages = Pages(s["keys"], s["values"], s["positions"], s["key_scales"], s["value_scales"])
        if case["op"] == "attend":
            return paged_attention(pages, s["table"], s["lengths"], s["queries"], s["starts"], s["workspace"], s["flag"])
        if case["op"] == "append":
            queries = paged_append(pages, s["table"], s["lengths"], s["new_keys"], s["new_values"], s["new_positions"], s["starts"],
                                   s["flag"], s["rotary"], case["interleaved"], s["queries"])
            if case["bits"] == 16:
                return queries, s["keys"], s["values"], s["positions"]
            # The appended rows, as the values that they are held as.
            return queries, *paged_read(pages, s["table"], s["first_rows"], s["row_starts"], s["rows"], DTYPES[case["dtype"]], s["flag"])
        return paged_read(pages, s["table"], s["first_rows"], s["row_starts"], s["rows"], DTYPES[case["dtype"]], s["flag"])
    if case["op"] == "attend":
        return _attend(s, case)
    if case["op"] == "append":
        queries = _append(s, case)
        return (queries, s["keys"], s["values"], s["positions"]) if case["bits"] == 16 else (queries, *_read(s, case))
    return _read(s, case)


# --------------------------------------------------------- 64-bit results

def exact(case, seed):
    s = prepare(case, seed)
    H, G, D, P = (case[k] for k in ("heads", "groups", "dim", "page"))
    lengths, starts, table = s["lengths"].tolist(), s["starts"].tolist(), s["table"].long()

    def held(name, slot, first, end):
        row = torch.arange(first, end, device="cuda")
        page, line = table[slot, row // P], row % P
        x = s[name + "s"][page, line]
        if case["bits"] == 16:
            return x.double()
        p = s[name + "_scales"][page, line].double()
        codes = torch.empty(len(row), D, dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = (x % 16).double(), (x // 16).double()
        each = p.repeat_interleave(case["group"], 1)
        return each[..., 1] + each[..., 0] * (codes - 8)

    if case["op"] == "attend":
        if s["longest"] * s["total"] * H * G > 4e9:
            return None
        out = torch.zeros(s["total"], H * G, D, dtype=torch.float64, device="cuda")
        lse = torch.full((s["total"], H * G), float("-inf"), dtype=torch.float64, device="cuda")
        for slot, length in enumerate(lengths):
            a, b = starts[slot // H], starts[slot // H + 1]
            h = slot % H
            keys, values = held("key", slot, 0, length), held("value", slot, 0, length)
            scores = torch.einsum("tgd,rd->tgr", s["queries"][a:b, h * G:h * G + G].double(), keys) / math.sqrt(D)
            visible = torch.arange(length, device="cuda")[None] < (length - (b - a) + 1 + torch.arange(b - a, device="cuda"))[:, None]
            scores = torch.where(visible[:, None], scores, -math.inf)
            total = torch.logsumexp(scores, -1)
            weight = torch.where(visible[:, None], torch.exp(scores - total[..., None]), 0.0)
            out[a:b, h * G:h * G + G] = torch.einsum("tgr,rd->tgd", weight, values)
            lse[a:b, h * G:h * G + G] = total
        return out, lse

    if case["op"] == "read":
        rows = [(held("key", i, 0, n), held("value", i, 0, n)) for i, n in enumerate(lengths)]
        return torch.cat([k for k, _ in rows]), torch.cat([v for _, v in rows]), None

    R = case["rotary"]
    cs = s["rotary"].double()[s["new_positions"]]

    def turned(x):
        z = x.double().clone()
        first = torch.arange(R // 2, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else R // 2)
        u, v = x.double()[..., first], x.double()[..., second]
        angle_cos, angle_sin = cs[:, None, :R // 2], cs[:, None, R // 2:]
        z[..., first], z[..., second] = u * angle_cos - v * angle_sin, u * angle_sin + v * angle_cos
        return z

    queries, keys, values = turned(s["queries"]), turned(s["new_keys"]), s["new_values"].double()
    if case["bits"] == 4:
        def through(x):  # the nearest of the sixteen values that the group's float16 scale and offset give
            y = x.reshape(*x.shape[:-1], -1, case["group"])
            bottom = y.min(-1, keepdim=True).values
            step = ((y.max(-1, keepdim=True).values - bottom) / CODE_LEVELS).half().double()
            middle = (bottom + 8 * step).half().double()
            level = torch.clamp(torch.round((y - middle) / torch.where(step > 0, step, 1.0)), -8, 7)
            return (middle + step * level).reshape(x.shape)

        keys, values = through(keys), through(values)
        counts = [b - a for a, b in zip(starts, starts[1:])]
        pick = lambda x: torch.cat([x[starts[i]:starts[i + 1]].transpose(0, 1).reshape(-1, D) for i in range(len(counts))])  # noqa: E731
        return queries, pick(keys), pick(values), None
    pool_keys, pool_values = s["keys"].double(), s["values"].double()
    for slot, length in enumerate(lengths):
        a, b = starts[slot // H], starts[slot // H + 1]
        row = torch.arange(length - (b - a), length, device="cuda")
        pool_keys[table[slot, row // P], row % P] = keys[a:b, slot % H]
        pool_values[table[slot, row // P], row % P] = values[a:b, slot % H]
    return queries, pool_keys, pool_values, None


# -------------------------------------------------------------------- work

def work(case):
    D, H, G = case["dim"], case["heads"], case["groups"]
    mean = lambda low, high: (low + high) / 2  # noqa: E731
    tokens = case["sequences"] * (case["tokens"] if case["even"] else mean(1, case["tokens"]))
    row = 2 * (2 * D if case["bits"] == 16 else D // 2 + 4 * D // case["group"])  # key and value
    if case["op"] == "append":
        moved = tokens * (2 * D * (2 * H + 2 * H * G) + H * (row + 4) + 8 + 4 * case["rotary"])
        if case["bits"] == 4:  # and read back
            moved += tokens * H * (row + 4 + 4 * D + 4)
        return {"bytes": moved, "flops": 3 * tokens * (H + H * G) * case["rotary"]}
    rows = case["sequences"] * H * mean(case["low"], case["high"])
    if case["op"] == "read":
        return {"bytes": rows * (row + 4 + 4 * D + 4), "flops": 2 * rows * 2 * D}
    each = tokens / case["sequences"]
    return {"bytes": rows * (row + 4 / case["page"]) + tokens * H * G * (4 * D + 4), "flops": 4.0 * D * G * rows * each}
