"""The token operators over the sizes they are used at: cases, their plain forms and their exact values.

One step of a token model in low-bit form: the norms around a block with its gate and residual scale, appending
rotated keys and values to a paged cache held in 4 bits (and reading stored tokens back), attention over that
cache, and products of a few rows with 4-bit weight matrices. ``run`` computes each either in plain 32-bit torch
operations or, where ``own`` is set, through ``nvcr_b200.tokens``.

The 4-bit form is the same everywhere: a group of consecutive values is held as codes c in 0..15 with an FP16
scale s and an FP16 minimum m, and stands for c * s + m. Two codes share a byte, the even index in the low half.
Appending takes m = fp16(min), s = fp16((max - min) / 15), or 2^-24 where that is 0 and the range is not, and
c = clamp(rint((x - m) / s), 0, 15), from FP32.
"""
import math

import torch

own = False

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ----

def listed():
    return [
        # norms: one token of a narrow model; a long prompt of a wide one; a short batch of an odd width in FP32
        {"name": "norm one token", "op": "norm", "rows": 1, "width": 2048, "type": "float16", "kind": "rms",
         "post": True, "gate": "channel"},
        {"name": "norm prompt", "op": "norm", "rows": 4096, "width": 4096, "type": "bfloat16", "kind": "rms",
         "post": True, "gate": "row"},
        {"name": "norm odd width", "op": "norm", "rows": 77, "width": 1111, "type": "float32", "kind": "layer",
         "post": False, "gate": "none"},
        # append: one token of one sequence; a prompt of 8192 tokens
        {"name": "append one token", "op": "append", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "group": 64, "rotary": 128, "interleaved": False, "page": 16, "type": "float16"},
        {"name": "append prompt", "op": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "group": 32, "rotary": 64, "interleaved": True, "page": 64, "type": "bfloat16"},
        # attention: a short answer's step; a served batch of unequal lengths; one long document; a few new tokens
        # for each of five sequences, every query head with a cache of its own
        {"name": "attend short", "op": "attend", "batch": 1, "length": 200, "least": 200, "queries": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "group": 64, "page": 16, "type": "float16"},
        {"name": "attend batch", "op": "attend", "batch": 32, "length": 4096, "least": 1, "queries": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "group": 64, "page": 64, "type": "bfloat16"},
        {"name": "attend long", "op": "attend", "batch": 1, "length": 131072, "least": 131072, "queries": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "group": 128, "page": 64, "type": "float16"},
        {"name": "attend few tokens", "op": "attend", "batch": 5, "length": 777, "least": 100, "queries": 4,
         "heads": 6, "kv_heads": 6, "dim": 64, "group": 32, "page": 48, "type": "bfloat16"},
        # products: one token through a square projection; a batch of 16 through a wide one; odd sizes
        {"name": "multiply one token", "op": "multiply", "rows": 1, "inputs": 4096, "outputs": 4096, "group": 128,
         "bias": False, "type": "float16"},
        {"name": "multiply batch", "op": "multiply", "rows": 16, "inputs": 4096, "outputs": 16384, "group": 64,
         "bias": False, "type": "bfloat16"},
        {"name": "multiply odd", "op": "multiply", "rows": 5, "inputs": 1088, "outputs": 1001, "group": 32,
         "bias": True, "type": "float16"},
    ]


def _spread(rng, low, high):
    """A whole number in low..high, evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attend", "attend", "multiply", "multiply"])
    if op == "norm":
        width = _spread(rng, 64, 16384)
        if rng.random() < 0.5:
            width = max(64, width // 64 * 64)
        return {"op": op, "rows": _spread(rng, 1, min(8192, (1 << 24) // width)), "width": width,
                "type": rng.choice(["float16", "bfloat16"]), "kind": rng.choice(["rms", "rms", "layer"]),
                "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "row"])}
    if op == "multiply":
        group = rng.choice([32, 64, 128])
        inputs = _spread(rng, 256, 16384) // group * group
        return {"op": op, "rows": _spread(rng, 1, 16), "inputs": inputs,
                "outputs": _spread(rng, 64, min(16384, (1 << 26) // inputs)), "group": group,
                "bias": rng.random() < 0.3, "type": rng.choice(["float16", "bfloat16"])}
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim <= 4 * g])
    kv_heads = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 48, 64, 128])
    kind = rng.choice(["float16", "bfloat16"])
    if op == "append":
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        most = min(8192, (8192 * 40 * 128) // ((heads + kv_heads) * dim))
        return {"op": op, "tokens": _spread(rng, 1, most), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "group": group, "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4,
                "page": page, "type": kind}
    heads = kv_heads * rng.choice([1, 2, 4, 6, 8, 16])
    queries = rng.choice([1, 1, 1, 2, 5])
    room = (1 << 27) // (kv_heads * dim * queries * max(1, heads // kv_heads // 4))
    batch = _spread(rng, 1, 64)
    length = _spread(rng, 16, max(16, min(131072, room // batch)))
    return {"op": op, "batch": batch, "length": length, "least": max(queries, length // rng.choice([1, 2, 8])),
            "queries": queries, "heads": heads, "kv_heads": kv_heads, "dim": dim, "group": group, "page": page,
            "type": kind}


# ---- what the program has in hand ----

def _lengths(case):
    """The sequences' lengths: evenly from `least` to `length`."""
    n = case["batch"]
    return [case["length"] - (case["length"] - case["least"]) * i // max(1, n - 1) for i in range(n)]


def _counts(case):
    """The sequences' numbers of new tokens: 1 to `queries`, `queries` first."""
    return [case["queries"] - i % case["queries"] for i in range(case["batch"])]


def _codes(x, group):
    """The 4-bit form of x along its last axis: codes (one a byte), scales and minimums."""
    g = x.float().unflatten(-1, (-1, group))
    low, high = g.amin(-1), g.amax(-1)
    minimums = low.half()
    scales = ((high - low) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).half()
    scales = torch.where((scales == 0) & (high > low), torch.full_like(scales, 2.0 ** -24), scales)
    s = scales.float().unsqueeze(-1)
    codes = torch.where(s > 0, torch.round((g - minimums.float().unsqueeze(-1)) / s), torch.zeros_like(g))
    return codes.clamp(0, 15).to(torch.uint8).flatten(-2), scales, minimums


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _normal(shape, make, spread=1.0, mean=0.0):
    return torch.randn(shape, generator=make, device="cuda", dtype=torch.float32) * spread + mean


def _prepare_norm(case, make):
    kind, rows, width = TYPES[case["type"]], case["rows"], case["width"]
    layer = case["kind"] == "layer"
    state = {"block": _normal((rows, width), make, 0.7, 0.1).to(kind),
             "residual": _normal((rows, width), make, 3.0).to(kind),
             "pre_weight": _normal((width,), make, 0.2, 1.0).to(kind),
             "pre_bias": _normal((width,), make, 0.1).to(kind) if layer else None,
             "post_weight": _normal((width,), make, 0.2, 1.0).to(kind) if case["post"] else None,
             "post_bias": _normal((width,), make, 0.1).to(kind) if layer and case["post"] else None}
    shape = {"none": None, "channel": (width,), "row": (rows, width)}[case["gate"]]
    state["gate"] = None if shape is None else _normal(shape, make, 0.3, 0.5).to(kind)
    state["residual_scale"], state["epsilon"] = 0.875, 1e-6
    return state


def _empty_cache(case, pages):
    shape = (pages, case["kv_heads"], case["page"])
    parts = case["dim"] // case["group"]
    make = lambda *tail, kind: torch.zeros(shape + tail, dtype=kind, device="cuda")  # noqa: E731
    return {"key_codes": make(case["dim"] // 2, kind=torch.uint8), "key_scales": make(parts, 2, kind=torch.float16),
            "value_codes": make(case["dim"] // 2, kind=torch.uint8),
            "value_scales": make(parts, 2, kind=torch.float16)}


def _prepare_append(case, make):
    kind, tokens, page = TYPES[case["type"]], case["tokens"], case["page"]
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    pages = -(-tokens // page) + 3
    order = torch.randperm(pages, generator=make, device="cuda")
    at = torch.arange(tokens, device="cuda")
    first = int(torch.randint(0, 1000, (1,), generator=make, device="cuda"))
    angles = torch.outer(torch.arange(tokens + 1000, device="cuda", dtype=torch.float64),
                         10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64)
                                     / case["rotary"]))
    # queries, keys and values are one projection's output, as slices of its rows
    rows = _normal((tokens, heads + 2 * kv_heads, dim), make)
    rows[:, heads:heads + kv_heads, : dim // 16] *= 6.0  # keys have a few channels of large values
    rows = rows.to(kind)
    return {"queries": rows[:, :heads], "keys": rows[:, heads:heads + kv_heads], "values": rows[:, heads + kv_heads:],
            "slots": order[at // page] * page + at % page, "positions": (at + first).to(torch.int32),
            "cosines": angles.cos().float(), "sines": angles.sin().float(), **_empty_cache(case, pages)}


def _prepare_attend(case, make):
    kind, page, dim = TYPES[case["type"]], case["page"], case["dim"]
    lengths, counts = _lengths(case), _counts(case)
    most = -(-case["length"] // page)
    pages = case["batch"] * most + 2
    state = _empty_cache(case, pages)
    for part, mean in (("key", 0.3), ("value", 0.0)):
        for first in range(0, pages, 256):  # a part at a time: the FP32 form of the whole would be large
            some = slice(first, min(pages, first + 256))
            shape = state[part + "_codes"][some].shape[:3] + (dim,)
            codes, scales, minimums = _codes(_normal(shape, make, 1.0, mean), case["group"])
            state[part + "_codes"][some] = _pack(codes)
            state[part + "_scales"][some] = torch.stack((scales, minimums), -1)
    order = torch.randperm(case["batch"], generator=make, device="cuda").tolist()
    lengths, counts = [lengths[i] for i in order], [counts[i] for i in order]
    table = torch.randperm(pages, generator=make, device="cuda")[: case["batch"] * most]
    state["table"] = table.view(case["batch"], most).to(torch.int32)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
    state["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    state["queries"] = _normal((offsets[-1], case["heads"], dim), make, 1.5).to(kind)
    state["scale"] = dim ** -0.5
    return state


def _prepare_multiply(case, make):
    kind, rows, inputs, outputs = TYPES[case["type"]], case["rows"], case["inputs"], case["outputs"]
    codes, scales, minimums = _codes(_normal((outputs, inputs), make, inputs ** -0.5), case["group"])
    x = _normal((rows, inputs), make)
    x[:, :: inputs // 8] *= 10.0  # activations have a few channels of large values
    return {"x": x.to(kind), "codes": _pack(codes), "scales": scales, "minimums": minimums,
            "bias": _normal((outputs,), make, 0.1).to(kind) if case["bias"] else None}


def prepare(case, seed):
    make = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"norm": _prepare_norm, "append": _prepare_append, "attend": _prepare_attend,
             "multiply": _prepare_multiply}[case["op"]](case, make)
    state["case"] = case
    if own:
        from nvcr_b200 import tokens

        if case["op"] in ("append", "attend"):
            state["cache"] = tokens.PagedCache(state["key_codes"], state["key_scales"], state["value_codes"],
                                               state["value_scales"])
        if case["op"] == "attend":
            state["context"] = tokens.TokenContext()
        if case["op"] == "multiply":
            state["matrix"] = tokens.PackedMatrix(state["codes"], state["scales"], state["minimums"])
    return state


# ---- one pass ----

def _plain_normed(x, weight, bias, layer, epsilon):
    if layer:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + epsilon) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm(s):
    layer, kind = s["case"]["kind"] == "layer", s["block"].dtype
    p = s["block"].float()
    if s["post_weight"] is not None:
        p = _plain_normed(p, s["post_weight"], s["post_bias"], layer, s["epsilon"])
    if s["gate"] is not None:
        p = p * s["gate"].float()
    hidden = s["residual"].float() * s["residual_scale"] + p
    normed = _plain_normed(hidden, s["pre_weight"], s["pre_bias"], layer, s["epsilon"])
    return {"hidden": hidden.to(kind), "normed": normed.to(kind)}


def _plain_values(codes, scales):
    """What packed codes [..., n / 2] with scales [..., groups, 2] stand for, in 32 bits."""
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (scales.shape[-2], -1))
    s = scales.float()
    return (pairs.float() * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def _plain_rotated(x, cosines, sines, rotary, interleaved):
    x = x.float()
    turned, rest = x[..., :rotary], x[..., rotary:]
    c, s = cosines.unsqueeze(1), sines.unsqueeze(1)
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turned[..., : rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(s):
    case, kind = s["case"], s["keys"].dtype
    place, cosines, sines = s["positions"].long(), s["cosines"], s["sines"]
    turn = lambda x: _plain_rotated(x, cosines[place], sines[place], case["rotary"], case["interleaved"])  # noqa: E731
    at, within = s["slots"] // case["page"], s["slots"] % case["page"]
    out = {"queries": turn(s["queries"]).to(kind)}
    for part, x in (("key", turn(s["keys"])), ("value", s["values"])):
        codes, scales, minimums = _codes(x, case["group"])
        s[part + "_codes"][at, :, within] = _pack(codes)
        s[part + "_scales"][at, :, within] = torch.stack((scales, minimums), -1)
        out[part + "s"] = _plain_values(s[part + "_codes"][at, :, within], s[part + "_scales"][at, :, within]).to(kind)
    return out


def _plain_attend(s):
    case, kind = s["case"], s["queries"].dtype
    batch, queries, heads, kv_heads = case["batch"], case["queries"], case["heads"], case["kv_heads"]
    table, offsets, lengths = s["table"].long(), s["offsets"].long(), s["lengths"].long()
    here = torch.arange(table.shape[1] * case["page"], device="cuda")
    inside = here < lengths.view(batch, 1)

    def whole(part):  # [batch, kv_heads, places, dim], nothing past a sequence's end
        x = _plain_values(s[part + "_codes"][table], s[part + "_scales"][table]).transpose(1, 2).flatten(2, 3)
        return torch.where(inside.view(batch, 1, -1, 1), x, torch.zeros((), device="cuda"))

    nth = torch.arange(queries, device="cuda")
    counts = offsets[1:] - offsets[:-1]
    rows = (offsets[:-1, None] + nth).clamp(max=s["queries"].shape[0] - 1)
    q = s["queries"].float()[rows].unflatten(2, (kv_heads, heads // kv_heads))
    scores = torch.einsum("bqhgd,bhtd->bhgqt", q, whole("key")) * s["scale"]
    last = lengths[:, None] - counts[:, None] + nth  # each row's own position
    seen = inside[:, None, :] & (here <= last[:, :, None])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = weights.sum(-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.einsum("bhgqt,bhtd->bqhgd", weights, whole("value")).flatten(2, 3).to(kind)
    token = torch.arange(s["queries"].shape[0], device="cuda")
    sequence = torch.searchsorted(offsets, token, right=True) - 1
    return out[sequence, token - offsets[sequence]]


def _plain_multiply(s):
    weights = _plain_values(s["codes"], torch.stack((s["scales"], s["minimums"]), -1))
    y = s["x"].float() @ weights.t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend,
                "multiply": _plain_multiply}[op](s)
    if op == "norm":
        from nvcr_b200 import tokens

        hidden, normed = tokens.block_norm(
            s["block"], residual=s["residual"], gate=s["gate"], post=s["post_weight"] is not None,
            post_weight=s["post_weight"], post_bias=s["post_bias"], pre_weight=s["pre_weight"],
            pre_bias=s["pre_bias"], kind=s["case"]["kind"], residual_scale=s["residual_scale"], epsilon=s["epsilon"])
        return {"hidden": hidden, "normed": normed}
    if op == "append":
        turned = s["cache"].append(s["keys"], s["values"], s["slots"], queries=s["queries"], positions=s["positions"],
                                   cosines=s["cosines"], sines=s["sines"], interleaved=s["case"]["interleaved"])
        keys, values = s["cache"].read(s["slots"], s["keys"].dtype)
        return {"queries": turned, "keys": keys, "values": values}
    if op == "attend":
        return s["context"].attend(s["queries"], s["cache"], s["table"], s["lengths"], query_offsets=s["offsets"],
                                   max_queries=s["case"]["queries"], max_length=s["case"]["length"], scale=s["scale"])
    return s["matrix"].multiply(s["x"], bias=s["bias"])


# ---- what a pass cannot do without ----

def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "norm":
        n, width = case["rows"] * case["width"], case["width"]
        vectors = (2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1)
        gates = {"none": 0, "channel": width, "row": n}[case["gate"]]
        return {"bytes": size * (4 * n + gates + vectors * width), "flops": 12 * n}
    if case["op"] == "multiply":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": outputs * (inputs // 2 + 4 * (inputs // case["group"])) + size * rows * (inputs + outputs),
                "flops": 2 * rows * inputs * outputs}
    stored = 2 * case["kv_heads"] * (case["dim"] // 2 + 4 * (case["dim"] // case["group"]))  # of one token
    if case["op"] == "append":
        tokens, dim = case["tokens"], case["dim"]
        read = (case["heads"] + 2 * case["kv_heads"]) * dim * size + 12
        return {"bytes": tokens * (2 * read + 2 * stored + 4 * case["rotary"]),
                "flops": tokens * dim * (3 * case["heads"] + 15 * case["kv_heads"])}
    lengths, counts = _lengths(case), _counts(case)
    return {"bytes": stored * sum(lengths) + 2 * size * case["heads"] * case["dim"] * sum(counts),
            "flops": 4 * case["heads"] * case["dim"] * sum(n * c - c * (c - 1) // 2 for n, c in zip(lengths, counts))}


# ---- exact values, from the definitions in 64 bits ----

def _exact_unpack(codes, scales, minimums):
    """codes [..., n / 2] of bytes, scales and minimums [..., groups]: the values, in 64 bits."""
    n = codes.shape[-1] * 2
    out = torch.empty(codes.shape[:-1] + (n,), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    group = n // scales.shape[-1]
    return out * scales.double().repeat_interleave(group, -1) + minimums.double().repeat_interleave(group, -1)


def _exact_norm(s):
    def normed(x, weight, bias):
        if s["case"]["kind"] == "layer":
            y = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + s["epsilon"])
        else:
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["epsilon"])
        return y * weight.double() + (0.0 if bias is None else bias.double())

    x = s["block"].double()
    if s["case"]["post"]:
        x = normed(x, s["post_weight"], s["post_bias"])
    gate = 1.0 if s["gate"] is None else s["gate"].double()
    hidden = s["residual"].double() * s["residual_scale"] + gate * x
    return {"hidden": hidden, "normed": normed(hidden, s["pre_weight"], s["pre_bias"])}


def _exact_append(s):
    case, half = s["case"], s["case"]["rotary"] // 2
    place = s["positions"].long()
    phase = torch.complex(s["cosines"].double()[place], s["sines"].double()[place])[:, None, :]

    def turned(x):
        x = x.double().clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        z = torch.complex(x[..., first], x[..., second]) * phase
        x[..., first], x[..., second] = z.real, z.imag
        return x

    def stored(x):
        parts = x.double().reshape(*x.shape[:-1], -1, case["group"])
        low, high = parts.min(-1, keepdim=True).values, parts.max(-1, keepdim=True).values
        m, step = low.half().double(), ((high - low) / 15).half().double()
        step = step.clamp(min=2.0 ** -24) * (high > low)  # the smallest FP16 for a range too small for it
        level = torch.where(step > 0, (parts - m) / step.clamp(min=1e-30), torch.zeros_like(parts)).round()
        return (level.clamp(0, 15) * step + m).reshape(x.shape)

    return {"queries": turned(s["queries"]), "keys": stored(turned(s["keys"])), "values": stored(s["values"])}


def _exact_attend(s):
    case, out = s["case"], []
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()
    ratio = case["heads"] // case["kv_heads"]
    for b, length in enumerate(lengths):
        pages = s["table"][b, : -(-length // case["page"])].long()

        def line(part):  # [kv_heads, length, dim]
            x = _exact_unpack(s[part + "_codes"][pages], s[part + "_scales"][pages][..., 0],
                              s[part + "_scales"][pages][..., 1])
            return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length]

        keys, values = line("key"), line("value")
        count = offsets[b + 1] - offsets[b]
        q = s["queries"][offsets[b]:offsets[b + 1]].double().reshape(count, case["kv_heads"], ratio, case["dim"])
        rows = q.permute(1, 0, 2, 3).reshape(case["kv_heads"], count * ratio, case["dim"])
        scores = torch.bmm(rows, keys.transpose(1, 2)) * s["scale"]
        own_place = torch.arange(length - count, length, device="cuda").repeat_interleave(ratio)
        hidden = torch.arange(length, device="cuda")[None, :] > own_place[:, None]
        mixed = torch.bmm(torch.softmax(scores.masked_fill(hidden, -math.inf), -1), values)
        out.append(mixed.reshape(case["kv_heads"], count, ratio, case["dim"]).transpose(0, 1).flatten(1, 2))
    return torch.cat(out)


def _exact_multiply(s):
    y = s["x"].double() @ _exact_unpack(s["codes"], s["scales"], s["minimums"]).t()
    return y if s["bias"] is None else y + s["bias"].double()


def exact(case, seed):
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend,
            "multiply": _exact_multiply}[case["op"]](prepare(case, seed))
