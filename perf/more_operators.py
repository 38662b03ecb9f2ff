"""The 8-bit token operators over the sizes they are used at: cases, their plain forms and their exact values.

Products in 8-bit integers with a scale a token and a scale a channel, the same product by experts, the routing that
chooses the experts, and the choice of the next symbol from logits. ``run`` computes each either in plain torch
operations or, where ``own`` is set, through ``nvcr_b200.tokens``.

A row x is taken as codes q = clamp(rint(x * (1 / s)), -127, 127) with s = max(max|x| * (1 / 127), 2^-126), each an
FP32 operation, and stands for q * s; a weight row is codes in int8 and an FP32 scale. Choices are made in 64 bits,
so that which expert or symbol is chosen does not hang on a rounding.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ----

def listed():
    return [
        # products: one token through a square projection; a served batch through a wide one; a long prompt; odd
        # sizes in FP32
        {"name": "product one token", "op": "product", "rows": 1, "inputs": 4096, "outputs": 4096, "bias": False,
         "type": "float16"},
        {"name": "product batch", "op": "product", "rows": 32, "inputs": 4096, "outputs": 16384, "bias": False,
         "type": "bfloat16"},
        {"name": "product prompt", "op": "product", "rows": 8192, "inputs": 4096, "outputs": 16384, "bias": False,
         "type": "bfloat16"},
        {"name": "product odd", "op": "product", "rows": 77, "inputs": 1111, "outputs": 1001, "bias": True,
         "type": "float32"},
        # experts: one token into its eight experts; a served batch out of them, weighted and summed; a prompt into
        # them, some experts far more asked for than others; odd sizes with tokens that chose fewer experts
        {"name": "experts one token", "op": "experts", "tokens": 1, "chosen": 8, "experts": 64, "inputs": 2048,
         "outputs": 1024, "sum": False, "skew": 1.0, "absent": 0.0, "type": "bfloat16"},
        {"name": "experts batch", "op": "experts", "tokens": 64, "chosen": 8, "experts": 128, "inputs": 1024,
         "outputs": 2048, "sum": True, "skew": 1.0, "absent": 0.0, "type": "bfloat16"},
        {"name": "experts prompt", "op": "experts", "tokens": 4096, "chosen": 4, "experts": 32, "inputs": 2048,
         "outputs": 4096, "sum": False, "skew": 2.0, "absent": 0.0, "type": "bfloat16"},
        {"name": "experts odd", "op": "experts", "tokens": 300, "chosen": 3, "experts": 7, "inputs": 1000,
         "outputs": 520, "sum": True, "skew": 1.0, "absent": 0.1, "type": "float16"},
        # routing: one token; a prompt with a balancing bias, by groups
        {"name": "route one token", "op": "route", "tokens": 1, "experts": 64, "count": 8, "kind": "softmax",
         "bias": False, "groups": 1, "kept": 1, "renormalise": True, "masked": 0.0, "type": "bfloat16"},
        {"name": "route prompt", "op": "route", "tokens": 16384, "experts": 256, "count": 8, "kind": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "renormalise": True, "masked": 0.0, "type": "float32"},
        # sampling: one answer's step with every filter; a served batch from a large vocabulary
        {"name": "sample one row", "op": "sample", "rows": 1, "symbols": 32768, "top_k": 50, "top_p": 0.95,
         "min_p": 0.0, "temperature": 0.8, "masked": 0.0, "type": "float32"},
        {"name": "sample batch", "op": "sample", "rows": 256, "symbols": 131072, "top_k": 0, "top_p": 0.9,
         "min_p": 0.01, "temperature": 0.7, "masked": 0.1, "type": "bfloat16"},
    ]


def _spread(rng, low, high):
    """A whole number in low..high, evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """As _spread; half of them multiples of 64."""
    n = _spread(rng, low, high)
    return max(low, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["product", "product", "experts", "experts", "route", "sample", "sample"])
    kind = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    if op == "product":
        inputs, outputs = _size(rng, 64, 16384), _size(rng, 32, 16384)
        most = max(1, min(16384, (1 << 38) // (inputs * outputs)))
        return {"op": op, "rows": _spread(rng, 1, most), "inputs": inputs, "outputs": outputs,
                "bias": rng.random() < 0.3, "type": kind}
    if op == "experts":
        experts = rng.choice([4, 8, 16, 33, 64, 128])
        chosen = rng.choice([n for n in (1, 2, 4, 6, 8) if n <= experts])
        inputs, outputs = _size(rng, 64, 4096), _size(rng, 64, 4096)
        if experts * inputs * outputs > 1 << 28:
            inputs = max(64, (1 << 28) // (experts * outputs))
        most = max(1, (1 << 35) // (inputs * outputs * chosen))
        return {"op": op, "tokens": _spread(rng, 1, min(4096, most)), "chosen": chosen, "experts": experts, "inputs": inputs,
                "outputs": outputs, "sum": rng.random() < 0.5, "skew": rng.choice([0.0, 1.0, 2.0]),
                "absent": rng.choice([0.0, 0.0, 0.1]), "type": kind}
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.choice([2, 5, 8, 16, 32])
        kept = rng.choice([n for n in (1, 2, 3, 4, 8) if n <= groups])
        count = rng.choice([n for n in (1, 2, 4, 6, 8) if n <= kept * (experts // groups)])
        return {"op": op, "tokens": _spread(rng, 1, 16384), "experts": experts, "count": count,
                "kind": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups,
                "kept": kept, "renormalise": rng.random() < 0.7, "masked": rng.choice([0.0, 0.0, 0.3]), "type": kind}
    symbols = _size(rng, 1000, 160000)
    return {"op": op, "rows": _spread(rng, 1, max(1, min(512, (1 << 25) // symbols))), "symbols": symbols,
            "top_k": rng.choice([0, 0, 1, 40, 1000]), "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
            "min_p": rng.choice([0.0, 0.0, 0.01, 0.1]), "temperature": rng.choice([0.6, 0.8, 1.0, 1.3]),
            "masked": rng.choice([0.0, 0.1, 0.5]), "type": kind}


# ---- what the program has in hand ----

def _normal(shape, make, spread=1.0):
    return torch.randn(shape, generator=make, device="cuda", dtype=torch.float32) * spread


def _uniform(shape, make):
    return torch.rand(shape, generator=make, device="cuda", dtype=torch.float32)


def _weights(shape, make):
    """Weight rows in 8 bits: codes and scales. The codes are spread as a normal's are, the row's largest at 127."""
    codes = (torch.randn(shape, generator=make, device="cuda", dtype=torch.float16) * 34.0).clamp(-127, 127)
    scales = (_uniform(shape[:-1], make) + 0.5) * (shape[-1] ** -0.5 / 34.0)
    return codes.round().to(torch.int8), scales


def _activations(shape, make, kind):
    x = _normal(shape, make)
    x[..., :: max(1, shape[-1] // 8)] *= 10.0  # activations have a few channels of large values
    return x.to(kind)


def _prepare_product(case, make):
    kind, outputs = TYPES[case["type"]], case["outputs"]
    codes, scales = _weights((outputs, case["inputs"]), make)
    return {"x": _activations((case["rows"], case["inputs"]), make, kind), "codes": codes, "scales": scales,
            "bias": _normal((outputs,), make, 0.1).to(kind) if case["bias"] else None}


def _prepare_experts(case, make):
    tokens, chosen, experts = case["tokens"], case["chosen"], case["experts"]
    codes, scales = _weights((experts, case["outputs"], case["inputs"]), make)
    # the experts that a token's scores are highest for; some experts' are higher for every token
    liking = _normal((tokens, experts), make) + _normal((1, experts), make, case["skew"])
    choices = liking.topk(chosen, -1).indices.to(torch.int32)
    choices = torch.where(_uniform((tokens, chosen), make) < case["absent"], torch.full_like(choices, -1), choices)
    # tokens enter their experts once for all of them, and leave each with a row of its own
    shape = (tokens, chosen, case["inputs"]) if case["sum"] else (tokens, case["inputs"])
    return {"x": _activations(shape, make, TYPES[case["type"]]), "codes": codes, "scales": scales, "choices": choices,
            "weights": torch.softmax(_normal((tokens, chosen), make), -1) if case["sum"] else None}


def _prepare_route(case, make):
    shape = (case["tokens"], case["experts"])
    scores = _normal(shape, make, 1.5).to(TYPES[case["type"]])
    scores = scores.masked_fill(_uniform(shape, make) < case["masked"], -math.inf)
    return {"scores": scores, "bias": _normal((case["experts"],), make, 0.05) if case["bias"] else None, "scale": 1.5}


def _prepare_sample(case, make):
    rows, symbols = case["rows"], case["symbols"]
    # a broad bulk and a tail of likely symbols; some rows are surer than others
    logits = _normal((rows, symbols), make) * (_uniform((rows, 1), make) + 1.5)
    logits = logits + torch.relu(_normal((rows, symbols), make) - 2.5) * 6.0
    logits = logits.to(TYPES[case["type"]]).masked_fill_(_uniform((rows, symbols), make) < case["masked"], -math.inf)
    each = lambda value, kind: torch.full((rows,), value, dtype=kind, device="cuda")  # noqa: E731
    return {"logits": logits, "uniforms": _uniform((rows,), make), "top_k": each(case["top_k"], torch.int32),
            "top_p": each(case["top_p"], torch.float32), "min_p": each(case["min_p"], torch.float32),
            "temperature": each(case["temperature"], torch.float32)}


def prepare(case, seed):
    make = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"product": _prepare_product, "experts": _prepare_experts, "route": _prepare_route,
             "sample": _prepare_sample}[case["op"]](case, make)
    state["case"] = case
    if own:
        from nvcr_b200 import tokens

        if case["op"] == "product":
            state["matrix"] = tokens.ByteMatrix(state["codes"], state["scales"])
        if case["op"] == "experts":
            state["matrix"] = tokens.ByteExperts(state["codes"], state["scales"])
    return state


# ---- one pass ----

def _plain_codes(x):
    """Rows as codes (whole numbers in FP32) and scales."""
    x = x.float()
    scales = (x.abs().amax(-1, keepdim=True) * (1.0 / 127.0)).clamp(min=2.0 ** -126)
    return torch.round(x * (1.0 / scales)).clamp(-127.0, 127.0), scales


def _plain_product(s):
    codes, scales = _plain_codes(s["x"])
    y = codes @ s["codes"].float().t() * s["scales"] * scales
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _plain_experts(s):
    choices, experts = s["choices"], s["case"]["experts"]
    tokens, chosen = choices.shape
    codes, scales = _plain_codes(s["x"])
    if codes.dim() == 2:
        codes, scales = (v.unsqueeze(1).expand(tokens, chosen, -1) for v in (codes, scales))
    # every expert's rows beside one another, then one product of all experts
    pairs = choices.flatten().long()
    order = torch.sort(pairs, stable=True).indices
    counts = torch.bincount(pairs + 1, minlength=experts + 1)
    first = torch.cumsum(counts, 0) - counts
    group = pairs[order]
    place = torch.arange(tokens * chosen, device="cuda") - first[group + 1]
    here = group >= 0
    order, group, place = order[here], group[here], place[here]
    rows = torch.zeros((experts, int(counts[1:].max()), s["case"]["inputs"]), device="cuda")
    rows[group, place] = codes.reshape(tokens * chosen, -1)[order]
    products = torch.bmm(rows, s["codes"].float().transpose(1, 2)) * s["scales"].unsqueeze(1)
    y = torch.zeros((tokens * chosen, s["case"]["outputs"]), device="cuda")
    y[order] = products[group, place] * scales.reshape(-1, 1)[order]
    y = y.view(tokens, chosen, -1)
    return (y if s["weights"] is None else (y * s["weights"].unsqueeze(-1)).sum(1)).to(s["x"].dtype)


def _plain_route(s):
    case, scores = s["case"], s["scores"].double()
    seen = scores > -math.inf
    if case["kind"] == "sigmoid":
        share = 1.0 / (1.0 + torch.exp(-scores))
    else:
        top = scores.amax(-1, keepdim=True)
        share = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
        total = share.sum(-1, keepdim=True)
        share = share / torch.where(total > 0, total, torch.ones_like(total))
    ranked = share if s["bias"] is None else share + s["bias"].double()
    ranked = torch.where(seen, ranked, -math.inf)
    if case["kept"] < case["groups"]:
        grouped = ranked.unflatten(-1, (case["groups"], -1))
        two = grouped.sort(dim=-1, descending=True).values[..., :2]
        value = torch.where(two > -math.inf, two, 0.0).sum(-1).masked_fill(two[..., 0] == -math.inf, -math.inf)
        place = value.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
        ranked = torch.where((place < case["kept"]).unsqueeze(-1), grouped, -math.inf).flatten(-2)
    value, choices = (v[..., : case["count"]] for v in ranked.sort(dim=-1, descending=True, stable=True))
    there = value > -math.inf
    weights = torch.where(there, share.gather(-1, choices), 0.0)
    if case["renormalise"]:
        total = weights.sum(-1, keepdim=True)
        weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    return {"choices": torch.where(there, choices, -1).to(torch.int32), "weights": (weights * s["scale"]).float()}


def _plain_sample(s):
    logits = s["logits"].double()
    top = logits.amax(-1, keepdim=True)
    some = top > -math.inf
    shares = torch.exp((logits - torch.where(some, top, 0.0)) / s["temperature"].double().unsqueeze(-1))
    ranked, order = logits.sort(dim=-1, descending=True, stable=True)
    sorted_shares = shares.gather(-1, order)
    nth = torch.arange(logits.shape[-1], device="cuda")
    most = s["top_k"].long().unsqueeze(-1)
    keep = (ranked > -math.inf) & ((nth < most) | (most <= 0))
    sums = torch.cumsum(torch.where(keep, sorted_shares, 0.0), -1)
    p = s["top_p"].double().unsqueeze(-1)
    reached = torch.cat((torch.zeros_like(p), sums[:, :-1]), -1) >= p * sums[:, -1:]  # before this one
    keep = keep & (~reached | (p >= 1.0) | (nth == 0)) & (sorted_shares >= s["min_p"].double().unsqueeze(-1))
    kept = torch.zeros_like(shares).scatter_(-1, order, torch.where(keep, sorted_shares, 0.0))
    sums = torch.cumsum(kept, -1)
    wanted = s["uniforms"].double().unsqueeze(-1) * sums[:, -1:]
    symbol = (sums > wanted).byte().argmax(-1, keepdim=True)
    probability = kept.gather(-1, symbol) / torch.where(some, sums[:, -1:], 1.0)
    return {"symbols": torch.where(some, symbol, -1).squeeze(-1), "probabilities": probability.float().squeeze(-1)}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"product": _plain_product, "experts": _plain_experts, "route": _plain_route,
                "sample": _plain_sample}[case["op"]](s)
    if case["op"] == "product":
        return s["matrix"].multiply(s["x"], bias=s["bias"])
    if case["op"] == "experts":
        return s["matrix"].multiply(s["x"], s["choices"], weights=s["weights"])
    from nvcr_b200 import tokens

    if case["op"] == "route":
        choices, weights = tokens.route(s["scores"], case["count"], kind=case["kind"], bias=s["bias"],
                                        groups=case["groups"], kept_groups=case["kept"],
                                        renormalise=case["renormalise"], scale=s["scale"])
        return {"choices": choices, "weights": weights}
    symbols, probabilities = tokens.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                           top_p=s["top_p"], min_p=s["min_p"])
    return {"symbols": symbols, "probabilities": probabilities}


# ---- what a pass cannot do without ----

def _asked_for(case):
    """How many experts some token is expected to have chosen, each as likely as another."""
    pairs = case["tokens"] * case["chosen"]
    return case["experts"] * (1.0 - (1.0 - 1.0 / case["experts"]) ** pairs)


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "product":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": outputs * (inputs + 4 + (size if case["bias"] else 0)) + size * rows * (inputs + outputs),
                "flops": 2 * rows * inputs * outputs}
    if case["op"] == "experts":
        tokens, pairs, inputs, outputs = (case["tokens"], case["tokens"] * case["chosen"], case["inputs"],
                                          case["outputs"])
        rows = pairs * inputs + tokens * outputs if case["sum"] else tokens * inputs + pairs * outputs
        return {"bytes": _asked_for(case) * outputs * (inputs + 4) + size * rows + 8 * pairs,
                "flops": 2 * pairs * inputs * outputs}
    if case["op"] == "route":
        n = case["tokens"] * case["experts"]
        return {"bytes": size * n + 8 * case["tokens"] * case["count"], "flops": 20 * n}
    n = case["rows"] * case["symbols"]
    return {"bytes": size * n + 28 * case["rows"], "flops": 20 * n}


# ---- exact values, from the definitions in 64 bits ----

def _exact_rows(x):
    """What rows stand for in 8 bits. Their scales and codes are FP32 by definition; the values are in 64 bits."""
    x = x.to(torch.float32)
    largest = torch.maximum(x.max(-1).values, -x.min(-1).values)
    step = torch.clamp_min(largest * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device), 2.0 ** -126)
    inverse = torch.reciprocal(step)
    return (x * inverse[..., None]).round().clamp(-127, 127).double() * step.double()[..., None]


def _exact_product(s):
    y = torch.einsum("tk,nk->tn", _exact_rows(s["x"]), s["codes"].double() * s["scales"].double()[:, None])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_experts(s):
    choices, out = s["choices"].long(), None
    tokens, chosen = choices.shape
    x = _exact_rows(s["x"])
    out = torch.zeros((tokens, chosen, s["case"]["outputs"]), dtype=torch.float64, device="cuda")
    for expert in range(s["case"]["experts"]):
        token, nth = torch.nonzero(choices == expert, as_tuple=True)
        if len(token):
            rows = x[token] if x.dim() == 2 else x[token, nth]
            matrix = s["codes"][expert].double() * s["scales"][expert].double()[:, None]
            out[token, nth] = rows @ matrix.t()
    return out if s["weights"] is None else torch.einsum("tjn,tj->tn", out, s["weights"].double())


def _exact_route(s):
    case = s["case"]
    scores = s["scores"].double().cpu().numpy()
    if case["kind"] == "sigmoid":
        share = np.exp(-np.logaddexp(0.0, -scores))
    else:
        with np.errstate(invalid="ignore"):
            share = np.exp(scores - np.logaddexp.reduce(scores, -1, keepdims=True))
        share = np.where(np.isneginf(scores), 0.0, share)
    ranked = share + (0.0 if s["bias"] is None else s["bias"].double().cpu().numpy())
    ranked[np.isneginf(scores)] = -np.inf
    choices = np.full((len(scores), case["count"]), -1, dtype=np.int32)
    weights = np.zeros((len(scores), case["count"]))
    size = case["experts"] // case["groups"]
    for t, row in enumerate(ranked):
        if case["kept"] < case["groups"]:
            pairs = np.sort(row.reshape(-1, size), -1)[:, ::-1][:, :2]
            best = [sum(v for v in p if v > -np.inf) if p[0] > -np.inf else -np.inf for p in pairs]
            for g in np.argsort([-v for v in best], kind="stable")[case["kept"]:]:
                row[g * size:(g + 1) * size] = -np.inf
        first = np.argsort(-row, kind="stable")[: case["count"]]
        first = first[row[first] > -np.inf]
        choices[t, : len(first)], weights[t, : len(first)] = first, share[t, first]
        total = weights[t].sum()
        if case["renormalise"] and total > 0:
            weights[t] /= total
    return {"choices": choices, "weights": weights * s["scale"]}


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    symbols, probabilities = [], []
    for r, row in enumerate(logits):
        index = np.flatnonzero(row > -np.inf)
        if not len(index):
            symbols.append(-1), probabilities.append(0.0)
            continue
        k, p = int(s["top_k"][r]), float(s["top_p"][r])
        index = index[np.argsort(-row[index], kind="stable")]
        index = index[: k if k > 0 else None]
        share = np.exp((row[index] - row[index[0]]) / float(s["temperature"][r]))
        n = len(index)
        if p < 1.0:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(share), p * share.sum())))
        n = min(n, int((share >= float(s["min_p"][r])).sum()))
        index, share = index[:n], share[:n]
        in_order = np.argsort(index)
        sums = np.cumsum(share[in_order])
        at = in_order[min(n - 1, int(np.searchsorted(sums, float(s["uniforms"][r]) * sums[-1], side="right")))]
        symbols.append(int(index[at])), probabilities.append(share[at] / sums[-1])
    return {"symbols": np.array(symbols, dtype=np.int64), "probabilities": np.array(probabilities)}


def exact(case, seed):
    return {"product": _exact_product, "experts": _exact_experts, "route": _exact_route,
            "sample": _exact_sample}[case["op"]](prepare(case, seed))
