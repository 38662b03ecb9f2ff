"""The token operators on the GPU against plain implementations in 64 bits.

Tolerances are error bounds of the operators' arithmetic, derived here:
* an output of a type with unit roundoff u (2^-11, 2^-8, 2^-24 for float16,
  bfloat16, float32) is rounded once: u |y|, and 2^-25 absolute for a float16
  below its normal range;
* a sum of FP32 terms in d steps is off by at most d 2^-24 of the sum of their
  magnitudes; tensor-core sums of 16 terms are taken at 2^-23 a step;
* softmax weights may be rounded to FP16 (2^-11), and an error e of a score
  changes a weight by a factor of up to 1 + 2 e;
* products with bfloat16 may hold a code as 128 + c (exact in bfloat16), whose
  offset leaves the sum again within its group.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def kind_of(name):
    import torch

    return getattr(torch, name)


def near(got, want, tolerance, name):
    """Every element of `got` within `tolerance` (elementwise) of `want`, non-finite ones alike."""
    import torch

    got = got.double()
    unit = UNIT[name]
    limit = tolerance + unit * want.abs() * 1.001 + (2.0 ** -25 if name == "float16" else 0.0)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = torch.where(finite, (got - want).abs() - limit, torch.zeros_like(want))
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0.0, (
        f"element {worst} of {off.numel()}: {got.flatten()[worst]} for {want.flatten()[worst]}, "
        f"{int((off > 0).sum())} outside")


def normal(shape, seed, spread=1.0, mean=0.0):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=make, device="cuda", dtype=torch.float32) * spread + mean


# ---- norms ----

def plain_normed(x, weight, bias, layer, epsilon, offset):
    import torch

    if layer:
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon)
    if weight is not None:
        x = x * (weight.double() + offset)
    return x if bias is None else x + bias.double()


def check_norm(block, residual=None, gate=None, post=False, weights=(None,) * 4, layer=False, scale=1.0, offset=0.0,
               epsilon=1e-6, **more):
    from nvcr_b200 import tokens

    name = str(block.dtype).removeprefix("torch.")
    hidden, normed = tokens.block_norm(
        block, residual=residual, gate=gate, post=post, post_weight=weights[0], post_bias=weights[1],
        pre_weight=weights[2], pre_bias=weights[3], kind="layer" if layer else "rms", residual_scale=scale,
        weight_offset=offset, epsilon=epsilon, **more)
    width = block.shape[1]
    x = block.double()
    p = plain_normed(x, weights[0], weights[1], layer, epsilon, offset) if post else x
    g = 1.0 if gate is None else gate.double()
    r = 0.0 if residual is None else residual.double() * scale
    want = r + g * p
    # every FP32 step is at most 16 + width / 32 sums deep; a norm's error is relative to what it subtracts and adds
    step = (16 + width / 32) * 2.0 ** -24
    size = lambda v, w, b: ((v.abs() + (v.mean(-1, keepdim=True).abs() if layer else 0.0))  # noqa: E731
                            / ((v - v.mean(-1, keepdim=True) if layer else v).square().mean(-1, keepdim=True)
                               + epsilon).sqrt() * (1.0 if w is None else (w.double().abs() + abs(offset)))
                            + (0.0 if b is None else b.double().abs()))
    terms = (abs(r) if residual is not None else 0.0) + (abs(g) if gate is not None else 1.0) * (
        size(x, weights[0], weights[1]) if post else x.abs())
    if hidden is not None:
        near(hidden, want, step * terms, name)
    if normed is not None:
        after = plain_normed(want, weights[2], weights[3], layer, epsilon, offset)
        spread = ((want - want.mean(-1, keepdim=True)) if layer else want).square().mean(-1, keepdim=True)
        # an error d of the sum moves the norm by d / root, and by that of the whole row's through the root
        each = step * terms / (spread + epsilon).sqrt()
        each = each + each.square().mean(-1, keepdim=True).sqrt() * (1.0 + size(want, None, None))
        w = 1.0 if weights[2] is None else weights[2].double().abs() + abs(offset)
        near(normed, after, 2 * each * w + step * size(want, weights[2], weights[3]), name)
    return hidden, normed


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (1, 2048), (77, 1111), (5, 4096), (130, 64), (2, 16384),
                                        (2, 20001), (700, 256), (3, 33000)])
def test_norm(cuda, name, rows, width):
    kind = kind_of(name)
    block, residual = normal((rows, width), 1, 0.7, 0.2).to(kind), normal((rows, width), 2, 3.0, -0.5).to(kind)
    weights = [normal((width,), 10 + i, 0.3, 1.0 if i % 2 == 0 else 0.0).to(kind) for i in range(4)]
    channel, rowwise = normal((width,), 3, 0.5, 0.5).to(kind), normal((rows, width), 4, 0.5, 0.5).to(kind)
    check_norm(block, residual, channel, True, weights, False, 0.875)
    check_norm(block, residual, rowwise, True, weights, True, 1.0)
    check_norm(block, residual, None, False, (None, None, weights[2], None), False, 0.5, offset=1.0)
    check_norm(block, None, rowwise, True, (None, None, None, None), False, 1.0)
    check_norm(block, None, None, False, (None, None, weights[2], weights[3]), True, 1.0)


@pytest.mark.parametrize("name", ["float16", "float32"])
def test_norm_strides_parts_and_place(cuda, name):
    import torch

    from nvcr_b200 import tokens

    kind = kind_of(name)
    for width, first, pad in ((256, 0, 64), (256, 3, 64), (250, 0, 7)):
        wide = normal((9, width + pad), 5).to(kind)
        block, residual = wide[:, first:first + width], normal((9, width + pad), 6).to(kind)[:, first:first + width]
        gate = normal((18, width), 7).to(kind)[::2]
        weight = normal((width + 1,), 8, 0.2, 1.0).to(kind)
        check_norm(block, residual, gate, True, (weight[1:], None, weight[:-1], None), False, 1.0)
        check_norm(block, residual, gate, True, (weight[1:], None, weight[:-1], None), False, 1.0, normed=False)
        _, alone = check_norm(block, residual, gate, True, (weight[1:], None, weight[:-1], None), False, 1.0,
                              hidden=False)
        _, both = tokens.block_norm(block, residual=residual, gate=gate, post=True, post_weight=weight[1:],
                                    pre_weight=weight[:-1])
        assert torch.equal(alone, both)
    hidden, normed = tokens.block_norm(torch.zeros((0, 64), dtype=kind, device="cuda"))
    assert hidden.shape == normed.shape == (0, 64)


def test_norm_in_place(cuda):
    import torch

    from nvcr_b200.executor import _check, library
    from nvcr_b200 import tokens

    for width in (512, 500, 20000):
        block, residual = normal((6, width), 1).half(), normal((6, width), 2).half()
        hidden, normed = tokens.block_norm(block, residual=residual, post=True)
        _check(library().nvcr_sm100_token_norm(0, 0, 1, block.data_ptr(), width, residual.data_ptr(), width, None, 0,
                                               None, None, None, None, residual.data_ptr(), block.data_ptr(), 6, width,
                                               1.0, 0.0, 1e-6, None))
        torch.cuda.synchronize()
        assert torch.equal(residual, hidden) and torch.equal(block, normed)


def test_norm_of_extreme_rows(cuda):
    """A zero row gives its biases, a NaN or an infinity stays in its row, and large values do not overflow inside."""
    import torch

    from nvcr_b200 import tokens

    block = normal((6, 1000), 1).half()
    block[1] = 0.0
    block[2, 3] = float("nan")
    block[3, 5] = float("inf")
    block[4] = 60000.0 * block[4].sign()
    hidden, normed = tokens.block_norm(block)
    assert torch.equal(normed[1], torch.zeros_like(normed[1]))
    assert normed[2].isnan().all() and hidden[2].isnan().sum() == 1
    assert normed[3].isnan().sum() == 1 and normed[3, 0] == 0
    good = [0, 1, 4, 5]
    near(normed[good], plain_normed(block[good].double(), None, None, False, 1e-6, 0.0),
         torch.full((4, 1000), 2.0 ** -18, dtype=torch.float64, device="cuda"), "float16")


# ---- the cache ----

def make_tables(rows, rotary):
    import torch

    angles = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64),
                         10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary))
    return angles.cos().float(), angles.sin().float()


def plain_rotated(x, cosines, sines, interleaved):
    import torch

    x = x.double().clone()
    half = cosines.shape[1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, s = cosines.double()[:, None], sines.double()[:, None]
    first, second = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = first, second
    else:
        x[..., :half], x[..., half:2 * half] = first, second
    return x


def quantised_fp32(x, group):
    """The header's formula in FP32 on the host: (codes, scales, minimums) as NumPy arrays."""
    parts = x.reshape(x.shape[:-1] + (-1, group)).astype(np.float32)
    low, high = parts.min(-1), parts.max(-1)
    with np.errstate(all="ignore"):
        minimums = low.astype(np.float16)
        scales = ((high - low) * np.float32(1.0 / 15.0)).astype(np.float16)
        scales = np.where((scales == 0) & (high > low), np.float16(2.0 ** -24), scales)
        s, m = scales.astype(np.float32)[..., None], minimums.astype(np.float32)[..., None]
        level = np.where(s > 0, np.rint((parts - m) / np.where(s > 0, s, 1).astype(np.float32)), np.float32(0))
        level = np.where(np.isnan(level), 0, np.clip(level, 0, 15))
    return level.astype(np.uint8).reshape(x.shape), scales, minimums


def places(cache, slots):
    """(codes, scales, minimums) stored for keys and for values at slots, per token and head."""
    import torch

    page, within = slots // cache.page_size, slots % cache.page_size
    found = []
    for codes, scales in (cache.tensors[:2], cache.tensors[2:]):
        c, s = codes[page, :, within], scales[page, :, within]
        found.append((torch.stack((c & 15, c >> 4), -1).flatten(-2), s[..., 0], s[..., 1]))
    return found


APPENDS = [  # dim, group, kv_heads, heads, page, tokens, rotary, interleaved, type
    (128, 64, 8, 32, 16, 1, 128, False, "float16"),
    (128, 32, 2, 6, 48, 77, 128, True, "bfloat16"),
    (128, 128, 3, 3, 16, 50, 64, False, "bfloat16"),
    (64, 64, 1, 5, 32, 333, 64, True, "float16"),
    (64, 32, 4, 4, 64, 19, 30, False, "float16"),
    (256, 128, 2, 4, 16, 33, 256, False, "bfloat16"),
    (256, 64, 1, 16, 128, 200, 130, True, "float16"),
]


@pytest.mark.parametrize("dim,group,kv_heads,heads,page,tokens,rotary,interleaved,name", APPENDS)
def test_append_and_read(cuda, dim, group, kv_heads, heads, page, tokens, rotary, interleaved, name):
    check_append(dim, group, kv_heads, heads, page, tokens, rotary, interleaved, name, 1)


@pytest.mark.parametrize("dim,group,kv_heads,heads,page,tokens,rotary,interleaved,name", APPENDS + [
    (128, 64, 8, 32, 16, 2000, 128, False, "bfloat16"),
    (128, 32, 4, 20, 64, 700, 32, False, "float16"),
    (256, 64, 2, 2, 16, 65, 16, False, "bfloat16"),
    (64, 32, 2, 8, 32, 500, 8, True, "float16"),
    (256, 128, 1, 3, 16, 9, 128, True, "bfloat16"),
])
def test_append_and_read_aligned(cuda, dim, group, kv_heads, heads, page, tokens, rotary, interleaved, name):
    check_append(dim, group, kv_heads, heads, page, tokens, rotary, interleaved, name, 0)


def check_append(dim, group, kv_heads, heads, page, tokens, rotary, interleaved, name, pad):
    import torch

    from nvcr_b200.tokens import PagedCache

    kind = kind_of(name)
    pages = -(-tokens // page) + 2
    cache = PagedCache.empty(pages, kv_heads, page, dim, group)
    for i, t in enumerate(cache.tensors):
        t.view(torch.uint8).fill_(17 + i)
    before = [t.clone() for t in cache.tensors]
    rows = normal((tokens, heads + 2 * kv_heads, dim + pad), 3, 1.5, 0.3).to(kind)[:, :, pad:]  # 1: odd strides and start
    queries, keys, values = rows.split([heads, kv_heads, kv_heads], 1)
    make = torch.Generator(device="cuda").manual_seed(4)
    slots = torch.randperm(pages * page, generator=make, device="cuda")[:tokens]
    padding = torch.arange(tokens, device="cuda") % 5 == 4
    slots = torch.where(padding, -1 - slots, slots)
    positions = torch.randint(0, 5000, (tokens,), generator=make, device="cuda", dtype=torch.int32)
    cosines, sines = make_tables(5000, rotary)
    rotated = cache.append(keys, values, slots, queries=queries, positions=positions, cosines=cosines, sines=sines,
                           interleaved=interleaved)
    at = positions.long()
    want = plain_rotated(queries, cosines[at], sines[at], interleaved)
    size = 1.5 * queries.double().abs().amax(-1, keepdim=True)  # |a cos| + |b sin| at most
    near(rotated, want, (3 * 2.0 ** -24 * size).expand_as(want), name)
    assert torch.equal(rotated[..., rotary:], queries[..., rotary:])

    stored = slots[~padding]
    exact = (plain_rotated(keys, cosines[at], sines[at], interleaved)[~padding], values[~padding].double())
    got = places(cache, stored)
    read = cache.read(slots, torch.float32)
    for (codes, scales, minimums), x, back in zip(got, exact, read):
        assert int(codes.max()) <= 15
        parts = x.unflatten(-1, (-1, group))
        low, high = parts.amin(-1), parts.amax(-1)
        turn = 2.0 ** -22 * x.abs().amax(-1, keepdim=True)  # of the rotation in FP32
        s, m = scales.double(), minimums.double()
        assert ((m - low).abs() <= 2.0 ** -11 * low.abs() * 1.001 + 2.0 ** -25 + turn).all()
        assert ((s - (high - low) / 15).abs() <= 2.0 ** -11 * (high - low) / 15 * 1.001 + 2.0 ** -25 + turn).all()
        values_of = (codes.double().unflatten(-1, (-1, group)) * s[..., None] + m[..., None])
        # half a step, or at the ends what the rounded range misses (15 2^-11 of a step, and the minimum's rounding)
        limit = s * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -12) + 2.0 ** -11 * low.abs() + 2 * turn + 2.0 ** -19
        assert ((values_of - parts).abs() <= limit[..., None]).all()
        assert torch.equal(back[~padding].double(), values_of.flatten(-2).float().double())
        assert torch.count_nonzero(back[padding]) == 0
    # the bytes are the header's formula in FP32, and nothing else was written
    cpu = {n: t.float().cpu().numpy() for n, t in (("k", keys), ("v", values), ("c", cosines[at]), ("s", sines[at]))}
    turned, half = cpu["k"].copy(), rotary // 2
    c, s = cpu["c"][:, None], cpu["s"][:, None]
    one, two = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
    a, b = cpu["k"][..., one], cpu["k"][..., two]
    turned[..., one], turned[..., two] = a * c - b * s, b * c + a * s
    keep = ~padding.cpu().numpy()
    for (codes, scales, minimums), x in zip(got, (turned[keep], cpu["v"][keep])):
        want_codes, want_scales, want_minimums = quantised_fp32(x, group)
        assert np.array_equal(scales.cpu().numpy(), want_scales)
        assert np.array_equal(minimums.cpu().numpy(), want_minimums)
        assert np.array_equal(codes.cpu().numpy(), want_codes)
    mask = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    mask[stored] = True
    mask = mask.view(pages, 1, page).expand(pages, kv_heads, page)
    for t, old in zip(cache.tensors, before):
        assert torch.equal(t[~mask].view(torch.uint8), old[~mask].view(torch.uint8))
    cache.check()
    for dtype in (torch.float16, torch.bfloat16):
        for again, full in zip(cache.read(slots, dtype), read):
            near(again, full.double(), 2.0 ** -24 * full.double().abs(), str(dtype).removeprefix("torch."))


def test_append_extremes(cuda):
    """Constant groups, NaN, infinity, values past FP16, tokens without queries or rotation, none at all."""
    import torch

    from nvcr_b200.tokens import PagedCache

    cache = PagedCache.empty(2, 1, 16, 128, 32)
    keys, values = normal((6, 1, 128), 1).bfloat16(), normal((6, 1, 128), 2).bfloat16()
    keys[0] = 2.5
    values[0] = 0.0
    keys[1, 0, 40] = float("nan")
    values[2, 0, 70] = float("inf")
    values[3, 0, 0] = 3e38
    keys[4] = torch.linspace(-65504, 65504, 128, device="cuda").bfloat16()
    keys[4] = keys[4].clamp(-65280, 65280)
    keys[5] *= 1e-7
    slots = torch.arange(6, device="cuda") * 5
    assert cache.append(keys, values, slots) is None
    assert cache.append(keys[:0], values[:0], slots[:0]) is None
    k, v = cache.read(slots, torch.float32)
    assert torch.equal(k[0], torch.full_like(k[0], 2.5)) and torch.count_nonzero(v[0]) == 0
    assert k[1, 0, 32:64].isnan().all() and not k[1, 0, :32].isnan().any() and not k[1, 0, 64:].isnan().any()
    assert not torch.isfinite(v[2, 0, 64:96]).any() and torch.isfinite(v[2, 0, :64]).all()
    assert not torch.isfinite(v[3, 0, :32]).any() and torch.isfinite(v[3, 0, 32:]).all()
    assert torch.isfinite(k[4]).all() and torch.isfinite(k[5]).all()
    assert (k[4, 0] - keys[4, 0].float()).abs().max() <= 65536.0 * 2 / 4 / 15
    assert (k[5] - keys[5].float()).abs().max() <= 2.0 ** -24 * 1.01
    empty, _ = cache.read(slots[:0])
    assert empty.shape == (0, 1, 128)


def test_out_of_range_tokens_are_left_out_and_told(cuda):
    import torch

    from nvcr_b200.executor import ErrorCode, ExecutorError
    from nvcr_b200.tokens import PagedCache

    cache = PagedCache.empty(2, 2, 16, 64, 32)
    before = [t.clone() for t in cache.tensors]
    x = normal((3, 2, 64), 1).half()
    cosines, sines = make_tables(10, 64)
    good = torch.tensor([1, 2, 3], device="cuda")

    def told(what):
        with pytest.raises(ExecutorError) as error:
            cache.check()
        assert error.value.code == ErrorCode.invalid_argument and what in error.value.message
        cache.check()

    cache.append(x, x, torch.tensor([32, 1 << 40, 33], device="cuda"))
    told("slot")
    positions = torch.tensor([10, -1, 1 << 30], dtype=torch.int32, device="cuda")
    rotated = cache.append(x, x, good, queries=x, positions=positions, cosines=cosines, sines=sines)
    told("position")
    assert rotated.isnan().all()
    for t, old in zip(cache.tensors, before):
        assert torch.equal(t, old)
    k, v = cache.read(torch.tensor([32, 1 << 40], device="cuda"))
    told("slot")
    assert torch.count_nonzero(k) == 0 and torch.count_nonzero(v) == 0


# ---- attention ----

class Sequences:
    """A filled cache with shuffled pages, NaN scales and wild page numbers past each sequence's end."""

    def __init__(self, lengths, dim, group, kv_heads, page, seed=1, spread=1.0, pages=None):
        import torch

        from nvcr_b200.tokens import PagedCache

        make = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.page = lengths, page
        need = [-(-n // page) for n in lengths]
        columns = max(max(need), 1) + 1
        pages = sum(need) + 1 if pages is None else pages
        shape = (pages, kv_heads, page)
        if pages * kv_heads * page * dim < 1 << 28:
            codes = [torch.randint(0, 256, shape + (dim // 2,), generator=make, device="cuda").to(torch.uint8)
                     for _ in range(2)]
            scales = [torch.full(shape + (dim // group, 2), float("nan"), dtype=torch.float16, device="cuda")
                      for _ in range(2)]
        else:
            codes = [torch.empty(shape + (dim // 2,), dtype=torch.uint8, device="cuda") for _ in range(2)]
            scales = [torch.empty(shape + (dim // group, 2), dtype=torch.float16, device="cuda") for _ in range(2)]
        self.table = torch.full((len(lengths), columns), -7, dtype=torch.int32, device="cuda")
        self.table[:, 1::2] = 1 << 30
        # the last pages of the cache, in shuffled order
        order = pages - 1 - torch.randperm(sum(need), generator=make, device="cuda")
        self.slots, at = [], 0
        for b, n in enumerate(lengths):
            mine = order[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = mine.to(torch.int32)
            t = torch.arange(n, device="cuda")
            self.slots.append(mine[t // page] * page + t % page)
            for c, s in zip(codes, scales):
                c[mine] = torch.randint(0, 256, (len(mine), kv_heads, page, dim // 2), generator=make,
                                        device="cuda").to(torch.uint8)
                step = (torch.rand((n, kv_heads, dim // group), generator=make, device="cuda") + 0.05) * 0.25 * spread
                low = -step * (7.5 + torch.randn(step.shape, generator=make, device="cuda"))
                s[mine] = float("nan")
                s[mine[t // page], :, t % page] = torch.stack((step, low), -1).half()
        self.cache = PagedCache(codes[0], scales[0], codes[1], scales[1])
        self.lengths_on_device = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def line(self, b, codes, scales):
        """codes * scale and minimums of one sequence, [n, kv_heads, dim] each, in 64 bits."""
        import torch

        page, within = self.slots[b] // self.page, self.slots[b] % self.page
        c, s = codes[page, :, within], scales[page, :, within].double()
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2).double().unflatten(-1, (s.shape[-2], -1))
        return (c * s[..., 0:1]).flatten(-2), (0 * c + s[..., 1:2]).flatten(-2)

    def check(self, queries, counts, out, scale, name):
        """Every row against the formula in 64 bits."""
        import torch

        kv_heads, dim = self.cache.kv_heads, self.cache.head_dim
        ratio, first = queries.shape[1] // kv_heads, 0
        for b, (n, count) in enumerate(zip(self.lengths, counts)):
            q = queries[first:first + count].double().unflatten(1, (kv_heads, ratio))
            got = out[first:first + count]
            first += count
            if count == 0:
                continue
            ks, km = self.line(b, *self.cache.tensors[:2])
            vs, vm = self.line(b, *self.cache.tensors[2:])
            scores = torch.einsum("ihgd,thd->ihgt", q, ks + km) * scale
            seen = torch.arange(n, device="cuda") <= torch.arange(n - count, n, device="cuda")[:, None]
            seen = seen[:, None, None, :]
            scores = scores.masked_fill(~seen, -math.inf)
            top = scores.amax(-1, keepdim=True) if n else scores.new_full((count, kv_heads, ratio, 1), -math.inf)
            weights = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
            total = weights.sum(-1, keepdim=True)
            weights = weights / torch.where(total > 0, total, torch.ones_like(total))
            want = torch.einsum("ihgt,thd->ihgd", weights, vs + vm).flatten(1, 2)
            # a score's error: FP32 sums of dim products, at most 15 s + |m| each, and one of the final scaling
            size = torch.einsum("ihgd,thd->ihgt", q.abs(), ks.abs() + km.abs()) * abs(scale)
            slip = float(((dim / 16 + 24) * 2.0 ** -23 * torch.where(seen, size, 0.0)).max()) if n else 0.0
            share = 2.0 ** -11 + 2 * slip + (n / 16 + 64) * 2.0 ** -23 + 2.0 ** -20
            bound = torch.einsum("ihgt,thd->ihgd", weights, vs.abs() + vm.abs()).flatten(1, 2)
            near(got, want, share * bound, name)


def attend(seqs, counts, heads, name, scale=None, seed=7, spread=1.0, offsets=True, **more):
    import torch

    from nvcr_b200.tokens import TokenContext

    dim = seqs.cache.head_dim
    total = sum(counts)
    # a slice of wider rows, as a projection's output is
    queries = normal((total, heads + 3, dim + 2), seed, spread).to(kind_of(name))[:, 1:heads + 1, 2:]
    starts = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    scale = dim ** -0.5 if scale is None else scale
    with TokenContext() as context:
        call = lambda: context.attend(queries, seqs.cache, seqs.table, seqs.lengths_on_device,  # noqa: E731
                                      max_length=max(seqs.lengths), query_offsets=starts if offsets else None,
                                      max_queries=max(counts + [1]), scale=scale, **more)
        out = call()
        again = call()
        torch.cuda.synchronize()
    assert torch.equal(out, again)  # the same bits every time
    seqs.check(queries, counts, out, scale, name)
    seqs.cache.check()
    return out


SHORT = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 200, 255, 257]


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128)])
def test_attend_every_form(cuda, dim, group, name):
    """One token a sequence, lengths around every boundary, each head layout's width of a few heads."""
    attend(Sequences(SHORT, dim, group, 2, 16), [1] * len(SHORT), 8, name, offsets=False)
    attend(Sequences([777, 513, 64], dim, group, 1, 48), [1, 1, 1], 5, name)


@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (3, 3), (2, 4), (1, 6), (2, 16), (1, 9), (1, 16), (1, 17), (2, 64)])
def test_attend_head_layouts(cuda, kv_heads, heads):
    attend(Sequences([300, 41], 128, 64, kv_heads, 32), [1, 1], heads, "float16")
    attend(Sequences([300, 41], 64, 64, kv_heads, 32), [3, 2], heads, "bfloat16")


def test_attend_several_new_tokens(cuda):
    """Causal among the new tokens; sequences without any; rows that see nothing give zeros."""
    import torch

    seqs = Sequences([50, 0, 5, 130, 64, 1], 128, 64, 2, 16)
    attend(seqs, [4, 0, 5, 1, 17, 1], 8, "float16")
    seqs = Sequences([3, 0, 70], 64, 32, 1, 16)
    out = attend(seqs, [5, 2, 33], 3, "bfloat16")
    assert torch.count_nonzero(out[:2]) == 0 and torch.count_nonzero(out[5:7]) == 0


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 128)])
def test_attend_many_rows_of_many_sequences(cuda, dim, group, name):
    """More segments of 8 rows than SMs, with rows that do not fill 16, whole and cut among blocks."""
    counts = [5, 1, 4, 5, 0, 3, 2, 5, 1, 5] * 3
    lengths = [5, 1, 70, 129, 0, 257, 31, 200, 16, 64] * 3
    attend(Sequences(lengths, dim, group, 2, 16), counts, 12, name)
    lengths[3], lengths[17] = 3001, 1500
    attend(Sequences(lengths, dim, group, 2, 48), counts, 10, name)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,group,kv_heads,heads", [(64, 32, 2, 8), (128, 64, 1, 5), (128, 128, 2, 4), (256, 64, 1, 4)])
def test_attend_prompts(cuda, dim, group, kv_heads, heads, name):
    """Prompts of hundreds of tokens, alone and packed, some behind tokens that are cached already."""
    attend(Sequences([611], dim, group, kv_heads, 16), [611], heads, name)
    attend(Sequences([400, 1, 333, 900], dim, group, kv_heads, 48), [400, 1, 130, 257], heads, name)


@pytest.mark.parametrize("length", [1000, 4095, 20000])
def test_attend_long(cuda, length):
    """Work that is split over the length and joined."""
    attend(Sequences([length], 128, 64, 2, 64), [1], 8, "float16")
    attend(Sequences([length, 3, length // 2 + 1], 128, 128, 1, 16), [1, 1, 1], 4, "bfloat16")
    attend(Sequences([length // 2], 256, 128, 1, 32), [3], 4, "float16")


def test_attend_scores_of_every_size(cuda):
    """Peaked weights, scores in the thousands, no scale at all, values of very different scales."""
    attend(Sequences([500, 90], 128, 64, 2, 16, spread=4.0), [1, 2], 8, "float16", spread=8.0)
    attend(Sequences([500, 90], 128, 64, 2, 16), [1, 2], 8, "float16", scale=0.0)
    attend(Sequences([500, 90], 128, 64, 2, 16), [1, 2], 8, "bfloat16", scale=-0.05)
    seqs = Sequences([700], 128, 32, 1, 16)
    tiny = seqs.cache.tensors[3]
    tiny[::2] *= 2.0 ** -8
    tiny[:, :, :, 1, 0] *= 0.0  # a group of values that are their minimums alone
    attend(seqs, [2], 4, "float16")


@pytest.mark.parametrize("factor,lengths,spread", [(2.0 ** -17, [40, 23], 1.0), (1.0, [700, 90], 1.0),
                                                   (2.0 ** 14, [3000, 500], 6.0)])
@pytest.mark.parametrize("share", [0.5, 1.0])
def test_attend_negative_scales(cuda, factor, lengths, spread, share):
    """Groups of keys and values whose scale is negative, some or all of them: values whose weights are float16's smallest
    numbers unless they are scaled, ordinary ones, and ones whose weights pass float16 with a rising maximum."""
    import torch

    seqs = Sequences(lengths, 128, 32, 1, 16)
    make = torch.Generator(device="cuda").manual_seed(9)
    for which, by in ((1, 1.0), (3, factor)):
        pairs = seqs.cache.tensors[which]
        turned = torch.rand(pairs.shape[:-1], generator=make, device="cuda") < share
        scales, minimums = pairs[..., 0].float() * by, pairs[..., 1].float() * by
        pairs[..., 0] = torch.where(turned, -scales, scales).half()
        pairs[..., 1] = torch.where(turned, minimums + 15.0 * scales, minimums).half()  # nearly the same values' range
    attend(seqs, [2, 1], 4, "bfloat16", spread=spread)


def test_attend_large_queries(cuda):
    """bfloat16 queries past FP16's range, and float16 ones at its ends."""
    attend(Sequences([90, 40], 128, 64, 1, 16), [1, 1], 8, "bfloat16", spread=1e6, scale=1e-7)
    attend(Sequences([90, 40], 128, 64, 1, 16), [1, 1], 8, "bfloat16", spread=1e-20, scale=1.0)
    attend(Sequences([90, 40], 128, 64, 1, 16), [1, 1], 8, "float16", spread=15000.0, scale=1e-5)
    attend(Sequences([90, 40], 128, 64, 1, 16), [1, 1], 8, "float16", spread=1e-6, scale=1e5)


def test_attend_not_a_number(cuda):
    """A NaN key spoils the rows that see it; a NaN query its own row; nothing else."""
    import torch

    from nvcr_b200.tokens import TokenContext

    seqs = Sequences([100, 100], 128, 64, 2, 16)
    page, within = int(seqs.slots[0][99]) // 16, int(seqs.slots[0][99]) % 16
    seqs.cache.tensors[1][page, 1, within, 0, 0] = float("nan")
    queries = normal((4, 4, 128), 3).half()
    queries[3, 2, 5] = float("nan")
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    with TokenContext() as context:
        out = context.attend(queries, seqs.cache, seqs.table, seqs.lengths_on_device, max_length=100,
                             query_offsets=starts, max_queries=2)
        torch.cuda.synchronize()
    spoiled = out.isnan().any(-1)
    want = torch.zeros((4, 4), dtype=torch.bool, device="cuda")
    want[1, 2:] = True
    want[3, 2] = True
    assert torch.equal(spoiled, want)


def test_attend_past_32_bits(cuda):
    """Pages whose codes lie more than 2^32 bytes into the cache."""
    page_bytes = 8 * 128 * 128
    seqs = Sequences([300, 129], 256, 128, 8, 128, pages=(1 << 32) // page_bytes + 700)
    assert int(seqs.table[0, 0]) * page_bytes > 1 << 32
    attend(seqs, [1, 2], 16, "float16")
    del seqs


def test_attend_device_data_out_of_range(cuda):
    import torch

    from nvcr_b200.executor import ErrorCode, ExecutorError
    from nvcr_b200.tokens import TokenContext

    def told(seqs, what):
        with pytest.raises(ExecutorError) as error:
            seqs.cache.check()
        assert error.value.code == ErrorCode.invalid_argument and what in error.value.message
        seqs.cache.check()

    with TokenContext() as context:
        queries = normal((2, 4, 64), 3).half()
        seqs = Sequences([40, 40], 64, 64, 2, 16)
        good = context.attend(queries, seqs.cache, seqs.table, seqs.lengths_on_device, max_length=40)
        seqs.table[0, 1] = 1 << 30
        out = context.attend(queries, seqs.cache, seqs.table, seqs.lengths_on_device, max_length=40)
        told(seqs, "page number")
        assert torch.equal(out[1], good[1]) and torch.isfinite(out).all()
        seqs = Sequences([40, 40], 64, 64, 2, 16)
        out = context.attend(queries, seqs.cache, seqs.table, torch.tensor([50, 40], dtype=torch.int32, device="cuda"),
                             max_length=40)
        told(seqs, "length")
        assert torch.equal(out[1], good[1])
        out = context.attend(queries, seqs.cache, seqs.table, seqs.lengths_on_device, max_length=40, max_queries=1,
                             query_offsets=torch.tensor([0, 9, 2], dtype=torch.int32, device="cuda"))
        told(seqs, "length")
        empty = context.attend(queries[:0], seqs.cache, seqs.table[:0], seqs.lengths_on_device[:0], max_length=0)
        assert empty.shape == (0, 4, 64)


def attend_into(out, context, seqs, queries, lengths, offsets, max_queries, max_length):
    """Attention through the C ABI into a buffer of the caller's (FP16)."""
    import ctypes

    from nvcr_b200.executor import _check, library

    table = seqs.table
    _check(library().nvcr_sm100_token_attend(
        context._handle, ctypes.addressof(seqs.cache._struct), 0, queries.data_ptr(), queries.stride(0),
        queries.stride(1), queries.shape[0], queries.shape[1], table.data_ptr(), table.stride(0), table.shape[1],
        lengths.data_ptr(), lengths.shape[0], None if offsets is None else offsets.data_ptr(), max_queries, max_length,
        queries.shape[2] ** -0.5, out.data_ptr(), None))


@pytest.mark.parametrize("repeat", [1, 40])
def test_attend_tokens_of_no_sequence_are_zeros(cuda, repeat):
    """Every row is written: tokens before the first sequence, after the last, and of sequences that are left out.
    40 repeats of the sequences are more than one to a lane."""
    import torch

    from nvcr_b200.executor import ExecutorError
    from nvcr_b200.tokens import TokenContext

    lengths, counts = [60, 33, 5] * repeat, [3, 1, 2] * repeat
    seqs, tokens = Sequences(lengths, 64, 32, 2, 16), sum(counts) + 6
    queries = normal((tokens, 4, 64), 5).half()
    starts = [2 + sum(counts[:i]) for i in range(len(counts) + 1)]
    on_device = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    with TokenContext() as context:
        def call(lengths, offsets, max_queries=3, queries=queries):
            out = torch.full((queries.shape[0], 4, 64), float("nan"), dtype=torch.float16, device="cuda")
            attend_into(out, context, seqs, queries, lengths, offsets, max_queries, 60)
            torch.cuda.synchronize()
            return out

        def told():
            with pytest.raises(ExecutorError, match="length or offset"):
                seqs.cache.check()

        whole = call(seqs.lengths_on_device, on_device(starts))
        seqs.cache.check()  # tokens around the sequences' are padding, and no fault
        assert torch.count_nonzero(whole[:2]) == 0 and torch.count_nonzero(whole[-4:]) == 0
        seqs.check(queries[2:-4], counts, whole[2:-4], 64 ** -0.5, "float16")

        def left_out(lengths, offsets, gone, max_queries=3):
            out = call(lengths, offsets, max_queries)
            told()
            kept = torch.ones(tokens, dtype=torch.bool, device="cuda")
            kept[gone] = False
            assert torch.count_nonzero(out[~kept]) == 0 and torch.equal(out[kept], whole[kept])

        first = slice(starts[0], starts[1])
        for bad in (61, -1):
            left_out(on_device([bad] + lengths[1:]), on_device(starts), first)
        # a sequence of more tokens than the call said; one past the tokens' end; ends before starts, and so overlaps
        left_out(seqs.lengths_on_device, on_device([0] + starts[1:]), first, 4)
        last = slice(starts[-2], starts[-1])
        left_out(seqs.lengths_on_device, on_device(starts[:-1] + [tokens + 1]), last)
        left_out(seqs.lengths_on_device, on_device([-3] + starts[1:]), first)
        left_out(seqs.lengths_on_device, on_device(starts[:-1] + [starts[-2] - 1]), last)

        one = normal((len(lengths), 4, 64), 6).half()
        good = call(seqs.lengths_on_device, None, 1, one)
        out = call(on_device(lengths[:-1] + [1000]), None, 1, one)
        told()
        assert torch.count_nonzero(out[-1]) == 0 and torch.equal(out[:-1], good[:-1])
        none = call(seqs.lengths_on_device[:0], on_device([0]))
        assert torch.count_nonzero(none) == 0


def test_attend_refuses_more_work_than_it_can_count(cuda):
    """Upper bounds of the schedule past 32 bits, and past 64."""
    import torch

    from nvcr_b200.executor import ErrorCode, ExecutorError
    from nvcr_b200.tokens import PagedCache, TokenContext

    cache, queries = PagedCache.empty(1, 1, 16, 64, 32), torch.zeros((1, 64, 64), dtype=torch.float16, device="cuda")
    lengths = torch.zeros((65535,), dtype=torch.int32, device="cuda")
    offsets = torch.zeros((65536,), dtype=torch.int32, device="cuda")
    with TokenContext() as context:
        for columns, length, most in ((1, 16, 65535), (1 << 23, 1 << 27, 65535), (1 << 23, 1 << 27, 1)):
            table = torch.zeros((1, columns), dtype=torch.int32, device="cuda").expand(65535, columns)
            with pytest.raises(ExecutorError) as error:
                context.attend(queries, cache, table, lengths, query_offsets=offsets, max_queries=most, max_length=length)
            assert error.value.code == ErrorCode.invalid_argument


# ---- products ----

def check_multiply(rows, inputs, outputs, group, name, bias=False, spread=1.0, x=None):
    import torch

    from nvcr_b200.tokens import PackedMatrix

    kind = kind_of(name)
    make = torch.Generator(device="cuda").manual_seed(rows * 7 + inputs)
    codes = torch.randint(0, 256, (outputs, inputs // 2), generator=make, device="cuda").to(torch.uint8)
    scales = ((torch.rand((outputs, inputs // group), generator=make, device="cuda") + 0.1) * inputs ** -0.5).half()
    minimums = (-scales.float() * (7.5 + torch.randn(scales.shape, generator=make, device="cuda"))).half()
    if x is None:
        x = normal((rows, inputs + 24), 5, spread)[:, 8:inputs + 8].to(kind)
    b = normal((outputs,), 6).to(kind) if bias else None
    matrix = PackedMatrix(codes, scales, minimums)
    y = matrix.multiply(x, bias=b)
    assert torch.equal(matrix.multiply(x, bias=b), y) or y.isnan().any()
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).double()
    s, m = (t.double().repeat_interleave(group, 1) for t in (scales, minimums))
    want = x.double() @ (c * s + m).t()
    size = x.double().abs() @ (15 * s + m.abs()).t()  # of the groups' sums
    inner = x.double().abs() @ ((143 if name == "bfloat16" else 15) * s + m.abs()).t()  # of what a group adds up
    if b is not None:
        want, size = want + b.double(), size + b.double().abs()
    tolerance = (group / 16 + 2) * 2.0 ** -23 * inner + (inputs / group / 4 + 24) * 2.0 ** -24 * size
    return y, want, tolerance


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 33, 70])
def test_multiply_rows(cuda, name, rows):
    y, want, tolerance = check_multiply(rows, 512, 100, 64, name)
    near(y, want, tolerance, name)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("inputs,outputs", [(128, 1), (128, 15), (256, 16), (384, 17), (1152, 1001), (4096, 333),
                                            (16384, 70), (640, 5000)])
def test_multiply_shapes(cuda, group, inputs, outputs):
    for name, rows in (("float16", 1), ("bfloat16", 3), ("float16", 12), ("bfloat16", 16)):
        y, want, tolerance = check_multiply(rows, inputs, outputs, group, name, bias=rows == 3)
        near(y, want, tolerance, name)


@pytest.mark.parametrize("inputs,outputs,rows,group", [
    (2048, 16, 1, 128), (4096, 16, 16, 64), (8192, 40, 3, 32), (8192, 1500, 16, 128), (6016, 300, 12, 32),
    (32768, 33, 16, 64), (98304, 20, 9, 128), (98304, 20, 1, 32), (128, 40000, 2, 128), (256, 20000, 16, 32),
])
def test_multiply_divisions(cuda, inputs, outputs, rows, group):
    """Inputs divided among the blocks of a cluster, rows too long for 16 at a time, many outputs a block."""
    for name in ("float16", "bfloat16"):
        y, want, tolerance = check_multiply(rows, inputs, outputs, group, name, bias=True)
        near(y, want, tolerance, name)


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("inputs,outputs,rows", [(4224, 1001, 9), (1152, 4000, 16), (16384, 300, 12), (98304, 50, 16),
                                                 (512, 100, 40), (2048, 2048, 32), (2048, 2049, 31)])
def test_multiply_sixteen_rows(cuda, inputs, outputs, rows, group, name):
    """16 rows at a time on both sides of where they begin, with clusters, and too long for that."""
    y, want, tolerance = check_multiply(rows, inputs, outputs, group, name, bias=True)
    near(y, want, tolerance, name)


def test_multiply_odd_inputs(cuda):
    for inputs in (32, 96, 160, 1056):
        for name, rows in (("float16", 1), ("bfloat16", 9)):
            y, want, tolerance = check_multiply(rows, inputs, 50, 32, name)
            near(y, want, tolerance, name)
    y, want, tolerance = check_multiply(4, 192, 50, 64, "float16")
    near(y, want, tolerance, "float16")


def test_multiply_values_of_every_size(cuda):
    import torch

    for name, spread in (("bfloat16", 1e25), ("bfloat16", 1e-25), ("float16", 1e4), ("float16", 2e-6)):
        y, want, tolerance = check_multiply(3, 1024, 200, 128, name, spread=spread)
        over = want.abs() > 65504 * (1 - 2.0 ** -12) if name == "float16" else want.abs() > 3e38
        near(torch.where(over, 0.0, y.double()), torch.where(over, 0.0, want), tolerance, name)
    x = normal((5, 1024), 1).half()
    x[1, 17] = float("nan")
    x[3, 1000] = float("inf")
    y, want, tolerance = check_multiply(5, 1024, 200, 64, "float16", x=x)
    assert y[1].isnan().all() and not torch.isfinite(y[3]).any()
    near(y[[0, 2, 4]], want[[0, 2, 4]], tolerance[[0, 2, 4]], "float16")


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("inputs,outputs,rows", [(512, 100, 7), (4096, 16, 16), (8192, 1500, 9), (384, 2500, 3)])
def test_multiply_infinities(cuda, inputs, outputs, rows, group, name):
    """An infinity times a weight has the weight's sign, opposite ones and zero weights give NaN; other rows are as ever."""
    import torch

    make = torch.Generator(device="cuda").manual_seed(inputs + rows)
    x = normal((rows, inputs), 5).to(kind_of(name))
    at = torch.randint(0, inputs, (rows,), generator=make, device="cuda")
    for row in range(0, rows, 2):
        x[row, at[row]] = math.inf if row % 4 == 0 else -math.inf
    x[rows - 1, at[0]], x[rows - 1, at[rows - 1]] = math.inf, -math.inf
    y, want, tolerance = check_multiply(rows, inputs, outputs, group, name, x=x)
    near(y, want, tolerance, name)
    infinite = want.isinf()
    assert infinite.any() and torch.equal(y.double()[infinite], want[infinite])
    assert want[rows - 1].isnan().any() or at[0] == at[rows - 1]  # the row with both


def test_multiply_sums_past_a_row_of_codes(cuda):
    """bfloat16 rows whose products are finite while 128 times a group's sum is not."""
    import torch

    x = torch.full((2, 256), 2.0 ** 120, dtype=torch.bfloat16, device="cuda")
    x[1, ::2] = -(2.0 ** 120)
    y, want, tolerance = check_multiply(2, 256, 40, 128, "bfloat16", x=x)
    assert torch.isfinite(want).all() and float(want.abs().max()) < 3e38
    near(y, want, tolerance, "bfloat16")


def test_multiply_unaligned_rows(cuda):
    import torch

    x = normal((6, 1025 + 512), 1).half()
    for first in (0, 1):
        y, want, tolerance = check_multiply(6, 1024, 77, 64, "float16", x=x[:, first:first + 1024])
        near(y, want, tolerance, "float16")
    y, _, _ = check_multiply(0, 1024, 77, 64, "float16", x=x[:0, :1024])
    assert y.shape == (0, 77)


def test_quantised_matrix(cuda):
    import torch

    from nvcr_b200.tokens import PackedMatrix

    weights = normal((200, 512), 3, 0.05)
    matrix = PackedMatrix.quantise(weights, 32)
    eye = torch.eye(512, device="cuda").half()
    back = matrix.multiply(eye).double().t()
    parts = weights.unflatten(1, (-1, 32)).double()
    step = (parts.amax(-1) - parts.amin(-1)) / 15
    limit = (step * 0.51 + 2.0 ** -11 * parts.abs().amax(-1) * 2 + 2.0 ** -23)[..., None]
    assert ((back.unflatten(1, (-1, 32)) - parts).abs() <= limit).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_matrix_is_the_header_s_form(cuda, group):
    """The same codes, scales and minimums as the formula in FP32 on the host, ranges too small for a float16 step too."""
    import torch

    from nvcr_b200.tokens import PackedMatrix

    weights = normal((48, 512), 4, 0.05, 0.01)
    weights[::3] *= 1e-6  # steps among float16's smallest numbers, and below them
    weights[1::3] = weights[1::3] * 1e-8 + 2.0 ** -20
    weights[5] = 0.25
    weights[6] = 0.0
    codes, scales, minimums = quantised_fp32(weights.cpu().numpy(), group)
    assert (scales == 2.0 ** -24).any() and (scales == 0).any()
    on_device = [torch.from_numpy(a).cuda() for a in (codes[:, 0::2] | codes[:, 1::2] << 4, scales, minimums)]
    want, got = PackedMatrix(*on_device), PackedMatrix.quantise(weights, group)
    assert torch.equal(got.scales, want.scales) and torch.equal(got.codes, want.codes)


# ---- streams and graphs ----

def test_check_waits_for_other_streams(cuda):
    """What a kernel still to run on another stream finds is told by this check, and once."""
    import torch

    from nvcr_b200.executor import ExecutorError
    from nvcr_b200.tokens import PagedCache

    cache, side = PagedCache.empty(2, 2, 16, 64, 32), torch.cuda.Stream()
    x, slots = normal((3, 2, 64), 1).half(), torch.tensor([32, 33, 1], device="cuda")
    product, others = torch.zeros((4096, 4096), device="cuda"), slots - 30
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        product @ product
    cache.append(x, x, others, stream=side)  # loading a kernel would wait for the device
    cache.check()
    with torch.cuda.stream(side):
        for _ in range(20):
            product = product @ product
    cache.append(x, x, slots, stream=side)
    with pytest.raises(ExecutorError, match="slot"):
        cache.check()
    cache.check()


@pytest.mark.parametrize("as_handle", [False, True])
def test_quantised_on_another_stream(cuda, as_handle):
    """Weights that a busy stream is still writing, quantised on it: nothing of the call runs ahead of that, and what it
    releases is not reused before that stream has read it."""
    import torch

    from nvcr_b200.tokens import PackedMatrix

    weights, side = normal((512, 2048), 3, 0.05), torch.cuda.Stream()
    want = PackedMatrix.quantise(weights, 64)
    late, product = torch.zeros_like(weights), torch.zeros((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):  # milliseconds of work
            product = product @ product
        late.copy_(weights)
    matrix = PackedMatrix.quantise(late, 64, stream=side.cuda_stream if as_handle else side)
    for _ in range(8):  # takes what this stream's allocator has of the temporaries' sizes, and writes it
        [torch.full(shape, 255, dtype=torch.uint8, device="cuda") for shape in ((512, 1024), (512, 32, 2), (512, 2048, 4))]
    torch.cuda.synchronize()
    assert torch.equal(matrix.codes, want.codes) and torch.equal(matrix.scales, want.scales)


def test_another_stream_and_a_graph(cuda):
    """The operators run on torch's current stream, on a named one, and inside a captured graph with new inputs."""
    import torch

    from nvcr_b200 import tokens

    cache = tokens.PagedCache.empty(8, 2, 16, 64, 32)
    matrix = tokens.PackedMatrix.quantise(normal((256, 256), 1, 0.06), 64)
    cosines, sines = make_tables(200, 64)
    state = {"x": normal((2, 256), 2).half(), "slots": torch.tensor([3, 70], device="cuda"),
             "positions": torch.tensor([3, 6], dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor([4, 7], dtype=torch.int32, device="cuda"),
             "table": torch.tensor([[0, 1], [4, 5]], dtype=torch.int32, device="cuda")}
    context = tokens.TokenContext()

    def step(stream=None):
        _, normed = tokens.block_norm(state["x"], stream=stream)
        q = matrix.multiply(normed, stream=stream).view(2, 4, 64)
        turned = cache.append(q[:, :2], q[:, 2:], state["slots"], queries=q, positions=state["positions"],
                              cosines=cosines, sines=sines, stream=stream)
        return context.attend(turned, cache, state["table"], state["lengths"], max_length=32, stream=stream)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        here = step()
    there = step(stream=side)
    side.synchronize()
    assert torch.equal(here, want) and torch.equal(there, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (5, 6):
        state["x"].copy_(normal((2, 256), seed).half())
        graph.replay()
        torch.cuda.synchronize()
        replayed = captured.clone()
        assert torch.equal(step(), replayed)
    context.close()


def test_contexts_closed_around_captures(cuda):
    """Closing a context does not disturb a capture; one that a graph holds is not handed out again, others are."""
    import torch

    from nvcr_b200.tokens import TokenContext

    seqs = Sequences([20000], 128, 64, 2, 64)  # cut among blocks, which join in the context's memory
    queries = [normal((1, 8, 128), seed).half() for seed in (1, 2)]
    call = lambda context, q: context.attend(q, seqs.cache, seqs.table, seqs.lengths_on_device,  # noqa: E731
                                             max_length=20000)
    held, other = TokenContext(), TokenContext()
    want = [call(held, q) for q in queries]
    graph, holder = torch.cuda.CUDAGraph(), held._handle.value
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = call(held, queries[0])
        other.close()
        held.close()
    with TokenContext() as context:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(20):  # the graph and another context at once
            graph.replay()
            with torch.cuda.stream(side):
                out = call(context, queries[1])
        torch.cuda.synchronize()
        assert torch.equal(captured, want[0]) and torch.equal(out, want[1])
        ordinary = context._handle.value
    several = [TokenContext() for _ in range(24)]
    handles = {context._handle.value for context in several}
    assert ordinary in handles and holder not in handles
    for context in several:
        assert torch.equal(call(context, queries[0]), want[0])
        context.close()


def test_output_that_does_not_fit_raises_torch_s_error(cuda):
    """The allocator's refusal arrives as what a program around torch catches, and the next call runs."""
    import torch

    from nvcr_b200 import tokens

    block = torch.zeros((1, 1 << 20), dtype=torch.float16, device="cuda")
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.01)  # torch's own bound: no memory is taken
    try:
        with pytest.raises(torch.OutOfMemoryError):
            tokens.block_norm(block.expand(2000, 1 << 20))
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    hidden, _ = tokens.block_norm(block)
    assert torch.equal(hidden, block)
