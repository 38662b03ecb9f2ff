"""Products in 8 bits, products by experts, routing and sampling on the GPU against plain implementations in 64 bits.

Tolerances are error bounds of the operators' arithmetic, derived here:
* a product's sum of codes is exact; it becomes FP32 and is multiplied twice, three roundings of 2^-24 each of the
  product; adding a bias rounds the sum once more;
* a weighted sum over `chosen` products adds a rounding of each product's share and of each addition: (3 + 2 chosen)
  2^-24 of the sum of their magnitudes;
* an output of a type with unit roundoff u (2^-11, 2^-8, 2^-24) is rounded once: u |y|, and 2^-25 absolute for a
  float16 below its normal range, 2^-150 for the others;
* choices and symbols are equal: both sides decide in 64 bits; weights and probabilities are rounded to FP32 once,
  after FP64 arithmetic whose error (some 2^-50, and for a probability the 2^-43 of the weights' unit, of which a row
  has at most 2^18: 2^-25) is small beside it.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
LEAST = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150}
E = 2.0 ** -24
TYPES = ["float16", "bfloat16", "float32"]


def kind_of(name):
    import torch

    return getattr(torch, name)


def normal(shape, seed, spread=1.0):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=make, device="cuda", dtype=torch.float32) * spread


def some_codes(shape, seed):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=make, device="cuda", dtype=torch.int8)


def near(got, want, tolerance, name):
    """Every element of `got` within `tolerance` (elementwise) and a rounding of `want`, NaNs alike."""
    import torch

    got = got.double()
    limit = tolerance + UNIT[name] * want.abs() * 1.001 + LEAST[name]
    nan = torch.isnan(want)
    assert got.shape == want.shape and torch.equal(torch.isnan(got), nan)
    off = torch.where(nan, torch.zeros_like(want), (got - want).abs() - limit)
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0.0, (
        f"element {worst} of {off.numel()}: {got.flatten()[worst]} for {want.flatten()[worst]}, "
        f"{int((off > 0).sum())} outside")


def as_codes(x):
    """The header's codes and scales of rows, each step rounded to FP32 by numpy on the CPU."""
    import torch

    with np.errstate(all="ignore"):
        v = x.float().cpu().numpy()
        largest = np.abs(v).max(-1, keepdims=True)
        scale = np.maximum(largest * np.float32(1.0 / 127.0), np.float32(2.0 ** -126)).astype(np.float32)
        codes = np.rint(v * (np.float32(1.0) / scale))
        bad = ~np.isfinite(largest)
        codes = np.where(bad, 0.0, codes)
        scale = np.where(bad, np.nan, scale)
    assert codes.dtype == np.float32 and np.abs(codes).max(initial=0.0) <= 127
    return torch.from_numpy(codes).double().cuda(), torch.from_numpy(scale.astype(np.float64)).cuda()


def plain(x, codes, scales, bias=None):
    """Products in 64 bits and the tolerance of everything but the output's rounding. Codes' sums are exact."""
    q, s = as_codes(x)
    y = (q @ codes.double().transpose(-1, -2)) * scales.double() * s
    tolerance = 3.1 * E * y.abs() + 2.0 ** -148  # a factor may fall below FP32's normal range
    if bias is not None:
        y = y + bias.double()
        tolerance = tolerance + E * 1.1 * y.abs()
    return y, tolerance


# ---- one matrix ----

def check_matrix(rows, inputs, outputs, name, bias=False, seed=1, x=None, spread=1.0):
    from nvcr_b200.tokens import ByteMatrix

    codes, scales = some_codes((outputs, inputs), seed), normal((outputs,), seed + 1, 0.01).abs() + 1e-4
    x = (normal((rows, inputs), seed + 2, spread) if x is None else x).to(kind_of(name))
    b = normal((outputs,), seed + 3).to(kind_of(name)) if bias else None
    matrix = ByteMatrix(codes, scales)
    got = matrix.multiply(x, bias=b)
    want, tolerance = plain(x, codes, scales, b)
    assert got.dtype == x.dtype
    near(got, want, tolerance, name)
    matrix.check()
    return matrix, x, got


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 77, 128, 129, 255, 257, 300, 1000])
def test_matrix_rows(cuda, rows, name):
    check_matrix(rows, 300, 200, name, bias=rows % 2 == 1)


@pytest.mark.parametrize("inputs", [1, 15, 16, 17, 127, 128, 129, 1000, 1025, 2049, 4096, 9001])
@pytest.mark.parametrize("outputs", [1, 31, 128, 129, 500])
def test_matrix_shapes(cuda, inputs, outputs):
    check_matrix(5, inputs, outputs, TYPES[(inputs + outputs) % 3], bias=True)


@pytest.mark.parametrize("name", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,inputs,outputs", [(2000, 1024, 4096), (2049, 900, 5000), (1111, 128, 16400), (4096, 4096, 2048),
                                                 (5000, 2000, 1130)])
def test_matrix_of_many_rows(cuda, rows, inputs, outputs, name):
    """Sizes at which two blocks share a tile, with odd numbers of tiles and last tiles of a few rows."""
    check_matrix(rows, inputs, outputs, name, bias=rows % 2 == 1)


@pytest.mark.parametrize("rows,inputs,outputs", [
    (1, 4096, 4096), (16, 4096, 16384), (40, 16384, 1024), (64, 8192, 700), (512, 1024, 4096), (700, 512, 3000),
    (2048, 2048, 2048), (4099, 640, 1111), (3, 131072, 260)])
def test_matrix_divisions(cuda, rows, inputs, outputs):
    """Sizes at which a tile has one or several blocks, and blocks one or several tiles."""
    check_matrix(rows, inputs, outputs, "bfloat16" if rows % 2 else "float16")


def test_matrix_without_rows(cuda):
    import torch

    from nvcr_b200.tokens import ByteMatrix

    matrix = ByteMatrix(some_codes((5, 7), 1), torch.ones(5, device="cuda"))
    assert matrix.multiply(torch.empty((0, 7), device="cuda")).shape == (0, 5)


@pytest.mark.parametrize("name", TYPES)
def test_matrix_strides(cuda, name):
    """Rows apart by any stride, the same row again and again, and rows that begin anywhere."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    codes, scales = some_codes((70, 256), 1), torch.full((70,), 0.01, device="cuda")
    matrix = ByteMatrix(codes, scales)
    wide = normal((9, 801), 2).to(kind_of(name))
    for x in (wide[:, 3:259], wide[:, 16:272], wide[::2, 1:257], wide[:1, 5:261].expand(6, 256), wide[:, :512:2][:, :256].contiguous(),
              wide.flatten()[1:257].view(1, 256)):
        want, tolerance = plain(x, codes, scales)
        near(matrix.multiply(x), want, tolerance, name)


@pytest.mark.parametrize("name", TYPES)
def test_matrix_values_of_every_size(cuda, name):
    """Rows of zeros, the smallest and the largest values, one value alone, and rows that hold NaNs or infinities."""
    import torch

    kind = kind_of(name)
    least, most = {"float16": (2.0 ** -24, 60000.0), "bfloat16": (2.0 ** -133, 3e38), "float32": (2.0 ** -149, 3e38)}[name]
    x = normal((12, 200), 5)
    x[0] = 0.0
    x[1] = least
    x[2] = least * torch.arange(200, device="cuda") % 7
    x[3] = torch.sign(x[3]) * most
    x[4, 1:] = 0.0
    x[5] *= 1e-6
    x[6, 3] = math.nan
    x[7, 199] = math.inf
    x[8, 0] = -math.inf
    x[9] = math.nan
    x[10] = most / 100.0
    x = x.to(kind)
    from nvcr_b200.tokens import ByteMatrix

    codes, scales = some_codes((130, 200), 6), torch.full((130,), 2.0 ** -14, device="cuda")
    got = ByteMatrix(codes, scales).multiply(x)
    want, tolerance = plain(x, codes, scales)
    limit = torch.finfo(kind).max
    assert torch.isnan(got[6:10]).all()
    fits = want.abs() < limit  # beyond: an infinity
    near(torch.where(fits | torch.isnan(want), got, 0), torch.where(fits | torch.isnan(want), want, 0.0), tolerance, name)
    assert torch.equal(torch.isposinf(got), want >= limit * (1 + UNIT[name]))


def test_matrix_largest_sums(cuda):
    """131072 products of -128 and 127: the sum's largest magnitude, just inside 32 bits."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    codes = torch.full((3, 131072), -128, dtype=torch.int8, device="cuda")
    codes[1] = 127
    scales = torch.tensor([1.0, 1.0, 0.5], device="cuda")
    x = torch.ones((2, 131072), device="cuda")
    x[1] = -1.0
    want, tolerance = plain(x, codes, scales)
    near(ByteMatrix(codes, scales).multiply(x), want, tolerance, "float32")


def test_matrix_quantised(cuda):
    """`quantise` takes a weight row as `multiply` takes a row of x."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    weights = normal((150, 333), 4)
    weights[0] = 0.0
    weights[1] = 2.0 ** -140
    q, s = as_codes(weights)
    want = ByteMatrix(q.to(torch.int8), s.squeeze(1).float())
    for made in (ByteMatrix.quantise(weights), ByteMatrix.quantise(weights, stream=torch.cuda.Stream())):
        torch.cuda.synchronize()
        assert torch.equal(made.codes, want.codes) and torch.equal(made.scales, want.scales)
    default = torch.get_default_device()
    try:
        torch.set_default_device("cuda")
        assert torch.equal(ByteMatrix.quantise(weights).codes, want.codes)
    finally:
        torch.set_default_device(default)
    weights[2, 5] = math.nan
    y = ByteMatrix.quantise(weights).multiply(torch.ones((1, 333), device="cuda"))
    assert torch.isnan(y[0, 2]) and int(torch.isnan(y).sum()) == 1


def test_matrix_keeps_its_own_weights(cuda):
    """What is done to the codes and scales afterwards changes nothing."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    codes, scales, x = some_codes((256, 256), 1), torch.ones(256, device="cuda"), normal((4, 256), 2).half()
    matrix = ByteMatrix(codes, scales)
    want = matrix.multiply(x)
    codes.zero_(), scales.zero_()
    assert torch.equal(matrix.multiply(x), want)


# ---- experts ----

def check_experts(x, codes, scales, choices, weights, name):
    """x [tokens, inputs] or [tokens, chosen, inputs], of its type."""
    import torch

    from nvcr_b200.tokens import ByteExperts

    tokens, chosen = choices.shape
    experts, outputs = scales.shape
    matrices = ByteExperts(codes, scales)
    got = matrices.multiply(x, choices, weights)
    want = torch.zeros((tokens, chosen, outputs), dtype=torch.float64, device="cuda")
    tolerance = torch.zeros_like(want)
    for e in range(experts):
        token, nth = torch.nonzero(choices == e, as_tuple=True)
        if len(token):
            rows = x[token] if x.dim() == 2 else x[token, nth]
            want[token, nth], tolerance[token, nth] = plain(rows, codes[e], scales[e])
    if weights is not None:
        there = ((choices >= 0) & (choices < experts)).unsqueeze(-1)
        parts = torch.where(there, want * weights.double().unsqueeze(-1), 0.0)
        want = parts.sum(1)
        tolerance = (3.1 + 2 * chosen) * E * parts.abs().sum(1) + 2.0 ** -147
    assert got.dtype == x.dtype
    near(got, want, tolerance, name)
    matrices.check()


def some_choices(tokens, chosen, experts, seed, kind="spread"):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    choices = torch.randint(0, experts, (tokens, chosen), generator=make, device="cuda", dtype=torch.int32)
    if kind == "one":
        choices.fill_(experts - 1)
    if kind == "skewed":
        choices = torch.minimum(choices, torch.randint(0, experts, (tokens, chosen), generator=make, device="cuda",
                                                       dtype=torch.int32) // 4)
    if kind in ("absent", "outside"):
        drop = torch.rand((tokens, chosen), generator=make, device="cuda") < 0.3
        choices = torch.where(drop, -1 if kind == "absent" else experts + 5, choices)
        choices[tokens // 2] = -1  # a token with no expert at all
    return choices


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("rows_each", [False, True])
@pytest.mark.parametrize("kind", ["spread", "one", "skewed", "absent", "outside"])
def test_experts_forms(cuda, kind, rows_each, weighted, name):
    tokens, chosen, experts, inputs, outputs = 37, 3, 6, 300, 200
    x = normal((tokens, chosen, inputs) if rows_each else (tokens, inputs), 1).to(kind_of(name))
    weights = normal((tokens, chosen), 2) if weighted else None
    check_experts(x, some_codes((experts, outputs, inputs), 3), normal((experts, outputs), 4, 0.01).abs(),
                  some_choices(tokens, chosen, experts, 5, kind), weights, name)


@pytest.mark.parametrize("tokens,chosen,experts,inputs,outputs", [
    (1, 1, 1, 1, 1), (1, 8, 64, 2048, 1024), (1, 2, 1024, 64, 130), (7, 8, 8, 128, 128), (64, 8, 128, 256, 300),
    (1000, 2, 5, 129, 257), (2048, 4, 16, 512, 384), (5000, 1, 1000, 100, 50), (300, 6, 33, 1000, 520), (16, 1, 2, 4096, 64),
    (4000, 4, 8, 512, 1500), (6000, 2, 16, 1000, 1024), (2001, 8, 5, 256, 2100)])
def test_experts_shapes(cuda, tokens, chosen, experts, inputs, outputs):
    check_experts(normal((tokens, inputs), 1).bfloat16(), some_codes((experts, outputs, inputs), 3),
                  normal((experts, outputs), 4, 0.01).abs(), some_choices(tokens, chosen, experts, 5),
                  normal((tokens, chosen), 6) if tokens % 2 else None, "bfloat16")


def test_experts_strides(cuda):
    """Rows of a token and tokens any strides apart, beginning anywhere, or the same for all."""
    import torch

    codes, scales = some_codes((4, 90, 64), 1), torch.full((4, 90), 0.02, device="cuda")
    choices = some_choices(10, 2, 4, 2)
    wide = normal((10, 2, 200), 3).half()
    for x in (wide[:, :, 3:67], wide[:, :, 8:72], wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :64], wide[:, 0, 1:65],
              wide[:, :1, :64].expand(10, 2, 64), wide[:1, 0, :64].expand(10, 64)):
        check_experts(x, codes, scales, choices, None, "float16")


def test_experts_rows_without_numbers(cuda):
    """A row that holds a NaN spoils its own products only; the weight of no expert is not looked at."""
    import torch

    x = normal((20, 100), 1)
    x[4, 7], x[9, 0] = math.nan, math.inf
    choices = some_choices(20, 2, 3, 2)
    codes, scales = some_codes((3, 60, 100), 3), torch.full((3, 60), 0.01, device="cuda")
    check_experts(x, codes, scales, choices, None, "float32")
    choices[:, 1] = -1
    weights = torch.stack((torch.ones(20), torch.full((20,), math.nan)), 1).cuda()
    check_experts(x, codes, scales, choices, weights, "float32")


def test_experts_without_tokens(cuda):
    import torch

    from nvcr_b200.tokens import ByteExperts

    matrices = ByteExperts(some_codes((2, 5, 7), 1), torch.ones((2, 5), device="cuda"))
    choices = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    assert matrices.multiply(torch.empty((0, 7), device="cuda"), choices).shape == (0, 3, 5)


def test_experts_past_32_bits(cuda):
    """Matrices whose codes lie more than 2^32 bytes from the first, and products more than 2^31 from the first."""
    import torch

    from nvcr_b200.tokens import ByteExperts

    experts, outputs, inputs = 300, 4096, 3840
    codes = torch.empty((experts, outputs, inputs), dtype=torch.int8, device="cuda")
    codes[:-1] = 1
    codes[-1] = some_codes((outputs, inputs), 1)
    scales = torch.full((experts, outputs), 0.01, device="cuda")
    matrices = ByteExperts(codes, scales)
    x = normal((3, inputs), 2).half()
    choices = torch.tensor([[299, 0], [5, 299], [299, 298]], dtype=torch.int32, device="cuda")
    got = matrices.multiply(x, choices)
    for token, nth in ((0, 0), (1, 1), (2, 0), (0, 1), (2, 1)):
        e = int(choices[token, nth])
        want, tolerance = plain(x[token:token + 1], codes[e], scales[e])
        near(got[token:token + 1, nth], want, tolerance, "float16")
    del matrices, codes
    tokens, outputs = 140000, 16000
    codes, scales = some_codes((2, outputs, 32), 3), torch.full((2, outputs), 0.01, device="cuda")
    x = normal((tokens, 32), 4).half()
    got = ByteExperts(codes, scales).multiply(x, torch.ones((tokens, 1), dtype=torch.int32, device="cuda"))
    want, tolerance = plain(x[-3:], codes[1], scales[1])
    near(got[-3:, 0], want, tolerance, "float16")


# ---- routing ----

def plain_route(scores, count, kind, bias, groups, kept, renormalise, scale):
    """A token at a time, in numpy's 64 bits."""
    scores = scores.double().cpu().numpy()
    tokens, experts = scores.shape
    choices, weights = np.full((tokens, count), -1, np.int32), np.zeros((tokens, count))
    size = experts // groups
    for t, row in enumerate(scores):
        there = row > -np.inf
        share = np.zeros(experts)
        if kind == "sigmoid":
            with np.errstate(over="ignore"):
                share[there] = 1.0 / (1.0 + np.exp(-row[there]))
        elif there.any():
            top = row[there].max()
            with np.errstate(invalid="ignore"):
                share[there] = np.where(row[there] == top, 1.0, np.exp(row[there] - top))
            share /= share.sum()
        b = share + (0.0 if bias is None else bias.double().cpu().numpy())
        b = np.where(there & (b > -np.inf), b, -np.inf)
        if kept < groups:
            value = []
            for g in range(groups):
                two = sorted(b[g * size:(g + 1) * size], reverse=True)[:2]
                value.append(sum(v for v in two if v > -np.inf) if two[0] > -np.inf else -np.inf)
            for g in sorted(range(groups), key=lambda g: -value[g])[kept:]:
                b[g * size:(g + 1) * size] = -np.inf
        order = [e for e in np.argsort(-b, kind="stable")[:count] if b[e] > -np.inf]
        choices[t, :len(order)], weights[t, :len(order)] = order, share[order]
        total = weights[t].sum()
        if renormalise:
            weights[t] = weights[t] / total if total > 0 else 0.0
    return choices, weights * scale


def check_route(scores, count, kind="softmax", bias=None, groups=1, kept=1, renormalise=False, scale=1.0):
    from nvcr_b200 import tokens

    choices, weights = tokens.route(scores, count, kind=kind, bias=bias, groups=groups, kept_groups=kept,
                                    renormalise=renormalise, scale=scale)
    want, share = plain_route(scores, count, kind, bias, groups, kept, renormalise, np.float64(np.float32(scale)))
    assert np.array_equal(choices.cpu().numpy(), want)
    assert (np.abs(weights.cpu().double().numpy() - share) <= E * 1.001 * np.abs(share) + 2.0 ** -149).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,count,groups,kept", [
    (1, 1, 1, 1, 1), (1, 64, 8, 1, 1), (5, 33, 4, 1, 1), (100, 8, 2, 1, 1), (77, 256, 8, 8, 4), (9, 160, 6, 8, 3),
    (3, 1024, 1024, 1, 1), (4, 1000, 40, 4, 2), (6, 60, 10, 20, 5), (8, 96, 5, 96, 7), (7, 512, 33, 2, 1), (130, 128, 8, 4, 4)])
def test_route(cuda, tokens, experts, count, groups, kept, kind, name):
    scores = normal((tokens, experts), 1, 1.5).to(kind_of(name))
    bias = normal((experts,), 2, 0.05) if experts % 2 == 0 else None
    check_route(scores, count, kind, bias, groups, kept, renormalise=tokens % 2 == 1, scale=1.5)


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_route_masks_and_extremes(cuda, kind):
    """Experts that are left out, rows of nothing else, equal scores, infinities, NaNs, biases that exclude."""
    import torch

    scores = normal((14, 48), 3)
    scores[0] = -math.inf
    scores[1] = math.nan
    scores[2, 3:] = -math.inf
    scores[3] = 0.25
    scores[4, 7:20] = 9.0
    scores[5, 11] = math.inf
    scores[6, 5] = scores[6, 40] = math.inf
    scores[7, ::2] = math.nan
    scores[8] = -1000.0
    scores[9] = 1000.0
    scores[10, :24] = -math.inf
    scores[11] *= 1e-30
    scores[12, 0], scores[12, 1] = 0.0, -0.0
    scores[13, :47] = -math.inf
    bias = normal((48,), 4, 0.1)
    bias[2], bias[5] = -math.inf, math.nan
    for renormalise in (False, True):
        check_route(scores, 5, kind, None, renormalise=renormalise)
        check_route(scores, 5, kind, bias, renormalise=renormalise)
        check_route(scores, 6, kind, bias, 6, 2, renormalise, 2.5)
        check_route(scores, 48, kind, None, 48, 20, renormalise)
        check_route(scores, 5, kind, torch.zeros(48, device="cuda") - 3.0, 4, 1, renormalise, -1.0)


def test_route_strides(cuda):
    import torch

    from nvcr_b200 import tokens

    wide = normal((12, 101), 1)
    check_route(wide[::3, 5:37], 4)
    check_route(wide[:1, 1:65].expand(5, 64), 4)
    choices, weights = tokens.route(wide[:0], 3)
    assert choices.shape == (0, 3) and weights.dtype == torch.float32


def test_route_near_ties(cuda):
    """Scores whose order FP32 arithmetic would lose: sigmoids that agree to 2^-30, put in order by the bias."""
    import torch

    scores = torch.full((4, 64), 14.0, device="cuda") + torch.arange(64, device="cuda") * 2.0 ** -19
    bias = torch.zeros(64, device="cuda")
    bias[::7] = 2.0 ** -29
    check_route(scores, 12, "sigmoid", bias)
    check_route(-scores, 12, "softmax", bias, 8, 3, True)


def test_route_ties_before_a_larger_one(cuda):
    """Equal scores with the last places of the choice between them, and after them in FP32 one that is larger by a step."""
    import torch

    scores = torch.full((3, 40), -2.0, device="cuda")
    small = torch.tensor(1e-3, device="cuda")
    scores[:, 30] = 10.0
    scores[:, :2] = small
    scores[:, 2] = torch.nextafter(small, torch.tensor(1.0, device="cuda"))
    for count in (1, 2, 3, 4, 5):
        check_route(scores, count, "softmax")
        check_route(scores, count, "softmax", groups=4, kept=2)
        check_route(scores - 20.0, count, "sigmoid")


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_route_sums_that_agree(cuda, kind):
    """Biases that make up for the shares: every sum is the same but for a rounding, shares and so their errors are not."""
    import torch

    for seed, experts, count in ((1, 64, 6), (2, 256, 8), (3, 100, 31), (4, 32, 1)):
        scores = normal((200, experts), seed, 3.0)
        for row in range(0, 200, 8):
            wide = scores[row].double()
            share = torch.sigmoid(wide) if kind == "sigmoid" else torch.softmax(wide, 0)
            shift = normal((experts,), seed + 10, 4e-7).double()
            check_route(scores[row:row + 8], count, kind, (1.0 - share + shift).float())


# ---- sampling ----

def plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    logits = logits.double().cpu().numpy()
    rows = len(logits)
    each = lambda v, kind: (np.full(rows, v, kind) if not hasattr(v, "cpu") else v.cpu().numpy()).astype(kind)  # noqa: E731
    uniforms = uniforms.double().cpu().numpy()
    temperature, top_p, min_p = (each(v, np.float32).astype(np.float64) for v in (temperature, top_p, min_p))
    top_k = each(top_k, np.int64)
    symbols, probabilities = [], []
    for r, row in enumerate(logits):
        index = np.flatnonzero(row > -np.inf)
        if not len(index):
            symbols.append(-1), probabilities.append(0.0)
            continue
        index = index[np.argsort(-row[index], kind="stable")]
        if not temperature[r] > 0:
            symbols.append(index[0]), probabilities.append(1.0)
            continue
        if top_k[r] > 0:
            index = index[: top_k[r]]
        top = row[index[0]]
        with np.errstate(invalid="ignore"):
            share = np.where(row[index] == top, 1.0, np.exp((row[index] - top) / temperature[r]))
        share = np.nan_to_num(share)
        # sums are of multiples of 2^-43, as the header says: what is smaller does not tip two equal halves
        units = np.rint(share * 2.0 ** 43)
        n = len(index)
        if top_p[r] < 1.0:
            n = 1 + int(np.searchsorted(np.cumsum(units), max(top_p[r], 0.0) * units.sum()))
        if min_p[r] > 0:
            n = min(n, int((share >= min(min_p[r], 1.0)).sum()))
        n = max(1, min(n, len(index)))
        index, share, units = index[:n], share[:n], units[:n]
        order = np.argsort(index)
        sums = np.cumsum(units[order])
        u = 0.0 if not uniforms[r] > 0 else uniforms[r]
        at = int(np.searchsorted(sums, u * sums[-1], side="right")) if u < 1.0 else n
        at = order[min(at, np.flatnonzero(units[order])[-1])]
        symbols.append(index[at]), probabilities.append(share[at] * 2.0 ** 43 / sums[-1])
    return np.array(symbols), np.array(probabilities)


def check_sample(logits, uniforms=None, seed=1, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    import torch

    from nvcr_b200 import tokens

    if uniforms is None:
        uniforms = torch.rand(len(logits), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    symbols, probabilities = tokens.sample(logits, uniforms, **settings)
    want, share = plain_sample(logits, uniforms, **settings)
    assert symbols.dtype == torch.int64 and np.array_equal(symbols.cpu().numpy(), want)
    off = np.abs(probabilities.cpu().double().numpy() - share)
    assert (off <= (E + 2.0 ** -25) * 1.01 * share + 2.0 ** -149).all(), off.max()
    return symbols


SETTINGS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=3000), dict(top_p=0.9), dict(top_p=0.0), dict(min_p=0.02),
            dict(top_k=40, top_p=0.8, min_p=0.01), dict(temperature=0.0), dict(temperature=0.6, top_p=0.95),
            dict(temperature=2.0, top_p=0.99), dict(temperature=1.3, top_k=1000, top_p=0.5), dict(min_p=1.0),
            dict(temperature=0.01, top_p=0.5)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("rows,symbols", [(1, 1), (3, 7), (20, 1000), (9, 32768), (5, 50001), (2, 200003), (3, 262144), (2, 300001)])
def test_sample(cuda, rows, symbols, settings, name):
    import torch

    logits = normal((rows, symbols), rows, 2.0) + torch.relu(normal((rows, symbols), 7) - 2.5) * 6.0
    check_sample(logits.to(kind_of(name)), **settings)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sample_of_many_rows(cuda, settings, name):
    """So many rows that their parts are looked at one by one; flat and sharp ones, odd sizes, masks and extremes among
    them."""
    import torch

    rows, symbols = 301, {"float16": 33001, "bfloat16": 40000, "float32": 17000}[name]
    logits = normal((rows, symbols), 1, 2.0) + torch.relu(normal((rows, symbols), 7) - 2.5) * 6.0
    logits *= torch.rand((rows, 1), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 2.0
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 100:] = -math.inf
    logits[3, ::2] = math.nan
    logits[4] = 0.0
    logits[5] = -3.0
    logits[5, symbols - 1] = 4.0
    logits[6, 13] = math.inf
    logits[7, 13] = logits[7, symbols - 2] = math.inf
    logits[8] *= 1000.0
    logits[9, : symbols // 2] -= 200.0
    logits[10] = torch.round(logits[10])
    logits[11] = torch.where(torch.arange(symbols, device="cuda") % 3 == 0, 5.0, -5.0)
    logits[12, 20:] = -math.inf
    logits[12, :20] = torch.finfo(torch.float16).min
    check_sample(logits.to(kind_of(name)), **settings)


def test_sample_of_many_rows_settings_of_each_row(cuda):
    import torch

    rows = 400
    logits = normal((rows, 40001), 8, 3.0).half()
    pick = lambda values, kind: torch.tensor([values[i % len(values)] for i in range(rows)], dtype=kind, device="cuda")  # noqa: E731
    check_sample(logits, seed=5, temperature=pick([1.0, 0.0, 0.5, -1.0, math.nan, 1e-30, 1e30, math.inf, 0.02], torch.float32),
                 top_k=pick([0, 5, -3, 100000, 64, 700], torch.int32),
                 top_p=pick([1.0, 0.5, math.nan, -1.0, 2.0, 0.9, 1e-9], torch.float32),
                 min_p=pick([0.0, 0.1, -1.0, 5.0, math.nan, 0.01, 0.5, 0.0, 1e-30], torch.float32))


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("spread", [0.0, 0.01, 30.0, 1000.0])
def test_sample_flat_and_sharp(cuda, spread, settings):
    """All symbols alike, nearly alike, and one far above the rest."""
    check_sample(normal((30, 5000), 3, spread), **settings)
    check_sample(normal((30, 5000), 3, spread).bfloat16(), **settings)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sample_masks_and_extremes(cuda, settings):
    import torch

    logits = normal((16, 777), 5, 3.0)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, :776] = -math.inf
    logits[3, ::2] = math.nan
    logits[4, 100:] = torch.finfo(torch.float32).min
    logits[5] = torch.finfo(torch.float32).min
    logits[6, 13] = math.inf
    logits[7, 13] = logits[7, 600] = math.inf
    logits[8, ::2], logits[8, 1::2] = 0.0, -0.0
    logits[9] = torch.round(logits[9])
    logits[10] = 1e38 * torch.sign(logits[10])
    logits[11, 5:] = -math.inf
    check_sample(logits, **settings)
    check_sample(logits, uniforms=torch.zeros(16, device="cuda"), **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=5), dict(top_p=0.7)])
def test_sample_uniforms_at_the_ends(cuda, settings):
    """0, the largest below 1, and numbers that no uniform source gives."""
    import torch

    logits = normal((9, 500), 2, 1.0)
    uniforms = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -149, -0.5, 1.0, 3.0, math.nan, math.inf, 0.5], device="cuda")
    check_sample(logits, uniforms, **settings)


def test_sample_settings_of_each_row(cuda):
    """Every row its own settings, the ones that switch a filter off and those that no table gives among them."""
    import torch

    rows = 40
    logits = normal((rows, 3000), 8, 3.0)
    pick = lambda values, kind: torch.tensor([values[i % len(values)] for i in range(rows)], dtype=kind, device="cuda")  # noqa: E731
    check_sample(logits, seed=5, temperature=pick([1.0, 0.0, 0.5, -1.0, math.nan, 1e-30, 1e30], torch.float32),
                 top_k=pick([0, 5, -3, 100000, 64], torch.int32), top_p=pick([1.0, 0.5, math.nan, -1.0, 2.0, 0.9, 1e-9], torch.float32),
                 min_p=pick([0.0, 0.1, -1.0, 5.0, math.nan, 0.01, 0.5, 0.0], torch.float32))


def test_sample_strides_and_no_rows(cuda):
    import torch

    from nvcr_b200 import tokens

    wide = normal((12, 2001), 1)
    for name in TYPES:
        some = wide.to(kind_of(name))
        check_sample(some[::2, 3:1500], top_p=0.9)
        check_sample(some[:, 1:1990], top_k=7)
        check_sample(some[:1, 1:1990].expand(30, 1989))
    symbols, _ = tokens.sample(wide[:0], torch.empty(0, device="cuda"))
    assert symbols.shape == (0,)


def test_sample_follows_the_weights(cuda):
    """Uniform numbers spread evenly give every symbol its share of them."""
    import torch

    from nvcr_b200 import tokens

    logits = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5], device="cuda")
    n = 4096
    uniforms = (torch.arange(n, device="cuda") + 0.5) / n
    symbols, _ = tokens.sample(logits.expand(n, 5), uniforms)
    share = torch.softmax(logits.double(), 0)
    # an interval of length s holds s n numbers 1 / n apart, one more or less
    assert (torch.bincount(symbols, minlength=5).double() - share * n).abs().max() <= 1.0
    assert torch.equal(symbols, symbols.sort().values)


# ---- together ----

def test_streams_and_graphs(cuda):
    """A routed block and a sample on the current stream, on a named one, and inside two captured graphs at once."""
    import torch

    from nvcr_b200 import tokens

    experts = tokens.ByteExperts.quantise(normal((8, 256, 128), 1, 0.1))
    back = tokens.ByteExperts.quantise(normal((8, 128, 256), 2, 0.1))
    head = tokens.ByteMatrix.quantise(normal((1000, 128), 3, 0.1))
    scores = tokens.ByteMatrix.quantise(normal((8, 128), 4, 0.1))
    x, u = normal((6, 128), 5).half(), torch.rand(6, device="cuda")

    def step(stream=None):
        choices, weights = tokens.route(scores.multiply(x, stream=stream), 2, renormalise=True, stream=stream)
        inner = experts.multiply(x, choices, stream=stream)
        y = back.multiply(inner, choices, weights, stream=stream)
        logits = head.multiply(y, stream=stream)
        return (logits, *tokens.sample(logits, u, temperature=0.7, top_k=50, top_p=0.9, stream=stream))

    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        here = step()
    there = step(stream=side)
    side.synchronize()
    assert same(here, want) and same(there, want)
    for handle in (side.cuda_stream, 0):
        there = step(stream=handle)
        torch.cuda.synchronize()
        assert same(there, want)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed in (7, 8, 9):
        x.copy_(normal((6, 128), seed).half())
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs[0]]
        assert same(outs[1], replayed) and same(step(), replayed)


def test_large_calls_in_graphs(cuda):
    """A prompt's product, experts of many pairs and the sampling of many rows, captured twice and replayed at once on two
    streams with new inputs, and with shares of the work that change from replay to replay."""
    import torch

    from nvcr_b200 import tokens

    matrix = tokens.ByteMatrix.quantise(normal((2100, 512), 1, 0.1))
    experts = tokens.ByteExperts.quantise(normal((6, 700, 512), 2, 0.1))
    x, weights = normal((1500, 512), 3).bfloat16(), torch.rand((1500, 2), device="cuda")
    choices = some_choices(1500, 2, 6, 4)
    logits, u = normal((200, 40000), 5, 3.0).bfloat16(), torch.rand(200, device="cuda")
    top_p = torch.full((200,), 0.8, device="cuda")

    def step():
        return (matrix.multiply(x), experts.multiply(x, choices, weights), experts.multiply(x, choices),
                *tokens.sample(logits, u, temperature=0.9, top_p=top_p))

    same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
    step()
    torch.cuda.synchronize()
    side, graphs, outs = torch.cuda.Stream(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed, kind in ((7, "one"), (8, "absent"), (9, "skewed")):
        x.copy_(normal((1500, 512), seed).bfloat16())
        choices.copy_(some_choices(1500, 2, 6, seed, kind))
        logits.copy_(normal((200, 40000), seed, float(seed - 5)).bfloat16())
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs[0]]
        assert same(outs[1], replayed) and same(step(), replayed)
    matrix.check(), experts.check()


def test_weights_written_just_before(cuda):
    """A product enqueued right behind the kernels that write its weights, again and again with other ones."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    x = torch.ones((1, 4096), device="cuda")
    codes = torch.empty((4096, 4096), dtype=torch.int8, device="cuda")
    scales = torch.ones(4096, device="cuda")
    out = []
    for n in range(30):
        codes.fill_(n + 1)
        out.append(ByteMatrix(codes, scales).multiply(x))
    for n, y in enumerate(out):
        want = (n + 1) * 127 * 4096 * torch.tensor(1.0 / 127.0)
        assert (y - want).abs().max() <= 4 * E * want, n


def test_results_are_the_same_bits_again(cuda):
    """Whatever atomics decide inside: the same calls give the same bits."""
    import torch

    from nvcr_b200 import tokens

    experts = tokens.ByteExperts(some_codes((9, 300, 256), 1), normal((9, 300), 2, 0.01).abs())
    x, weights, choices = normal((3000, 256), 3).half(), normal((3000, 3), 4), some_choices(3000, 3, 9, 5, "absent")
    logits, u = normal((180, 50001), 6, 2.0).half(), torch.rand(180, device="cuda")
    calls = [lambda: (experts.multiply(x, choices, weights),), lambda: tokens.sample(logits, u, top_p=0.95),
             lambda: tokens.sample(logits[:1], u[:1], top_k=2000), lambda: tokens.route(logits[:, :256], 8, kind="sigmoid")]
    for call in calls:
        first = [t.clone() for t in call()]
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_workspaces_of_a_given_stream_are_its_own(cuda):
    """A call on a busy stream keeps its working memory until that stream has run it."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    matrix, x = ByteMatrix.quantise(normal((512, 1024), 1)), normal((64, 1024), 2).half()
    want, side = matrix.multiply(x), torch.cuda.Stream()
    product = torch.zeros((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            product = product @ product
    got = matrix.multiply(x, stream=side)
    for size in (1 << 16, 64 * 1024, 64 * 1024 + 256, 1 << 17):  # this stream's work over what the call has released
        [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_check_tells_of_waits_that_ran_out(cuda):
    from nvcr_b200.executor import ErrorCode, ExecutorError
    from nvcr_b200.tokens import ByteMatrix

    matrix = ByteMatrix.quantise(normal((8, 8), 1))
    matrix.check()
    matrix.status.fill_(1)  # as a kernel would
    with pytest.raises(ExecutorError, match="wait") as error:
        matrix.check()
    assert error.value.code == ErrorCode.backend_error
    matrix.check()


def test_wrong_tensors_are_refused(cuda):
    import torch

    from nvcr_b200 import tokens
    from nvcr_b200.executor import ErrorCode, ExecutorError

    def of(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    whole, real = torch.int32, torch.float32
    matrix = tokens.ByteMatrix(of(4, 64, dtype=torch.int8), of(4, dtype=real))
    experts = tokens.ByteExperts(of(2, 4, 64, dtype=torch.int8), of(2, 4, dtype=real))
    x, choices, scores, uniforms = of(3, 64), of(3, 2, dtype=whole), of(3, 8), of(3, dtype=real)
    refused = [
        lambda: tokens.ByteMatrix(of(4, 64), of(4, dtype=real)),
        lambda: tokens.ByteMatrix(of(4, 64, dtype=torch.int8), of(4)),
        lambda: tokens.ByteMatrix(of(4, 64, dtype=torch.int8), of(5, dtype=real)),
        lambda: tokens.ByteMatrix(of(64, 4, dtype=torch.int8).t(), of(4, dtype=real)),
        lambda: tokens.ByteMatrix(of(4, 0, dtype=torch.int8), of(4, dtype=real)),
        lambda: tokens.ByteMatrix(of(1, 131073, dtype=torch.int8), of(1, dtype=real)),
        lambda: tokens.ByteExperts(of(2, 4, 64, dtype=torch.int8), of(2, 5, dtype=real)),
        lambda: tokens.ByteExperts(of(1025, 1, 1, dtype=torch.int8), of(1025, 1, dtype=real)).multiply(of(1, 1), of(1, 1, dtype=whole)),
        lambda: matrix.multiply(of(3, 65)), lambda: matrix.multiply(of(64)), lambda: matrix.multiply(of(3, 64, dtype=torch.int8)),
        lambda: matrix.multiply(of(64, 3).t()), lambda: matrix.multiply(x, of(5)), lambda: matrix.multiply(x, of(4, dtype=real)),
        lambda: matrix.multiply(x.cpu()), lambda: matrix.multiply(None),
        lambda: experts.multiply(of(2, 64), choices), lambda: experts.multiply(of(3, 3, 64), choices),
        lambda: experts.multiply(x, of(3, 2)), lambda: experts.multiply(x, of(3, dtype=whole)),
        lambda: experts.multiply(x, of(2, 3, dtype=whole).t()), lambda: experts.multiply(x, of(3, 0, dtype=whole)),
        lambda: experts.multiply(x, choices, of(3, 2)), lambda: experts.multiply(x, choices, of(3, 3, dtype=real)),
        lambda: experts.multiply(of(64), choices), lambda: experts.multiply(x, choices.cpu()),
        lambda: tokens.route(scores, 9), lambda: tokens.route(scores, 0), lambda: tokens.route(scores, 2, groups=3),
        lambda: tokens.route(scores, 2, groups=2, kept_groups=3), lambda: tokens.route(scores, 2, scale=math.inf),
        lambda: tokens.route(scores, 2, bias=of(8)), lambda: tokens.route(scores, 2, bias=of(7, dtype=real)),
        lambda: tokens.route(of(8, 3).t(), 2), lambda: tokens.route(of(2, 1025), 2),
        lambda: tokens.sample(scores, of(3)), lambda: tokens.sample(scores, of(4, dtype=real)),
        lambda: tokens.sample(scores, uniforms.cpu()), lambda: tokens.sample(scores, uniforms, top_k=of(3, dtype=torch.int64)),
        lambda: tokens.sample(scores, uniforms, top_p=of(3, dtype=torch.float64)),
        lambda: tokens.sample(scores, uniforms, temperature=of(4, dtype=real)), lambda: tokens.sample(of(8, 3).t(), uniforms),
        lambda: tokens.sample(of(3, (1 << 20) + 1), uniforms), lambda: tokens.sample(of(3, 0), uniforms),
        lambda: tokens.sample(scores, uniforms, top_k=1 << 40),
    ]
    for nth, call in enumerate(refused):
        with pytest.raises(ExecutorError) as error:
            call()
        assert error.value.code == ErrorCode.invalid_argument, nth
    for call in (lambda: tokens.sample(scores, uniforms, top_p="0.9"), lambda: tokens.route(scores, 2.5)):
        with pytest.raises(TypeError):
            call()
