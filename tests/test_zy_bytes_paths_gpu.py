"""Products in 8 bits by each of their kernels, on the GPU, where the sizes of the other tests leave one out: experts whose
tiles two blocks share, such calls captured, and weights that are written right before each kernel reads them.

Which kernel a size takes: up to two rows, or a few with little to multiply, one launch without the tensor cores; few tiles
one by four blocks each; many inputs and rows (or rows an expert) a pair of blocks each; others a block each. Tolerances: a
product's sum of codes is exact and is rounded three times to 2^-24 on its way to FP32 (a fourth time, to the output's
type); a weighted sum over `chosen` products adds two roundings of each."""
from __future__ import annotations

import pytest

from tests.test_zy_bytes_gpu import E, check_experts, check_matrix, normal, some_choices, some_codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("kind", ["spread", "skewed", "absent"])
def test_experts_by_pairs_of_blocks(cuda, kind, weighted, name):
    """An odd number of output tiles, the last of a few outputs; inputs that end within a block; rows of an expert that
    are no multiple of a pair's step."""
    tokens, chosen, experts, inputs, outputs = 1500, 3, 4, 3900, 1161
    x = normal((tokens, inputs), 1).to(getattr(__import__("torch"), name))
    weights = normal((tokens, chosen), 2) if weighted else None
    check_experts(x, some_codes((experts, outputs, inputs), 3), normal((experts, outputs), 4, 0.01).abs(),
                  some_choices(tokens, chosen, experts, 5, kind), weights, name)


def test_experts_by_pairs_with_rows_of_their_own(cuda):
    x = normal((1200, 2, 4096), 1).bfloat16()
    check_experts(x, some_codes((3, 2000, 4096), 3), normal((3, 2000), 4, 0.01).abs(), some_choices(1200, 2, 3, 5), None, "bfloat16")


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,inputs,outputs", [(1000, 4096, 4096), (1037, 4000, 2100), (2048, 4096, 1161), (4100, 8192, 129)])
def test_matrix_by_pairs_of_blocks(cuda, rows, inputs, outputs, name):
    check_matrix(rows, inputs, outputs, name, bias=rows % 2 == 1)


def test_pairs_of_blocks_in_graphs(cuda):
    """Captured twice and replayed at once on two streams with new inputs and choices: as eager calls."""
    import torch

    from nvcr_b200.tokens import ByteExperts, ByteMatrix

    matrix = ByteMatrix.quantise(normal((2100, 4096), 1, 0.1))
    experts = ByteExperts.quantise(normal((4, 1161, 4096), 2, 0.1))
    x, choices, weights = normal((1500, 4096), 3).half(), some_choices(1500, 2, 4, 4), normal((1500, 2), 5)

    def step():
        return matrix.multiply(x), experts.multiply(x, choices), experts.multiply(x, choices, weights)

    step()
    torch.cuda.synchronize()
    side, graphs, outs = torch.cuda.Stream(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for seed, kind in ((7, "one"), (8, "absent"), (9, "skewed")):
        x.copy_(normal((1500, 4096), seed).half())
        choices.copy_(some_choices(1500, 2, 4, seed, kind))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for eager, one, other in zip(step(), *outs):
            assert torch.equal(eager, one) and torch.equal(eager, other)
    matrix.check(), experts.check()


@pytest.mark.parametrize("rows,inputs,outputs", [(1, 4096, 4096), (32, 4096, 4096), (40, 16384, 1024), (32, 512, 20000),
                                                 (1000, 4096, 4096)])
def test_products_right_behind_their_weights(cuda, rows, inputs, outputs):
    """Weights laid out, or copied over, right before the product that reads them, behind kernels that let the next ones start
    early: one matrix's weights are on their way to shared memory before the product waits for the kernel before it."""
    import torch

    from nvcr_b200.tokens import ByteMatrix

    x = torch.ones((rows, inputs), device="cuda")
    codes = torch.empty((outputs, inputs), dtype=torch.int8, device="cuda")
    scales = torch.ones(outputs, device="cuda")
    ahead = ByteMatrix(torch.ones((512, 512), dtype=torch.int8, device="cuda"), torch.ones(512, device="cuda"))
    one_row = torch.ones((1, 512), device="cuda")
    kept = ByteMatrix(codes.fill_(0), scales)
    made, copied = [], []
    for n in range(30):
        codes.fill_(n + 1)
        ahead.multiply(one_row)
        matrix = ByteMatrix(codes, scales)
        made.append(matrix.multiply(x)[:: max(1, rows - 1)])
        ahead.multiply(one_row)
        kept.codes.copy_(matrix.codes)
        copied.append(kept.multiply(x)[:: max(1, rows - 1)])
    for n, ys in enumerate(zip(made, copied)):
        want = (n + 1) * 127 * inputs * torch.tensor(1.0 / 127.0)
        for y in ys:
            assert (y - want).abs().max() <= 4 * E * want, n


def test_experts_right_behind_their_weights(cuda):
    import torch

    from nvcr_b200.tokens import ByteExperts

    scales, choices = torch.ones((4, 1024), device="cuda"), some_choices(64, 2, 4, 1)
    x = torch.ones((64, 2048), device="cuda")
    made = []
    codes = torch.empty((4, 1024, 2048), dtype=torch.int8, device="cuda")
    for n in range(30):
        codes.fill_(n + 1)
        made.append(ByteExperts(codes, scales).multiply(x, choices))
    for n, y in enumerate(made):
        want = (n + 1) * 127 * 2048 * torch.tensor(1.0 / 127.0)
        assert (y - want).abs().max() <= 4 * E * want, n
