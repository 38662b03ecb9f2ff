"""Waits that run out in the products of 8-bit weights, on the GPU and without a fault: one block of the product's kernel is
told to copy nothing, so that the waits for its copies give up after 20 ms. The call ends, says so in the status word,
and writes either a product's right value or nothing; the next call is as always."""
from __future__ import annotations

import ctypes

import pytest

pytestmark = pytest.mark.gpu

LIMIT_MS = 20
MARK = -12345.5  # no product here has it: a factor of every scale is 2^-9, of MARK's 2^-1
FLOAT32 = 2


def lib():
    from nvcr_b200.executor import library

    return library()


def some(shape, seed):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=make, device="cuda")


def codes_of(shape, seed):
    import torch

    make = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=make, device="cuda", dtype=torch.int8)


def room_of(bytes):
    """A workspace of bytes that stand for no sensible numbers: 0x7f7f7f7f is 3.4e38."""
    import torch

    return torch.full((bytes,), 0x7F, dtype=torch.uint8, device="cuda")


def given_up(run, shape, want):
    """One call with a block of it given up and one without: which elements the first one wrote."""
    import torch

    y = torch.full(shape, MARK, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    run(y, status)
    torch.cuda.synchronize()
    written = y != MARK
    assert int(status.item()) == 1
    assert torch.equal(y[written], want[written])
    status.zero_()
    again = torch.full(shape, MARK, device="cuda")
    run(again, status, test=False)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and torch.equal(again, want)
    return written


def matrix_case(rows, inputs, outputs, block):
    import torch

    from nvcr_b200.tokens import ByteMatrix

    matrix = ByteMatrix(codes_of((outputs, inputs), 1), torch.full((outputs,), 2.0 ** -9, device="cuda"))
    x = some((rows, inputs), 2)
    want = matrix.multiply(x)
    size = ctypes.c_size_t(0)
    assert lib().nvcr_sm100_token_bytes_workspace(rows, outputs, inputs, ctypes.byref(size)) == 0
    room = room_of(size.value)

    other = some((rows, inputs), 4)

    def run(y, status, test=True):
        matrix.multiply(other)  # whose sums stay in shared memory
        if test:
            assert lib().nvcr_sm100_token_test_wait_timeout(LIMIT_MS, block) == 0
        assert lib().nvcr_sm100_token_bytes_multiply(
            FLOAT32, x.data_ptr(), x.stride(0), rows, matrix._addresses[0], matrix._addresses[1], outputs, inputs, None,
            y.data_ptr(), room.data_ptr(), size.value, status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0

    return given_up(run, (rows, outputs), want)


def experts_case(tokens, chosen, experts, inputs, outputs, block, weighted):
    import torch

    from nvcr_b200.tokens import ByteExperts

    matrices = ByteExperts(codes_of((experts, outputs, inputs), 1), torch.full((experts, outputs), 2.0 ** -9, device="cuda"))
    x = some((tokens, inputs), 2)
    choices = (torch.arange(tokens * chosen, device="cuda", dtype=torch.int32) % experts).view(tokens, chosen)
    weights = some((tokens, chosen), 3) if weighted else None
    want = matrices.multiply(x, choices, weights)
    size = ctypes.c_size_t(0)
    assert lib().nvcr_sm100_token_experts_workspace(tokens, chosen, int(weighted), experts, outputs, inputs, ctypes.byref(size)) == 0
    room = room_of(size.value)

    other = some((tokens, inputs), 4)

    def run(y, status, test=True):
        room.fill_(0x7F)
        matrices.multiply(other, choices)
        if test:
            assert lib().nvcr_sm100_token_test_wait_timeout(LIMIT_MS, block) == 0
        assert lib().nvcr_sm100_token_experts_multiply(
            FLOAT32, x.data_ptr(), x.stride(0), 0, 0, tokens, choices.data_ptr(), chosen,
            weights.data_ptr() if weighted else None, matrices._addresses[0], matrices._addresses[1], experts, outputs, inputs,
            y.data_ptr(), room.data_ptr(), size.value, status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0

    return given_up(run, tuple(want.shape), want)


@pytest.mark.parametrize("block", [0, 1, 3, 6])
def test_a_block_of_a_shared_tile_gives_up(cuda, block):
    """Four blocks have a part of a tile's inputs each: without one of them there is no sum, and none is stored."""
    written = matrix_case(20, 2048, 300, block)
    assert not written.all() and written.any()


@pytest.mark.parametrize("block", [0, 5])
def test_a_block_of_a_shared_tile_of_experts_gives_up(cuda, block):
    written = experts_case(100, 2, 4, 2048, 300, block, weighted=False)
    assert not written.all() and written.any()


@pytest.mark.parametrize("block", [0, 100])
def test_a_block_with_tiles_of_its_own_gives_up(cuda, block):
    written = matrix_case(300, 256, 20000, block)
    assert not written.all() and written.any()
    written = experts_case(1000, 2, 5, 129, 257, block, weighted=False)
    assert not written.all() and written.any()


@pytest.mark.parametrize("block", [0, 1, 17])
def test_a_block_of_a_pair_gives_up(cuda, block):
    written = matrix_case(2048, 4096, 2048, block)
    assert not written.all() and written.any()
    written = experts_case(2000, 2, 4, 4096, 2048, block, weighted=False)
    assert not written.all() and written.any()


@pytest.mark.parametrize("block", [0, 5])
@pytest.mark.parametrize("tokens,chosen,experts,inputs,outputs", [(100, 2, 4, 2048, 300), (1000, 2, 5, 129, 257), (2000, 2, 4, 4096, 2048)])
def test_sums_over_experts_of_a_call_that_gave_up_are_not_written(cuda, tokens, chosen, experts, inputs, outputs, block):
    """Every token's sum needs products of several blocks, so none of the call's is stored."""
    assert not experts_case(tokens, chosen, experts, inputs, outputs, block, weighted=True).any()
