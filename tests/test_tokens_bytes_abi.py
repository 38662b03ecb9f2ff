"""Refusals of the products in 8 bits, the routing and the sampling (no GPU): each call refuses, with
NVCR_SM100_INVALID_ARGUMENT and before any launch, what its header comment
excludes; and the Python wrappers refuse tensors they cannot hand on. Only
refused cases reach the C ABI here, so the buffers may be host memory."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

INVALID = 1  # NVCR_SM100_INVALID_ARGUMENT
LAST = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(built_library):
    from nvcr_b200.executor import library

    return library()


@pytest.fixture(scope="module")
def room():
    """A 16-byte aligned host address."""
    array = np.zeros(4096 + 16, np.uint8)
    yield (array.ctypes.data + 15) // 16 * 16
    del array


def size():
    return ctypes.byref(ctypes.c_size_t(0))


SHAPES = [(0, 64), (-1, 64), (4, 0), (4, -5), (4, 131073), ((1 << 24) + 1, 64), (LAST, 64)]


def test_shapes_are_refused(lib, room):
    for outputs, inputs in SHAPES:
        assert lib.nvcr_sm100_token_bytes_packed(1, outputs, inputs, size()) == INVALID
        assert lib.nvcr_sm100_token_bytes_pack(room, 1, outputs, inputs, room, None) == INVALID
        assert lib.nvcr_sm100_token_bytes_workspace(1, outputs, inputs, size()) == INVALID
        assert lib.nvcr_sm100_token_bytes_multiply(0, room, 64, 1, room, room, outputs, inputs, None, room, room, 4096,
                                                   None, None) == INVALID
        assert lib.nvcr_sm100_token_experts_workspace(1, 1, 0, 2, outputs, inputs, size()) == INVALID
        assert lib.nvcr_sm100_token_experts_multiply(0, room, 64, 0, 0, 1, room, 1, None, room, room, 2, outputs, inputs,
                                                     room, room, 4096, None, None) == INVALID
    assert lib.nvcr_sm100_token_bytes_packed(0, 4, 64, size()) == INVALID
    assert lib.nvcr_sm100_token_bytes_packed(1, 4, 64, None) == INVALID
    assert lib.nvcr_sm100_token_bytes_workspace(1, 4, 64, None) == INVALID
    assert lib.nvcr_sm100_token_bytes_workspace(-1, 4, 64, size()) == INVALID
    assert lib.nvcr_sm100_token_bytes_workspace(LAST, 4, 64, size()) == INVALID
    assert lib.nvcr_sm100_token_bytes_pack(None, 1, 4, 64, room, None) == INVALID
    assert lib.nvcr_sm100_token_bytes_pack(room, 1, 4, 64, None, None) == INVALID
    assert lib.nvcr_sm100_token_bytes_pack(room, 1, 4, 64, room + 8, None) == INVALID


def test_packed_sizes(lib):
    """128 x 128 blocks, past 32 bits too."""
    for matrices, outputs, inputs, blocks in ((1, 1, 1, 1), (1, 128, 128, 1), (2, 129, 300, 12), (1024, 1 << 15, 1 << 14, 1 << 25)):
        found = ctypes.c_size_t(0)
        assert lib.nvcr_sm100_token_bytes_packed(matrices, outputs, inputs, ctypes.byref(found)) == 0
        assert found.value == blocks * 16384


def multiply(lib, room, **changes):
    fields = dict(type=0, x=room, stride=64, rows=2, packed=room, scales=room, outputs=4, inputs=64, bias=None, y=room,
                  workspace=room, bytes=4096, status=None, stream=None)
    fields.update(changes)
    return lib.nvcr_sm100_token_bytes_multiply(*fields.values())


def test_multiply_refuses(lib, room):
    need = ctypes.c_size_t(0)
    assert lib.nvcr_sm100_token_bytes_workspace(2, 4, 64, ctypes.byref(need)) == 0
    for changes in (dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=LAST), dict(x=None), dict(packed=None),
                    dict(scales=None), dict(y=None), dict(workspace=None), dict(packed=room + 8), dict(workspace=room + 4),
                    dict(bytes=need.value - 1), dict(bytes=0)):
        assert multiply(lib, room, **changes) == INVALID, changes
    assert multiply(lib, room, rows=0, x=None, y=None, workspace=None, bytes=0) == 0  # nothing to launch


def experts(lib, room, **changes):
    fields = dict(type=0, x=room, stride=64, row_stride=0, each=0, tokens=2, choices=room, chosen=2, weights=None, packed=room,
                  scales=room, experts=4, outputs=4, inputs=64, y=room, workspace=room, bytes=1 << 20, status=None, stream=None)
    fields.update(changes)
    return lib.nvcr_sm100_token_experts_multiply(*fields.values())


def test_experts_refuse(lib, room):
    need = ctypes.c_size_t(0)
    assert lib.nvcr_sm100_token_experts_workspace(2, 2, 0, 4, 4, 64, ctypes.byref(need)) == 0
    for changes in (dict(type=3), dict(tokens=-1), dict(tokens=1 << 30), dict(chosen=0), dict(chosen=-1), dict(experts=0),
                    dict(experts=1025), dict(x=None), dict(choices=None), dict(packed=None), dict(scales=None), dict(y=None),
                    dict(workspace=None), dict(packed=room + 8), dict(workspace=room + 8), dict(bytes=need.value - 1),
                    dict(weights=room, bytes=need.value)):
        assert experts(lib, room, **changes) == INVALID, changes
    assert experts(lib, room, tokens=0, x=None, choices=None, y=None, workspace=None, bytes=0) == 0
    for shape in ((1, 0, 0, 4), (-1, 1, 0, 4), (1 << 30, 2, 0, 4), (1, 1, 0, 0), (1, 1, 0, 1025)):
        assert lib.nvcr_sm100_token_experts_workspace(*shape, 4, 64, size()) == INVALID
    assert lib.nvcr_sm100_token_experts_workspace(1, 1, 0, 4, 4, 64, None) == INVALID


def test_route_refuses(lib, room):
    def call(**changes):
        fields = dict(type=0, scores=room, stride=8, tokens=2, experts=8, count=2, sigmoid=0, bias=None, groups=1, kept=1,
                      renormalise=0, scale=1.0, choices=room, weights=room, stream=None)
        fields.update(changes)
        return lib.nvcr_sm100_token_route(*fields.values())

    for changes in (dict(type=3), dict(type=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(experts=0), dict(experts=1025),
                    dict(count=0), dict(count=9), dict(groups=0), dict(groups=3), dict(groups=16), dict(kept=0), dict(kept=2),
                    dict(groups=4, kept=5), dict(scale=math.nan), dict(scale=math.inf), dict(scores=None),
                    dict(choices=None), dict(weights=None)):
        assert call(**changes) == INVALID, changes
    assert call(tokens=0, scores=None, choices=None, weights=None) == 0


def test_sample_refuses(lib, room):
    def call(**changes):
        fields = dict(type=0, logits=room, stride=8, rows=2, symbols=8, uniforms=room, temperatures=None, temperature=1.0,
                      top_ks=None, top_k=0, top_ps=None, top_p=1.0, min_ps=None, min_p=0.0, chosen=room, probabilities=room,
                      workspace=None, bytes=0, stream=None)
        fields.update(changes)
        return lib.nvcr_sm100_token_sample(*fields.values())

    for changes in (dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 31), dict(symbols=0), dict(symbols=(1 << 20) + 1),
                    dict(logits=None), dict(uniforms=None), dict(chosen=None), dict(probabilities=None), dict(workspace=room + 8),
                    dict(rows=1000, symbols=100000), dict(rows=1000, symbols=100000, workspace=room, bytes=4096)):
        assert call(**changes) == INVALID, changes
    for changes in ((3, 1, 8), (0, -1, 8), (0, 1 << 31, 8), (0, 1, 0), (0, 1, (1 << 20) + 1)):
        assert lib.nvcr_sm100_token_sample_workspace(*changes, size()) == INVALID
    assert lib.nvcr_sm100_token_sample_workspace(0, 1, 8, None) == INVALID
    assert call(rows=0, logits=None, uniforms=None, chosen=None, probabilities=None) == 0


def test_wrappers_refuse_host_tensors(built_library):
    import torch

    from nvcr_b200 import tokens
    from nvcr_b200.executor import ErrorCode, ExecutorError

    scores = torch.zeros(2, 8)
    refused = [
        lambda: tokens.ByteMatrix(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)),
        lambda: tokens.ByteMatrix(torch.zeros(4, dtype=torch.int8), torch.zeros(4)),
        lambda: tokens.ByteMatrix.quantise(torch.zeros(4, 32)),
        lambda: tokens.ByteMatrix.quantise(torch.zeros(4)),
        lambda: tokens.ByteExperts(torch.zeros(2, 4, 32, dtype=torch.int8), torch.zeros(2, 4)),
        lambda: tokens.ByteExperts(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4)),
        lambda: tokens.ByteExperts.quantise(torch.zeros(4, 32)),
        lambda: tokens.ByteExperts.quantise(torch.zeros(2, 4, 32)),
        lambda: tokens.route(scores, 2),
        lambda: tokens.route(scores, 2, kind="tanh"),
        lambda: tokens.route(scores.int(), 2),
        lambda: tokens.route(scores[0], 2),
        lambda: tokens.sample(scores, torch.zeros(2)),
        lambda: tokens.sample(scores.int(), torch.zeros(2)),
        lambda: tokens.sample(scores[0], torch.zeros(2)),
    ]
    for call in refused:
        with pytest.raises(ExecutorError) as error:
            call()
        assert error.value.code == ErrorCode.invalid_argument


def test_tensors_of_another_device_are_refused(built_library, room):
    """Fake tensors stand for another device's; each call refuses before it takes an address from one or launches."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    from nvcr_b200 import tokens
    from nvcr_b200.executor import ErrorCode, ExecutorError

    if torch.cuda.is_available():
        pytest.skip("where there is a GPU, fake tensors want the device to exist")

    def there(*shape, dtype=torch.float16):
        with FakeTensorMode():
            return torch.empty(shape, dtype=dtype, device="cuda:1")

    native = tokens._native()
    refused = [
        lambda: native.bytes_multiply(room, room, 4, 64, room, 1, there(1, 64), None, None),
        lambda: native.experts_multiply(room, room, 2, 4, 64, room, 1, there(1, 64), there(1, 2, dtype=torch.int32), None, None),
        lambda: tokens.route(there(2, 8), 2),
        lambda: tokens.sample(there(2, 8), there(2, dtype=torch.float32)),
        lambda: tokens.ByteMatrix(there(4, 64, dtype=torch.int8), there(4, dtype=torch.float32)),
        lambda: tokens.ByteExperts(there(2, 4, 64, dtype=torch.int8), there(2, 4, dtype=torch.float32)),
    ]
    for call in refused:
        with pytest.raises(ExecutorError, match="not the current CUDA device") as error:
            call()
        assert error.value.code == ErrorCode.invalid_argument
