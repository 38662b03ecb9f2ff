"""The token operators' refusals (no GPU): each call refuses, with
NVCR_SM100_INVALID_ARGUMENT and before any launch, what its header comment
excludes; and the Python wrappers refuse tensors they cannot hand on. Only
refused cases reach the C ABI here, so the buffers may be host memory."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

INVALID = 1  # NVCR_SM100_INVALID_ARGUMENT


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


def cache(room, **changes):
    from nvcr_b200.tokens import _Cache

    fields = dict(key_codes=room, key_scales=room, value_codes=room, value_scales=room, status=None, pages=4,
                  kv_heads=2, page_size=16, head_dim=128, group=64)
    fields.update(changes)
    return _Cache(**fields)


CACHES = [dict(key_codes=None), dict(value_scales=None), dict(pages=0), dict(kv_heads=0), dict(page_size=0),
          dict(page_size=24), dict(head_dim=96), dict(head_dim=512), dict(group=16), dict(group=128, head_dim=64),
          dict(group=32, head_dim=256), dict(group=256, head_dim=256)]


def append_args(room, **changes):
    fields = dict(type=0, keys=room, ks=256, kh=128, values=room, vs=256, vh=128, slots=room, tokens=1, queries=None,
                  qs=0, qh=0, heads=0, rotated=None, positions=None, cosines=None, sines=None, rows=0, rotary=0,
                  interleaved=0, stream=None)
    fields.update(changes)
    return list(fields.values())


def attend_args(room, **changes):
    fields = dict(type=0, queries=room, qs=1024, qh=128, tokens=3, heads=8, table=room, ts=4, columns=4, lengths=room,
                  batch=3, offsets=None, max_queries=1, max_length=64, scale=1.0, output=room, stream=None)
    fields.update(changes)
    return list(fields.values())


def test_norm_refuses(lib, room):
    def call(**changes):
        fields = dict(type=0, layer=0, post=0, block=room, bs=8, residual=None, rs=0, gate=None, gs=0, pw=None, pb=None,
                      qw=None, qb=None, hidden=room, normed=None, rows=2, width=8, scale=1.0, offset=0.0, epsilon=1e-6,
                      stream=None)
        fields.update(changes)
        return lib.nvcr_sm100_token_norm(*fields.values())

    for changes in (dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 31), dict(width=0), dict(block=None),
                    dict(hidden=None), dict(epsilon=-1.0), dict(epsilon=float("nan"))):
        assert call(**changes) == INVALID, changes


def test_cache_shapes_are_refused(lib, room):
    for changes in CACHES + [dict(key_codes=room + 8)]:
        bad = cache(room, **changes)
        at = ctypes.addressof(bad)
        assert lib.nvcr_sm100_token_append(at, *append_args(room)) == INVALID, changes
        assert lib.nvcr_sm100_token_read(at, 0, room, 1, room, room, None) == INVALID, changes
        assert lib.nvcr_sm100_token_attend(room, at, *attend_args(room)) == INVALID, changes
    assert lib.nvcr_sm100_token_append(None, *append_args(room)) == INVALID
    assert lib.nvcr_sm100_token_read(None, 0, room, 1, room, room, None) == INVALID


def test_append_and_read_refuse(lib, room):
    good = cache(room)
    at = ctypes.addressof(good)
    table = dict(positions=room, cosines=room, sines=room, rows=4, rotary=128)
    for changes in (dict(type=2), dict(type=5), dict(tokens=-1), dict(keys=None), dict(values=None), dict(slots=None),
                    dict(queries=room, heads=4), dict(queries=room, rotated=room, heads=0),
                    {**table, "cosines": None}, {**table, "rows": 0}, {**table, "rotary": 0}, {**table, "rotary": 63},
                    {**table, "rotary": 130}):
        assert lib.nvcr_sm100_token_append(at, *append_args(room, **changes)) == INVALID, changes
    for call in ((3, room, 1, room, room), (0, None, 1, room, room), (0, room, -1, room, room), (0, room, 1, None, room),
                 (0, room, 1, room, None)):
        assert lib.nvcr_sm100_token_read(at, *call, None) == INVALID, call


def test_attend_refuses(lib, room):
    good = cache(room)
    at = ctypes.addressof(good)
    assert lib.nvcr_sm100_token_attend(None, at, *attend_args(room)) == INVALID
    for changes in (dict(type=2), dict(tokens=-1), dict(batch=-1), dict(heads=0), dict(heads=7), dict(max_queries=0),
                    dict(tokens=4), dict(max_length=65), dict(max_length=-1), dict(scale=float("inf")),
                    dict(scale=float("nan")), dict(queries=None), dict(table=None), dict(lengths=None),
                    dict(output=None)):
        assert lib.nvcr_sm100_token_attend(room, at, *attend_args(room, **changes)) == INVALID, changes
    assert lib.nvcr_sm100_token_context_create(None) == INVALID


def test_matrices_refuse(lib, room):
    sizes = [ctypes.byref(ctypes.c_size_t(0)) for _ in range(2)]
    for shape in ((0, 64, 64), (4, 0, 64), (4, 96, 64), (4, 64, 16), (4, 64, 48), (-1, 64, 64)):
        assert lib.nvcr_sm100_token_packed_bytes(*shape, *sizes) == INVALID, shape
        assert lib.nvcr_sm100_token_pack(room, room, room, *shape, room, room, None) == INVALID, shape
        assert lib.nvcr_sm100_token_multiply(0, room, 64, 1, room, room, *shape, None, room, None) == INVALID, shape
    assert lib.nvcr_sm100_token_packed_bytes(4, 64, 64, None, sizes[1]) == INVALID
    assert lib.nvcr_sm100_token_packed_bytes(4, 64, 64, *sizes) == 0
    for bad in range(5):
        pointers = [room] * 5
        pointers[bad] = None
        assert lib.nvcr_sm100_token_pack(*pointers[:3], 4, 64, 64, *pointers[3:], None) == INVALID, bad
    assert lib.nvcr_sm100_token_pack(room, room, room, 4, 64, 64, room + 4, room, None) == INVALID
    for changes in ((2, room, 64, 1, room, room), (0, None, 64, 1, room, room), (0, room, 64, -1, room, room),
                    (0, room, 64, 1, None, room), (0, room, 64, 1, room, None), (0, room, 64, 1, room + 2, room)):
        assert lib.nvcr_sm100_token_multiply(*changes, 4, 64, 64, None, room, None) == INVALID, changes
    assert lib.nvcr_sm100_token_multiply(0, room, 64, 1, room, room, 4, 64, 64, None, None, None) == INVALID


def test_wrappers_refuse_host_tensors(built_library):
    import torch

    from nvcr_b200 import tokens
    from nvcr_b200.executor import ErrorCode, ExecutorError

    refused = [
        lambda: tokens.block_norm(torch.zeros(2, 8)),
        lambda: tokens.block_norm(torch.zeros(2, 8, dtype=torch.int32)),
        lambda: tokens.block_norm(torch.zeros(8)),
        lambda: tokens.block_norm(torch.zeros(2, 8), kind="batch"),
        lambda: tokens.block_norm(torch.zeros(2, 8), hidden=False, normed=False),
        lambda: tokens.block_norm(torch.zeros(2, 8), residual=torch.zeros(2, 9)),
        lambda: tokens.block_norm(torch.zeros(2, 8), gate=torch.zeros(9)),
        lambda: tokens.block_norm(torch.zeros(2, 8), pre_weight=torch.zeros(8, dtype=torch.float16)),
        lambda: tokens.PagedCache.empty(2, 2, 16, 128, 64, device="cpu"),
        lambda: tokens.PagedCache.empty(2, 2, 16, 128, 48, device="cpu"),
        lambda: tokens.PackedMatrix(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1).half(),
                                    torch.zeros(4, 1).half()),
        lambda: tokens.PackedMatrix.quantise(torch.zeros(4, 65), 32),
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

    def there(*shape, dtype=torch.float16):
        with FakeTensorMode():
            return torch.empty(shape, dtype=dtype, device="cuda:1")

    keeper = cache(room)
    at, native = ctypes.addressof(keeper), tokens._native()
    keys, slots = there(1, 2, 128), there(1, dtype=torch.int64)
    assert keys.is_cuda and keys.get_device() == 1
    refused = [
        lambda: tokens.block_norm(there(2, 8)),
        lambda: native.append(at, 1, keys, keys, slots, None, None, None, None, False, None),
        lambda: native.read(at, 1, slots, 0, None),
        lambda: native.attend(room, at, 1, there(1, 4, 128), there(1, 4, dtype=torch.int32), there(1, dtype=torch.int32),
                              None, 1, 64, None, None),
        lambda: native.multiply(room, room, 4, 64, 64, 1, there(1, 64), None, None),
        lambda: tokens.PackedMatrix(there(4, 32, dtype=torch.uint8), there(4, 1), there(4, 1)),
    ]
    for call in refused:
        with pytest.raises(ExecutorError, match="not the current CUDA device") as error:
            call()
        assert error.value.code == ErrorCode.invalid_argument


def test_places_past_the_page_table_become_no_slot():
    """The model's slots on the CPU, where an index out of range raises (on the device it would end the process)."""
    import torch

    from nvcr_b200.token_model import TokenModel

    pages = torch.tensor([[2, 0, 4], [3, 1, 4]], dtype=torch.int32)  # two columns, and one of no page
    places = torch.tensor([[0, 17, 31, 32, 33], [15, 16, 47, 48, 1 << 30]], dtype=torch.int32)
    slots = TokenModel._slots(pages, places, 16)
    assert slots.dtype == torch.int64
    assert slots.tolist() == [32, 1, 15, 64, 64, 63, 16, 64, 64, 64]


def test_sizes_past_32_bit_places_are_refused(lib, room):
    """A row, a sequence or a matrix whose last places' 32-bit successors would overflow."""
    last = (1 << 31) - 1
    sizes = [ctypes.byref(ctypes.c_size_t(0)) for _ in range(2)]
    for outputs in (last, last - 14):
        assert lib.nvcr_sm100_token_packed_bytes(outputs, 32, 32, *sizes) == INVALID
        assert lib.nvcr_sm100_token_multiply(0, room, 32, 1, room, room, outputs, 32, 32, None, room, None) == INVALID
    assert lib.nvcr_sm100_token_packed_bytes(last - 15, 32, 32, *sizes) == 0
    for width in (last, (1 << 30) + 1):
        assert lib.nvcr_sm100_token_norm(0, 0, 0, room, width, None, 0, None, 0, None, None, None, None, room, None, 2,
                                         width, 1.0, 0.0, 1e-6, None) == INVALID
    at = ctypes.addressof(keeper := cache(room))
    for length in (last, (1 << 30) + 1):
        changes = dict(max_length=length, columns=1 << 27)
        assert lib.nvcr_sm100_token_attend(room, at, *attend_args(room, **changes)) == INVALID
    del keeper


def test_binding_follows_torch(built_library, monkeypatch):
    """Built anew for another torch, not for the same one; without torch the library alone is built."""
    from nvcr_b200 import build

    class Compiled(Exception):
        pass

    def compiler(*_args, **_options):
        raise Compiled

    monkeypatch.setattr(build.subprocess, "run", compiler)
    assert build.build() == build.LIBRARY and build.build_binding() == build.BINDING
    monkeypatch.setattr(build.importlib.metadata, "version", lambda _name: "0.0.1")
    with pytest.raises(Compiled):
        build.build_binding()
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda _name: None)
    assert build.build_binding() is None and build.build() == build.LIBRARY
