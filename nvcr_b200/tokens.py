"""The token operators through the C ABI: one step of a language model in low-bit form.

``block_norm`` is the norms after and before a block with its gate and residual;
``PagedCache`` holds keys and values in 4 bits, rotated on the way in;
``TokenContext.attend`` is attention over such a cache; ``PackedMatrix`` is a
4-bit weight matrix with group scales. Tensors are torch tensors on the current
CUDA device (another one's are refused); work is enqueued on torch's current
stream unless ``stream`` names another (then the caller orders the two, and keeps
the tensors alive). What the operators refuse raises ``ExecutorError``; there is
no CPU fallback. They are forward operators: an output has no gradient, whether or
not an input requires one.

The same call on the same kind of GPU gives the same bits; a token's may change
with the rest of its call, as the other rows and sequences decide the order of sums.

The 4-bit group form, of caches and weights alike: a group of consecutive values
is held as codes c in 0..15, two a byte with the even index in the low half, an
FP16 scale s and an FP16 minimum m, and stands for ``c * s + m``.
"""
from __future__ import annotations

import contextlib
import ctypes
import importlib.machinery
import importlib.util

import torch

from .build import BINDING
from .executor import ErrorCode, ExecutorError, _check, _stream_handle, library

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_KINDS = {"rms": 0, "layer": 1}
_module = None


class _Cache(ctypes.Structure):
    _fields_ = [("key_codes", ctypes.c_void_p), ("key_scales", ctypes.c_void_p), ("value_codes", ctypes.c_void_p),
                ("value_scales", ctypes.c_void_p), ("status", ctypes.c_void_p), ("pages", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("group", ctypes.c_int32)]


def _refuse(message: str) -> None:
    raise ExecutorError(ErrorCode.invalid_argument, message)


def _require(condition: bool, message: str) -> None:
    if not condition:
        _refuse(message)


def _native():
    """The compiled binding, loaded at its first use (raises if it is not built)."""
    global _module
    if _module is None:
        if not BINDING.exists():
            raise FileNotFoundError(f"{BINDING} is not built; run nvcr_b200.build.build()")
        library()
        loader = importlib.machinery.ExtensionFileLoader("nvcr_tokens", str(BINDING))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("nvcr_tokens", loader))
        loader.exec_module(module)
        module.bind(_refuse, _check)
        _module = module
    return _module


def _stream(stream) -> int | None:
    return None if stream is None else _stream_handle(stream) or 0


def _on(stream, device: torch.device):
    """torch's own operations on a stream given as the operators take one (None: the current stream)."""
    if stream is None:
        return contextlib.nullcontext()
    if isinstance(stream, torch.cuda.Stream):
        return torch.cuda.stream(stream)
    handle = _stream(stream)
    return torch.cuda.stream(torch.cuda.ExternalStream(handle, device) if handle else torch.cuda.default_stream(device))


def _whole(tensor: torch.Tensor, name: str, kind: torch.dtype, shape: tuple, index: int) -> int:
    """The address of a contiguous tensor of a type and shape on CUDA device `index`."""
    if tensor.dtype is not kind or tensor.shape != shape or tensor.get_device() != index or not tensor.is_contiguous():
        _refuse(f"{name} must be a contiguous {kind} tensor of shape {tuple(shape)} on cuda:{index}")
    return tensor.data_ptr()


def block_norm(block: torch.Tensor, *, residual: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               post: bool = False, post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
               pre_weight: torch.Tensor | None = None, pre_bias: torch.Tensor | None = None, kind: str = "rms",
               residual_scale: float = 1.0, weight_offset: float = 0.0, epsilon: float = 1e-6,
               hidden: bool = True, normed: bool = True, stream=None):
    """``(hidden, normed)`` of a block's output [rows, width] (float16, bfloat16 or float32):

    p = N(block; post_weight, post_bias) if `post` else block;  hidden = residual_scale * residual + gate * p;
    normed = N(hidden; pre_weight, pre_bias). N is the root-mean-square norm ("rms") or the layer norm ("layer"),
    with weights taken as weight + weight_offset. `gate` is [width] or [rows, width]. block, residual and a gate of
    rows may have any row stride. ``hidden=False`` or ``normed=False`` leaves that output out (None)."""
    layer = _KINDS.get(kind)
    if layer is None:
        _refuse(f"kind must be one of {sorted(_KINDS)}")
    return (_module or _native()).norm(block, residual, gate, post, post_weight, post_bias, pre_weight, pre_bias, layer,
                                       residual_scale, weight_offset, epsilon, hidden, normed,
                                       None if stream is None else _stream(stream))


class PagedCache:
    """A paged cache of keys and values in 4 bits, over the caller's tensors:
    codes uint8 [pages, kv_heads, page_size, head_dim / 2] and scales float16
    [pages, kv_heads, page_size, head_dim / group, 2] (scale, minimum), for
    keys and for values. Slot p * page_size + i is place i of page p."""

    def __init__(self, key_codes: torch.Tensor, key_scales: torch.Tensor, value_codes: torch.Tensor,
                 value_scales: torch.Tensor) -> None:
        _require(key_codes.dim() == 4 and key_scales.dim() == 5, "codes have 4 dimensions and scales 5")
        _require(key_codes.is_cuda, "a cache is on a CUDA device")
        pages, kv_heads, page_size, half = key_codes.shape
        groups = key_scales.shape[3]
        _require(groups > 0 and (2 * half) % groups == 0, "scales hold a whole number of groups")
        device, index = key_codes.device, key_codes.get_device()
        code_shape, scale_shape = (pages, kv_heads, page_size, half), (pages, kv_heads, page_size, groups, 2)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.tensors = (key_codes, key_scales, value_codes, value_scales)
        self._struct = _Cache(_whole(key_codes, "key_codes", torch.uint8, code_shape, index),
                              _whole(key_scales, "key_scales", torch.float16, scale_shape, index),
                              _whole(value_codes, "value_codes", torch.uint8, code_shape, index),
                              _whole(value_scales, "value_scales", torch.float16, scale_shape, index),
                              self.status.data_ptr(), pages, kv_heads, page_size, 2 * half, 2 * half // groups)
        self._address = ctypes.addressof(self._struct)
        self.device, self.pages, self.kv_heads, self.page_size = device, pages, kv_heads, page_size
        self.head_dim, self.group, self._index = 2 * half, 2 * half // groups, index

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, group: int = 64,
              device: str | torch.device = "cuda") -> "PagedCache":
        """A cache of zeros."""
        _require(head_dim > 0 and group > 0 and head_dim % group == 0 and head_dim % 2 == 0,
                 "head_dim must be even and a multiple of group")
        place = (pages, kv_heads, page_size)
        codes = [torch.zeros(place + (head_dim // 2,), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(place + (head_dim // group, 2), dtype=torch.float16, device=device) for _ in range(2)]
        return cls(codes[0], scales[0], codes[1], scales[1])

    def append(self, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor, *,
               queries: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               cosines: torch.Tensor | None = None, sines: torch.Tensor | None = None, interleaved: bool = False,
               stream=None) -> torch.Tensor | None:
        """Stores keys and values [tokens, kv_heads, head_dim] (float16 or bfloat16) at int64 `slots` (negative: not
        stored; else distinct). With int32 `positions`, keys are rotated before they are stored, and `queries`
        [tokens, heads, head_dim] into the tensor that is returned, by rows of the float32 tables `cosines` and
        `sines` [rows, rotary / 2]: pairs (i, i + rotary / 2), or (2 i, 2 i + 1) if `interleaved`."""
        return (_module or _native()).append(self._address, self._index, keys, values, slots, queries, positions, cosines,
                                             sines, interleaved, None if stream is None else _stream(stream))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [n, kv_heads, head_dim] that the codes at int64 `slots` stand for (zeros outside)."""
        code = _TYPES.get(dtype)
        if code is None:
            _refuse("dtype is a float type")
        return (_module or _native()).read(self._address, self._index, slots, code,
                                           None if stream is None else _stream(stream))

    def check(self) -> None:
        """Waits for all streams of the device and raises if a kernel met a slot, position, page number, length or
        offset out of range since the last check (the token, page or sequence was left out)."""
        torch.cuda.synchronize(self.device)
        found = int(self.status.item())
        if found:
            self.status.bitwise_and_(~found)  # not the bits of calls that another thread makes meanwhile
            torch.cuda.current_stream(self.device).synchronize()  # before any stream's next call
            names = [name for bit, name in ((1, "slot"), (2, "position"), (4, "page number"), (8, "length or offset"))
                     if found & bit]
            _refuse(f"out of range on the device: {', '.join(names)}")


class TokenContext:
    """Working memory of attention on the current device; calls that share one, replays of graphs that captured one among
    them, belong on one stream. Make it before a capture; closing it waits for nothing, at any time."""

    def __init__(self) -> None:
        handle = ctypes.c_void_p()
        _check(library().nvcr_sm100_token_context_create(ctypes.byref(handle)))
        self._handle = handle

    def close(self) -> None:
        if self._handle:
            library().nvcr_sm100_token_context_destroy(self._handle)
            self._handle = ctypes.c_void_p()

    def __enter__(self) -> "TokenContext":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:
            pass

    def attend(self, queries: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
               max_length: int, query_offsets: torch.Tensor | None = None, max_queries: int = 1,
               scale: float | None = None, stream=None) -> torch.Tensor:
        """Attention of queries [tokens, heads, head_dim] over the cache, the new tokens' own keys and values already
        appended. int32 `lengths` [batch] (at most `max_length`) count the new tokens; sequence b's pages are row b
        of the int32 `page_table`; its new tokens are query_offsets[b] .. query_offsets[b + 1] - 1 (int32 [batch + 1],
        at most `max_queries` each; None: token b). A token sees the places up to its own; one that sees none, or is
        in no sequence, or in one whose length or offsets are out of range, gives zeros. `scale` defaults to
        1 / sqrt(head_dim)."""
        return (_module or _native()).attend(self._handle.value or 0, cache._address, cache._index, queries, page_table, lengths,
                                             query_offsets, max_queries, max_length, scale,
                                             None if stream is None else _stream(stream))


class PackedMatrix:
    """A 4-bit weight matrix [outputs, inputs] with group scales, laid out once:
    codes uint8 [outputs, inputs / 2], scales and minimums float16 [outputs, inputs / group]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, minimums: torch.Tensor, stream=None) -> None:
        _require(codes.dim() == 2 and scales.dim() == 2, "codes and scales have two dimensions")
        _require(codes.is_cuda, "weights are on a CUDA device")
        outputs, inputs, groups = codes.shape[0], 2 * codes.shape[1], scales.shape[1]
        _require(groups > 0 and inputs % groups == 0, "scales hold a whole number of groups")
        device, index, group = codes.device, codes.get_device(), inputs // groups
        (_module or _native()).on_current(index)
        addresses = (_whole(codes, "codes", torch.uint8, (outputs, inputs // 2), index),
                     _whole(scales, "scales", torch.float16, (outputs, groups), index),
                     _whole(minimums, "minimums", torch.float16, (outputs, groups), index))
        code_bytes, scale_bytes = ctypes.c_size_t(0), ctypes.c_size_t(0)
        _check(library().nvcr_sm100_token_packed_bytes(outputs, inputs, group, ctypes.byref(code_bytes),
                                                       ctypes.byref(scale_bytes)))
        self.outputs, self.inputs, self.group, self.device, self._index = outputs, inputs, group, device, index
        self.codes = torch.empty(code_bytes.value, dtype=torch.uint8, device=device)
        self.scales = torch.empty(scale_bytes.value, dtype=torch.uint8, device=device)
        self._addresses = (self.codes.data_ptr(), self.scales.data_ptr())
        handle = torch.cuda.current_stream(index).cuda_stream if stream is None else _stream(stream)
        _check(library().nvcr_sm100_token_pack(*addresses, outputs, inputs, group, *self._addresses, handle))

    @classmethod
    def quantise(cls, weights: torch.Tensor, group: int = 64, stream=None) -> "PackedMatrix":
        """From a float matrix [outputs, inputs], each group by its own range, as `PagedCache.append` stores one:
        m = fp16(min), s = fp16((max - min) * (1 / 15)), or 2^-24 where that is 0 and the range is not, and
        c = clamp(rint((x - m) / s), 0, 15), from FP32."""
        _require(weights.dim() == 2 and group > 0 and weights.shape[1] % group == 0,
                 "weights have two dimensions and inputs are a multiple of group")
        _require(weights.is_cuda, "weights are on a CUDA device")
        # all of it on one stream, whose allocator takes the codes back when this returns
        with _on(stream, weights.device):
            parts = weights.float().unflatten(1, (-1, group))
            low, high = parts.amin(-1), parts.amax(-1)
            fifteenth = torch.tensor(1.0 / 15.0, dtype=torch.float32, device="cpu")  # no copy, and a product in FP32
            minimums, scales = low.half(), ((high - low) * fifteenth).half()
            scales = torch.where((scales == 0) & (high > low), 2.0 ** -24, scales)
            steps = scales.float().unsqueeze(-1)
            codes = torch.where(steps > 0, torch.round((parts - minimums.float().unsqueeze(-1)) / steps), 0.0)
            codes = codes.clamp(0, 15).to(torch.uint8).flatten(1)
            codes = codes[:, 0::2] | codes[:, 1::2] << 4
        return cls(codes, scales, minimums, stream)

    def multiply(self, x: torch.Tensor, bias: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """x [rows, inputs] (float16 or bfloat16, any row stride) times the matrix's transpose, plus bias [outputs]."""
        return (_module or _native()).multiply(*self._addresses, self.outputs, self.inputs, self.group, self._index, x, bias,
                                               None if stream is None else _stream(stream))
