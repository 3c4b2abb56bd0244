"""The operators of an 8-bit decoder layer on torch tensors: ``quantize_rows``, ``matmul_scaled``, ``QuantizedLinear`` and the
paged int8 cache (``PagedCache``, ``PagedBatch``) with its attention.

Thin calls of the direct entry points in include/mlel_b200.h (``mlel_cuda_quantize_rows`` and the following), which say what
each computes.  Work is enqueued on torch's current stream of the tensors' device; nothing waits.  Every call may be captured
into a CUDA graph.  What the library refuses raises ``MlelError``.  They are for inference: results carry no gradients.

A decode step's kernels take a few microseconds each, so the way to them is kept short: objects that a program keeps
(weights, a cache, a batch) hold their descriptions ready, a call describes its own tensors and enters the library once.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import BF16, ERROR_DEVICE, F16, F32, I8, I32, MlelError, check, lib
from .runtime import _current_stream

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int8: I8, torch.int32: I32}
_TENSOR = struct.Struct("=Qii6q6q").pack  # mlel_tensor: address, type, rank, sizes, strides in bytes
_PADDED = [(0,) * (6 - rank) for rank in range(7)]
_SIX = (0,) * 6

_P, _I, _F, _U64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_uint64
_SIGNATURES = {
    "mlel_cuda_quantize_rows": (_P,) * 4,
    "mlel_cuda_matmul_scaled": (_P,) * 7,
    "mlel_cuda_quantized_linear": (_P,) * 6 + (_U64, _P),
    "mlel_cuda_paged_append": (_P,) * 8 + (_I, _P),
    "mlel_cuda_paged_attention": (_P,) * 4 + (_F, _I, _I, _F, _P, _U64, _P),
    "mlel_paged_attention_workspace": (_P,) * 4,
}


class _Entries:
    """The entry points, in function objects of this module's own, made when first used."""

    def __getattr__(self, name):
        fn = lib()[name]
        fn.argtypes, fn.restype = _SIGNATURES[name], ctypes.c_int
        setattr(self, name, fn)
        return fn


_entries = _Entries()


def _pack(t: torch.Tensor) -> bytes:
    """``t`` as an mlel_tensor."""
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"tensors of {t.dtype} are not taken")
    shape = t.shape
    rank = len(shape)
    if rank > 6:
        raise ValueError("tensors of more than 6 axes are not taken")
    if t.is_contiguous():
        return _TENSOR(t.data_ptr(), code, rank, *shape, *_PADDED[rank], *_SIX)
    size = t.element_size()
    strides = [size * n for n in t.stride()]
    if strides[0] == 0:  # a stride of 0 there stands for a packed tensor
        if shape[0] > 1:
            raise ValueError("a tensor that repeats along its first axis is not taken")
        strides[0] = size * max(1, t.numel())
    return _TENSOR(t.data_ptr(), code, rank, *shape, *_PADDED[rank], *strides, *_PADDED[rank])


def _device(first: torch.Tensor, *others) -> int:
    """The one CUDA device of all tensors (None among them are passed over)."""
    index = first.get_device()
    if index < 0:
        raise ValueError("tensors have to be on a CUDA device: there is no CPU implementation to fall back to")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors of one call have to be on one device")
    return index


def _enter(index: int, entry, *arguments) -> None:
    """``entry(*arguments, stream)`` with ``index`` as the current device and torch's stream of it."""
    before = torch.cuda.current_device()
    if before == index:
        status = entry(*arguments, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = entry(*arguments, _current_stream(index))
    if status != 0:
        check(status)


def quantize_rows(x: torch.Tensor, out: torch.Tensor | None = None, scales: torch.Tensor | None = None):
    """``(q, scales)``: the rows of ``x`` [..., K] (f32, f16 or bf16) in 8 bits with an f32 scale for each: ``scales = max|x| / 127``,
    ``q = round(x / scales)``.  ``out`` and ``scales`` are written where they are given ([M, K] int8 and [M], for M rows in all).  A new
    ``q`` is packed: where K is no multiple of 16 and a product follows, give an ``out`` whose rows lie on 16-byte boundaries."""
    index = _device(x, out, scales)
    shape = x.shape
    if len(shape) < 1:
        raise ValueError("x needs an axis")
    rows = x if len(shape) == 2 else x.reshape(-1, shape[-1])
    q = rows.new_empty(rows.shape, dtype=torch.int8) if out is None else out
    s = rows.new_empty(rows.shape[0], dtype=torch.float32) if scales is None else scales
    _enter(index, _entries.mlel_cuda_quantize_rows, _pack(rows), _pack(q), _pack(s))
    if len(shape) != 2:
        return (q if out is not None else q.view(shape)), (s if scales is not None else s.view(shape[:-1]))
    return q, s


def matmul_scaled(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, bias: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a @ b.T) * a_scales[:, None] * b_scales + bias`` for int8 ``a`` [M, K] (tokens) and ``b`` [N, K] (weights, a row per
    output channel), scales and bias in f32: the sums are exact, the result is rounded once to ``dtype`` (or ``out``'s type).  Tensor
    cores want the rows of both on 16-byte boundaries, as ``QuantizedLinear`` lays them out; packed rows of a K that is no multiple of
    16 go a far slower way."""
    index = _device(a, a_scales, b, b_scales, bias, out)
    if out is None:
        out = a.new_empty((a.shape[0], b.shape[0]), dtype=dtype)
    _enter(index, _entries.mlel_cuda_matmul_scaled, _pack(a), _pack(a_scales), _pack(b), _pack(b_scales),
           None if bias is None else _pack(bias), _pack(out))
    return out


class _Described:
    """What is described to the library once: an attribute that has been set is not set again (a new tensor is a new object)."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError(f"{name} is described to the library already: make a new {type(self).__name__}")
        super().__setattr__(name, value)


class QuantizedLinear(_Described):
    """A projection in 8 bits: ``linear(x)`` quantises the rows of ``x`` [..., K] and multiplies them with int8 ``weight`` [N, K],
    one f32 scale per output channel, optional f32 bias; the result has ``x``'s type.  The weights are laid out once: rows on
    16-byte boundaries, copied where they are not there already.  Calls use ``linear.weight``, ``scales`` and ``bias``, whose values may
    change between them; the attributes themselves stay."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None):
        for name, t, dtype in (("weight", weight, torch.int8), ("scales", scales, torch.float32), ("bias", bias, torch.float32)):
            if t is not None and t.dtype != dtype:  # (laying the rows out would convert them in silence)
                raise TypeError(f"{name} has to be {dtype}, not {t.dtype}")
        self.device = _device(weight, scales, bias)
        n, k = weight.shape
        self._padded = (k + 15) // 16 * 16
        if weight.stride(1) != 1 or weight.stride(0) % 16 != 0 or weight.data_ptr() % 16 != 0:
            rows = torch.zeros(n, self._padded, dtype=torch.int8, device=weight.device)
            rows[:, :k] = weight
            weight = rows[:, :k]
        self.weight, self.scales, self.bias = weight, scales.contiguous(), None if bias is None else bias.contiguous()
        self.in_features, self.out_features = k, n
        self._packed = _pack(self.weight), _pack(self.scales), None if bias is None else _pack(self.bias)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        if shape[-1] != self.in_features:
            raise ValueError(f"x has {shape[-1]} features, not {self.in_features}")
        if x.get_device() != self.device:
            raise ValueError("x has to be on the weights' device")
        rows = x if len(shape) == 2 else x.reshape(-1, shape[-1])
        m = rows.shape[0]
        y = x.new_empty((m, self.out_features))
        need = m * (self._padded + 4)
        space = x.new_empty(need, dtype=torch.int8)
        weight, scales, bias = self._packed
        _enter(self.device, _entries.mlel_cuda_quantized_linear, _pack(rows), weight, scales, bias, _pack(y), space.data_ptr(), need)
        return y if len(shape) == 2 else y.view(*shape[:-1], self.out_features)


class PagedBatch(_Described):
    """The sequences of one call: new tokens of sequence b are rows ``starts[b]`` to ``starts[b + 1] - 1`` of the token axis and the last
    of its ``lengths[b]`` tokens; token t lies in page ``page_table[b, t // page]``.  All int32 on the device, read when the kernels
    run (a decode loop or a captured graph changes their values in place); ``max_new`` and ``max_length`` are bounds that the host knows."""

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor, max_new: int, max_length: int):
        self.device = _device(starts, lengths, page_table)
        self.starts, self.lengths, self.page_table = starts, lengths, page_table
        self.max_new, self.max_length = int(max_new), int(max_length)
        self._packed = _pack(starts) + _pack(lengths) + _pack(page_table) + struct.pack("=ii", self.max_new, self.max_length)
        self._space = {}  # bytes of workspace by the sizes that decide them


class PagedCache(_Described):
    """Keys and values of a layer, int8 with a scale for each page and head.  ``data`` [2, pages, heads, page, head_dim] and
    ``scales`` f32 [2, pages, heads]: keys first, then values."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        if data.dim() != 5 or data.shape[0] != 2 or scales.shape != data.shape[:3]:
            raise ValueError("data has to be [2, pages, heads, page, head_dim] and scales [2, pages, heads]")
        self.device = _device(data, scales)
        self.data, self.scales = data, scales
        self._packed = _pack(data[0]) + _pack(data[1]) + _pack(scales[0]) + _pack(scales[1])
        self._sizes = tuple(data.shape[2:])

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, head_dim: int, device="cuda") -> "PagedCache":
        return cls(torch.zeros(2, pages, heads, page, head_dim, dtype=torch.int8, device=device),
                   torch.zeros(2, pages, heads, dtype=torch.float32, device=device))

    def append(self, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None, batch: PagedBatch,
               q: torch.Tensor | None = None, q_out: torch.Tensor | None = None, interleaved: bool = False):
        """Writes new keys and values [tokens, heads, head_dim] into the cache, the keys rotated by their positions; ``cos`` and ``sin``
        are [positions, rotated / 2], or None for no rotation.  Returns the rotated queries where ``q`` is given (``q_out``, which may
        be ``q`` itself, or a new tensor, in which rows of no sequence are undefined)."""
        if _device(k, v, cos, sin, q, q_out) != self.device or batch.device != self.device:
            raise ValueError("tensors have to be on the cache's device")
        if q is not None and q_out is None:
            q_out = q.new_empty(q.shape)
        _enter(self.device, _entries.mlel_cuda_paged_append, self._packed, batch._packed, _pack(k), _pack(v),
               None if cos is None else _pack(cos), None if sin is None else _pack(sin), None if q is None else _pack(q),
               None if q_out is None else _pack(q_out), 1 if interleaved else 0)
        return q_out

    def attend(self, q: torch.Tensor, batch: PagedBatch, out: torch.Tensor | None = None, scale: float | None = None, causal: bool = True,
               window: int = 0, softcap: float = 0.0) -> torch.Tensor:
        """Attention of the new tokens' queries [tokens, query_heads, head_dim] over the cache, which holds the new tokens already.
        ``scale`` defaults to head_dim ** -0.5; a ``window`` of 0 is none, and one as long as the sequence hides nothing; rows of no sequence are left as they are in ``out``, undefined in a new tensor."""
        if _device(q, out) != self.device or batch.device != self.device:
            raise ValueError("tensors have to be on the cache's device")
        if out is None:
            out = q.new_empty(q.shape)
        packed = _pack(q)
        sizes = (q.shape, self._sizes)
        need = batch._space.get(sizes)
        if need is None:
            value = ctypes.c_uint64()
            check(_entries.mlel_paged_attention_workspace(self._packed, batch._packed, packed, ctypes.addressof(value)))
            need = batch._space[sizes] = value.value
        space = q.new_empty(need, dtype=torch.int8) if need else None
        _enter(self.device, _entries.mlel_cuda_paged_attention, self._packed, batch._packed, packed, _pack(out),
               q.shape[-1] ** -0.5 if scale is None else scale, 1 if causal else 0, max(-1, min(window, 0x7fffffff)), softcap,
               None if space is None else space.data_ptr(), need)
        return out


def paged_error(device: int | None = None) -> int:
    """0, or what the cache's kernels left out on the device since the last call: 1 a sequence whose numbers contradict the batch's
    bounds, 2 a page outside the cache.  Waits for the device and clears the record.  Raises ``MlelError`` where the device cannot be
    read, and where a kernel gave up on a wait (its results are not complete)."""
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        code = lib().mlel_paged_error()
        if code < 0:
            check(code)
        wait = lib().mlel_device_error()
    if wait != 0:
        raise MlelError(ERROR_DEVICE, f"a kernel gave up on a wait that ran out (code {wait})")
    return code
