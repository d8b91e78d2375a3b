"""Microscaled 4-bit floating point: quantisation, and products with weights held in it.

Two formats.  ``"mxfp4"``: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign) under one power of two per 32 consecutive
values of a row.  ``"nvfp4"``: e2m1 values under one e4m3 scale per 16 consecutive values and one fp32 scale per tensor (or
expert).  Rows are stored as checkpoints hold them: two codes to a byte, the even value in the low nibble, and one scale byte
per block.  ``mx4_pack`` lays weights out once for the products; ``mx4_linear`` multiplies a layer, ``mx4_grouped_linear`` one
matrix per expert with ragged numbers of rows.  The operators run on the current stream of their tensors' device, take a
workspace from torch's allocator where they need one, read nothing back and can be captured into a CUDA graph.  They have no
gradients.  No counterpart in the reference, whose formats are the E8 shell and the trellis code.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from . import _lib

_FORMATS = {"mxfp4": _lib.MX4_MXFP4, "nvfp4": _lib.MX4_NVFP4}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_MOST = 2 ** 31 - 1                 # values of a row
_RAN_ON: set = set()                # devices whose status word a product may have set
_DTYPES = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, torch.float32: _lib.DT_F32}


class Mx4Tensor(NamedTuple):
    """Values in 4 bits: ``codes`` uint8 (..., ceil(cols / 2)), ``scales`` uint8 (..., ceil(cols / block)), both dense; for
    "nvfp4" ``tensor_scale``, fp32: one, or one per matrix of a three-dimensional tensor."""
    codes: torch.Tensor
    scales: torch.Tensor
    format: str
    cols: int
    tensor_scale: Optional[torch.Tensor] = None


class Mx4Weight:
    """Weights laid out for the products (``mx4_pack``): (out_features, in_features), or one such matrix per expert.  The
    attributes cannot be set (a new image, or one on another device, is a new weight; ``mx4_pack(..., out=)`` fills the same one)."""
    __slots__ = ("image", "tensor_scale", "format", "experts", "out_features", "in_features", "_desc", "_ref", "_index")

    def __init__(self, image, tensor_scale, format, experts, out_features, in_features):
        desc = _lib.Mx4WeightDesc(image.data_ptr(), tensor_scale.data_ptr() if tensor_scale is not None else 0,
                                  _FORMATS[format], experts or 1, out_features, in_features)
        values = (image, tensor_scale, format, experts, out_features, in_features, desc, C.byref(desc), image.get_device())
        for name, value in zip(self.__slots__, values):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"glq_b200: {name} of a packed weight cannot be set")

    def _holds(self, q: Mx4Tensor) -> bool:
        """Are q's rows of these sizes, format and device?"""
        lead = (self.out_features,) if self.experts is None else (self.experts, self.out_features)
        return (self.format, self.in_features, self._index, lead) == (q.format, q.cols, q.codes.get_device(), tuple(q.codes.shape[:-1]))


def _call(index, what, fn, *args):
    """fn(*args, current stream) with the tensors' device current: its kernels are launched there.  (torch's names are looked up here: a
    build of torch without CUDA has none of them, and imports this module all the same.)"""
    cuda = torch._C
    before = cuda._cuda_getDevice()
    if before == index:
        rc = fn(*args, cuda._cuda_getCurrentRawStream(index))
    else:
        cuda._cuda_setDevice(index)
        try:
            rc = fn(*args, cuda._cuda_getCurrentRawStream(index))
        finally:
            cuda._cuda_setDevice(before)
    if rc:
        _lib.check(rc, what)


def _format(format):
    if format not in _FORMATS:
        raise ValueError(f'glq_b200: format is "mxfp4" or "nvfp4", not {format!r}')
    return _FORMATS[format]


def _cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"glq_b200: {name} must be a CUDA tensor (there is no CPU path)")


def _same_device(t, x, name):
    _cuda(t, name)
    if t.get_device() != x.get_device():
        raise ValueError(f"glq_b200: {name} is on {t.device}, expected {x.device}")


def _dtype(dtype, what):
    d = _DTYPES.get(dtype)
    if d is None:
        raise ValueError(f"glq_b200: {what} is bf16, fp16 or fp32, not {dtype}")
    return d


def _counted(cols):
    if cols > _MOST:
        raise ValueError(f"glq_b200: rows of {cols} values: at most {_MOST} (the C ABI counts them in 32 bits)")


def _scale_ptr(t, x, name, count=1):
    _same_device(t, x, name)
    if t.dtype != torch.float32 or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"glq_b200: {name} must be {count} fp32 value{'s' if count > 1 else ''}, got {tuple(t.shape)} of {t.dtype}")
    return t.data_ptr()


def _new(x, lead, cols, dtype):
    """An empty dense (..., cols) tensor beside x (the two-dimensional case by the call that costs the host least)."""
    if len(lead) == 1:
        return torch.empty_strided((lead[0], cols), (cols, 1), dtype=dtype, device=x.device)
    return x.new_empty(lead + (cols,), dtype=dtype)


def _rows(x, cols):
    """x (..., cols) as rows of consecutive values; rows that overlap (an expanded tensor) are copied."""
    x2 = x if x.dim() == 2 else x.reshape(-1, cols)
    apart, step = x2.stride()
    if (step != 1 and cols > 1) or (apart < cols and x2.shape[0] > 1):
        x2 = x2.contiguous()
    return x2


def mx4_quantize(x, format="mxfp4", tensor_scale=None) -> Mx4Tensor:
    """x (..., cols) of bf16, fp16 or fp32 to 4 bits, each value to the nearest (ties to the even code) of its block's scale.
    "mxfp4": the scale is 2^(floor(log2 amax) - 2), values above six times it saturate.  "nvfp4": the block's scale is the
    e4m3 number nearest to amax / (6 t), with t the one fp32 value ``tensor_scale`` (positive), or, without it,
    max(largest finite |x| * fp32(1 / 2688), 2^-126), found by a first pass.  A block with an infinity or NaN becomes NaN."""
    fmt = _format(format)
    _cuda(x, "x")
    dt = _dtype(x.dtype, "x")
    shape = x.shape
    if not shape:
        raise ValueError("glq_b200: x needs at least one dimension")
    cols, lead, some = shape[-1], shape[:-1], x.numel() > 0
    _counted(cols)
    codes = _new(x, lead, (cols + 1) // 2, torch.uint8)
    scales = _new(x, lead, -(-cols // _BLOCK[format]), torch.uint8)
    given = own = None
    if format == "nvfp4":
        if tensor_scale is None:
            own = x.new_empty((_lib.MX4_SCALE_FLOATS,), dtype=torch.float32)
        else:
            given = _scale_ptr(tensor_scale, x, "tensor_scale")
    elif tensor_scale is not None:
        raise ValueError('glq_b200: "mxfp4" has no tensor_scale')
    if some:
        x2 = _rows(x, cols)
        _call(x.get_device(), "mx4_quantize", _lib.load().glqb_mx4_quantize, x2.data_ptr(), dt, x2.stride(0), x2.shape[0], cols, fmt, given,
              own.data_ptr() if own is not None else None, codes.data_ptr(), scales.data_ptr())
    elif own is not None:
        own.fill_(2.0 ** -126)
    return Mx4Tensor(codes, scales, format, cols, own[:1] if own is not None else tensor_scale)


def _checked(q: Mx4Tensor):
    """(format, rows, values per row, scales of the whole) of an Mx4Tensor."""
    codes, scales, format, cols, t = q
    fmt = _format(format)
    _cuda(codes, "codes")
    _same_device(scales, codes, "scales")
    shape = codes.shape
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not shape:
        raise ValueError("glq_b200: codes and scales are uint8 tensors of stored rows")
    lead = shape[:-1]
    _counted(cols)
    if shape[-1] != (cols + 1) // 2 or scales.shape != lead + (-(-cols // _BLOCK[format]),):
        raise ValueError(f"glq_b200: codes {tuple(shape)} and scales {tuple(scales.shape)} are not {format} rows of {cols} values")
    count = 0
    if format == "nvfp4":
        if t is None:
            raise ValueError('glq_b200: "nvfp4" needs its tensor_scale')
        count = t.numel()
        if count != 1 and not (len(lead) == 2 and count == lead[0]):
            raise ValueError(f"glq_b200: {count} tensor scales for rows of {tuple(lead)}")
        _scale_ptr(t, codes, "tensor_scale", count)
    return fmt, math.prod(lead), cols, count


def mx4_dequantize(q: Mx4Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values (..., cols) an ``Mx4Tensor`` stands for, formed in fp32 and rounded to ``dtype``."""
    fmt, rows, cols, count = _checked(q)
    dt = _dtype(dtype, "dtype")
    codes, sc = q.codes.contiguous(), q.scales.contiguous()
    out = _new(codes, codes.shape[:-1], cols, dtype)
    if rows and cols:
        _call(codes.get_device(), "mx4_dequantize", _lib.load().glqb_mx4_dequantize, codes.data_ptr(), sc.data_ptr(),
              q.tensor_scale.data_ptr() if count else None, rows // (count or 1), rows, cols, fmt, out.data_ptr(), dt)
    return out


def mx4_pack(q: Mx4Tensor, out: Optional[Mx4Weight] = None) -> Mx4Weight:
    """Weights (m, n), or (experts, m, n), laid out for ``mx4_linear`` / ``mx4_grouped_linear``: once, when they are loaded.
    The image has the size of codes and scales, rows rounded up to 128 and values to 256.  ``out``: a packed weight of the same
    sizes, format and device, whose memory takes these weights in place of its own (captured graphs that read it then multiply by
    them); what still reads it on another stream has to be waited for first."""
    fmt, rows, n, scales = _checked(q)
    if q.codes.dim() not in (2, 3):
        raise ValueError(f"glq_b200: weights are (m, n) or (experts, m, n), got codes of {tuple(q.codes.shape)}")
    experts, m = (q.codes.shape[0] if q.codes.dim() == 3 else None), q.codes.shape[-2]
    if rows == 0 or n == 0:
        raise ValueError(f"glq_b200: empty weights, codes of {tuple(q.codes.shape)}")
    if max(m, experts or 1) > _MOST:
        raise ValueError(f"glq_b200: codes of {tuple(q.codes.shape)}: at most {_MOST} rows and experts")
    if out is not None and (out.__class__ is not Mx4Weight or not out._holds(q)):
        raise ValueError(f"glq_b200: out is a packed {q.format} weight of {tuple(q.codes.shape[:-1]) + (n,)} on {q.codes.device}")
    codes, sc = q.codes.contiguous(), q.scales.contiguous()
    lib = _lib.load()
    image = codes.new_empty((lib.glqb_mx4_image_bytes(fmt, experts or 1, m, n),)) if out is None else out.image
    _call(codes.get_device(), "mx4_pack", lib.glqb_mx4_pack, codes.data_ptr(), sc.data_ptr(), fmt, experts or 1, m, n, image.data_ptr())
    t = q.tensor_scale
    if scales:
        t = t.reshape(-1).expand(experts or 1)
        if out is None:
            t = t.clone(memory_format=torch.contiguous_format)
        else:
            with torch.inference_mode():          # (the weight's may have been made under it)
                out.tensor_scale.copy_(t)
    return Mx4Weight(image, t, q.format, experts, m, n) if out is None else out


def _overlap(a, b):
    def span(t):
        first = t.data_ptr()
        return first, first + (sum((d - 1) * s for d, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _input(x, w, quantize_input, input_scale):
    """Checks of x and the weight; (x's type, pointer of its scale)."""
    if w.__class__ is not Mx4Weight:
        raise ValueError("glq_b200: weight is what mx4_pack returns")
    _cuda(x, "x")
    if x.get_device() != w._index:
        raise ValueError(f"glq_b200: x is on {x.device}, the weight on {w.image.device}")
    dt = _dtype(x.dtype, "x")
    if dt == _lib.DT_F32 and not quantize_input:
        raise ValueError("glq_b200: x is bf16 or fp16 (fp32 with quantize_input only)")
    shape = x.shape
    if not shape or shape[-1] != w.in_features:
        raise ValueError(f"glq_b200: x of {tuple(shape)} for a weight of {w.in_features} inputs")
    if input_scale is None:
        return dt, None
    if not quantize_input or w.format != "nvfp4":
        raise ValueError('glq_b200: input_scale belongs to quantize_input with "nvfp4" weights')
    return dt, _scale_ptr(input_scale, x, "input_scale")


def _product(x, dt, w, offsets, quantize_input, xs, y, y_dt, y_stride, accumulate, clear_rest):
    """The call itself: x and y two-dimensional with consecutive values in a row."""
    lib, rows, apart, at = _lib.load(), x.shape[0], x.stride(0), x.data_ptr()
    ws, size = None, 0
    if quantize_input or at & 15 or apart & 7 or w.in_features & 7:
        size = lib.glqb_mx4_workspace_bytes(w._ref, rows, apart, at, quantize_input)
        if size:
            ws = x.new_empty((size,), dtype=torch.uint8)
    _call(w._index, "mx4_product", lib.glqb_mx4_product, w._ref, at, dt, apart, rows, offsets.data_ptr() if offsets is not None else None,
          offsets is not None and offsets.dtype is torch.int64, quantize_input, xs, y.data_ptr(), y_dt, y_stride, accumulate, clear_rest,
          ws.data_ptr() if size else None, size)
    _RAN_ON.add(w._index)


def mx4_linear(x, weight: Mx4Weight, *, quantize_input=False, input_scale=None, out_dtype=None, accumulate_into=None):
    """x (..., n) times a packed (m, n) weight: (..., m), sums in fp32 and one rounding.  x is bf16 or fp16; with
    ``quantize_input`` (then fp32 too) it is brought to the weight's format first, as ``mx4_quantize`` does ("nvfp4": by
    ``input_scale``, one fp32 value, or by the scale of the whole of x), and the tensor cores multiply 4-bit values, at four times
    their 16-bit rate.  ``accumulate_into`` adds the result to that dense (..., m) tensor in place (residual add, before the
    rounding) and returns it."""
    dt, xs = _input(x, weight, quantize_input, input_scale)
    if weight.experts is not None:
        raise ValueError("glq_b200: mx4_linear takes one matrix, not one per expert")
    m, shape = weight.out_features, x.shape
    x2 = _rows(x, weight.in_features)
    rows = x2.shape[0]
    if accumulate_into is None:
        out = _new(x, shape[:-1], m, x.dtype if out_dtype is None else out_dtype)
    else:
        out = accumulate_into
        _same_device(out, x, "accumulate_into")
        if out_dtype not in (None, out.dtype):
            raise ValueError(f"glq_b200: accumulate_into is {out.dtype}, out_dtype {out_dtype}")
        if out.dim() < 1 or out.shape[-1] != m or out.numel() != rows * m or not out.is_contiguous():
            raise RuntimeError("glq_b200: accumulate_into must be a dense (tokens, out_features) tensor")
        if rows and _overlap(x2, out):
            raise ValueError("glq_b200: accumulate_into overlaps x")
    y_dt = _dtype(out.dtype, "the result")
    if rows:
        _product(x2, dt, weight, None, bool(quantize_input), xs, out, y_dt, m, accumulate_into is not None, False)
    return out


def mx4_grouped_linear(x, weight: Mx4Weight, offsets, *, quantize_input=False, input_scale=None, out_dtype=None, out=None):
    """Products grouped by expert: rows offsets[e] .. offsets[e + 1] - 1 of x (rows, n) times matrix e of a packed
    (experts, m, n) weight: (rows, m).  ``offsets``: experts + 1 ascending integers (int32 or int64) on the device, any number of
    rows per expert, none included; nothing is read back.  Rows of no expert (in front of offsets[0], behind offsets[experts])
    are zero in a new result and stay as they are in a given ``out`` (rows, m), whose rows may lie apart.  Offsets outside
    0 .. rows are held to that range, and one that is less than the one before it counts as that one.  At most 1024 experts.
    The other arguments as for ``mx4_linear``; "nvfp4" inputs without ``input_scale`` take the scale of the
    experts' rows (offsets[0] up to the largest offset, held to 0 .. rows)."""
    dt, xs = _input(x, weight, quantize_input, input_scale)
    if weight.experts is None:
        raise ValueError("glq_b200: mx4_grouped_linear takes one matrix per expert")
    if x.dim() != 2:
        raise ValueError(f"glq_b200: x is (rows, n), got {tuple(x.shape)}")
    _same_device(offsets, x, "offsets")
    if offsets.dtype not in (torch.int32, torch.int64) or offsets.shape != (weight.experts + 1,) or not offsets.is_contiguous():
        raise ValueError(f"glq_b200: offsets must be {weight.experts + 1} int32 or int64 values, got {tuple(offsets.shape)} of {offsets.dtype}")
    rows, m = x.shape[0], weight.out_features
    x2 = _rows(x, weight.in_features)
    fresh = out is None
    if fresh:
        out = _new(x, (rows,), m, x.dtype if out_dtype is None else out_dtype)
    else:
        _same_device(out, x, "out")
        if out_dtype not in (None, out.dtype):
            raise ValueError(f"glq_b200: out is {out.dtype}, out_dtype {out_dtype}")
        if out.shape != (rows, m) or (m > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < m):
            raise ValueError(f"glq_b200: out must be ({rows}, {m}) with consecutive values in a row, got {tuple(out.shape)}")
        if rows and _overlap(x2, out):
            raise ValueError("glq_b200: out overlaps x")
    y_dt = _dtype(out.dtype, "the result")
    if rows:
        _product(x2, dt, weight, offsets, bool(quantize_input), xs, out, y_dt, out.stride(0), False, fresh)
    return out


def mx4_check_status() -> None:
    """Synchronise the devices that products ran on and raise RuntimeError (code GLQB_E_DEVICE) if a bounded wait in one of them
    gave up since the last call: the results of that run are invalid."""
    for index in sorted(_RAN_ON):
        _call(index, "mx4 status", lambda stream: _lib.load().glqb_mx4_status(None))
