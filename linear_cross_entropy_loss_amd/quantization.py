"""An output layer in 8 bits: the logits that ``sample_logits`` and ``top_logits`` read, from a copy of the weight of a byte per number.

A row is quantised to whole numbers of -127 ... 127 with one scale: hidden states by token, within the call, a weight by column of the
vocabulary, once for as long as it stays the same.  The products are summed in whole numbers, exactly.  (No counterpart in the
reference.)  Not differentiable.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib, ops
from .ops import _on_device, _ptr, _stream


class Quantized(NamedTuple):
    """``values`` (..., H) int8, their last dimension dense and rows on 16-byte boundaries, and ``scales`` (...) float32: what the
    numbers stand for is ``values * scales[..., None]``."""

    values: torch.Tensor
    scales: torch.Tensor


def _check(t, what, depth):
    if not t.is_cuda:
        raise RuntimeError(f"{what} needs its tensors on an AMD GPU (device type 'cuda' under ROCm); there is no CPU path")
    _lib.dtype_code(t.dtype)
    if not 1 <= depth <= _lib.INT8_DEPTH:
        raise ValueError(f"{what}: 1 to {_lib.INT8_DEPTH} numbers share a scale, got {depth}")


def _row_bytes(depth):
    """Row stride of numbers that are laid out here: whole cache lines, but for short rows."""
    m = 128 if depth >= 64 else 16
    return -(-depth // m) * m


def _empty(others, depth, device):
    values = torch.empty((others, _row_bytes(depth)), dtype=torch.int8, device=device)
    return values[:, :depth], torch.empty(others, dtype=torch.float32, device=device)


@torch.library.custom_op("lce_amd::quantize_rows", mutates_args=(), device_types="cuda")
def _op_quantize_rows(t: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    depth = t.shape[-1]
    rows = t.detach().reshape(-1, depth)
    if rows.stride(1) != 1 and depth > 1:
        rows = rows.contiguous()
    with _on_device(t.device):
        values, scales = _empty(rows.shape[0], depth, t.device)
        if rows.shape[0]:
            rc = _lib.load().lce_quantize_rows(_ptr(rows), _lib.dtype_code(t.dtype), rows.shape[0], depth, rows.stride(0), _ptr(values),
                                               values.stride(0), _ptr(scales), _stream(t.device))
            _lib.raise_for_status(rc, "quantize_rows")
    return values.view(t.shape), scales.view(t.shape[:-1])


def _strides(shape):
    """Strides of `values` of that shape."""
    s = [1, _row_bytes(shape[-1])]
    for n in reversed(shape[1:-1]):
        s.append(s[-1] * n)
    return s[:len(shape)][::-1]


@_op_quantize_rows.register_fake
def _(t):
    return t.new_empty_strided(t.shape, _strides(t.shape), dtype=torch.int8), t.new_empty(t.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("lce_amd::quantize_columns", mutates_args=(), device_types="cuda")
def _op_quantize_columns(At: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    H, V = At.shape
    with _on_device(At.device):
        values, scales = _empty(V, H, At.device)
        if V:
            rc = _lib.load().lce_quantize_columns(_ptr(At), _lib.dtype_code(At.dtype), H, V, At.stride(0), _ptr(values), values.stride(0),
                                                  _ptr(scales), _stream(At.device))
            _lib.raise_for_status(rc, "quantize_weight")
    return values, scales


@_op_quantize_columns.register_fake
def _(At):
    H, V = At.shape
    return At.new_empty_strided((V, H), _strides((V, H)), dtype=torch.int8), At.new_empty((V,), dtype=torch.float32)


def _quantize(t, columns):
    depth = t.shape[0] if columns else t.shape[-1]
    if not torch.compiler.is_compiling() and t.device.index == torch._C._cuda_getDevice():
        done = _lib.host().quantize(t, columns, _row_bytes(depth), _stream(t.device))
        if done is not None and len(done) == 3:
            _lib.raise_for_status(*done[:2])
        if done is not None:
            return Quantized(*done)
    return Quantized(*(_op_quantize_columns if columns else _op_quantize_rows)(t.detach()))


def quantize_rows(t) -> Quantized:
    """Each row of ``t`` (..., H) in 8 bits: ``scales = max |t| / 127`` over the row, ``values`` the whole numbers nearest to
    ``127 * t / max |t|``, of two the even one.

    ``t``: bfloat16, float16 or float32, H up to 131072, any strides.  A row of zeros has a scale of 0, one with a NaN or an infinity
    a scale of NaN.
    """
    _check(t, "quantize_rows", t.shape[-1] if t.dim() else 0)
    return _quantize(t, False)


def quantize_weight(At) -> Quantized:
    """The weight (H, V) of an output layer in 8 bits, a scale for each of its V columns: ``values`` (V, H), transposed as
    ``quantized_logits`` reads them, and ``scales`` (V).  Any strides: a tied embedding (V, H) is handed over as ``weight.t()``.
    """
    if At.dim() != 2 or At.shape[1] < 1:
        raise ValueError(f"quantize_weight: weight must be 2-D with shape (in_features, out_features), got {tuple(At.shape)}")
    _check(At, "quantize_weight", At.shape[0])
    if At.stride(1) == 1 or At.shape[1] == 1:
        return _quantize(At, True)
    return _quantize(At.t(), False)


@torch.library.custom_op("lce_amd::quantized_logits", mutates_args=(), device_types="cuda")
def _op_quantized_logits(x: torch.Tensor, values: torch.Tensor, scales: torch.Tensor, logit_scale: float, dtype: torch.dtype) -> torch.Tensor:
    H, V, dev = x.shape[-1], values.shape[0], x.device
    rows = x.detach().reshape(-1, H)
    if rows.stride(1) != 1 and H > 1:
        rows = rows.contiguous()
    with _on_device(dev):
        if (values.stride(1) != 1 and H > 1) or values.stride(0) % 16 != 0 or values.data_ptr() % 16 != 0 or not (
                H <= values.stride(0) <= 2 * _lib.INT8_DEPTH):
            ops._warn_copy_once("8-bit weight", values, "rows must be contiguous and start on 16-byte boundaries")
            copy, _ = _empty(V, H, dev)
            values = copy.copy_(values)
        out = torch.empty((*x.shape[:-1], V), dtype=dtype, device=dev)
        N = rows.shape[0]
        b = ctypes.c_size_t(0)
        lib = _lib.load()
        _lib.raise_for_status(lib.lce_int8_logits_workspace_bytes(N, H, V, ctypes.byref(b)), "quantized_logits")
        ws = torch.empty(b.value, dtype=torch.uint8, device=dev)
        rc = lib.lce_int8_logits(_ptr(rows), _lib.dtype_code(x.dtype), N, H, V, rows.stride(0), _ptr(values), values.stride(0), _ptr(scales),
                                 logit_scale, _ptr(out), _lib.dtype_code(dtype), V, _ptr(ws), b.value, _stream(dev))
        _lib.raise_for_status(rc, "quantized_logits")
        del ws
    return out


@_op_quantized_logits.register_fake
def _(x, values, scales, logit_scale, dtype):
    return x.new_empty((*x.shape[:-1], values.shape[0]), dtype=dtype)


def quantized_logits(x, weight: Quantized, logit_scale: float = 1.0, dtype: Optional[torch.dtype] = None):
    """``logit_scale * x @ At`` (..., V) from the 8-bit copy of ``At`` that ``quantize_weight`` gives, the rows of ``x`` quantised alike.

    ``x``: hidden states (..., H), bfloat16, float16 or float32, any strides.  ``dtype``: of the result, any of these; that of x unless
    given.  The sums of products are exact; made float32 and multiplied by the scales there, they are off by at most 2^-21 of themselves
    (where x's scale times ``logit_scale``, and that times the sum, are normal numbers of float32) before they are rounded to ``dtype``.  Rows
    and columns with a NaN or an infinity give NaN.
    """
    values, scales = weight
    if not torch.compiler.is_compiling() and x.is_cuda and x.device.index == torch._C._cuda_getDevice() and (
            _lib.F32_ZERO < logit_scale < _lib.F32_INF) and (dtype is None or isinstance(dtype, torch.dtype)):
        done = _lib.host().quantized_logits(x, values, scales, logit_scale, dtype, _stream(x.device))
        if isinstance(done, torch.Tensor):
            return done
        if done is not None:
            _lib.raise_for_status(*done)
    if x.dim() < 1 or values.dim() != 2 or values.shape[1] != x.shape[-1]:
        raise ValueError(f"quantized_logits: x of shape {tuple(x.shape)} does not go with values of shape {tuple(values.shape)}")
    _check(x, "quantized_logits", x.shape[-1])
    if not (x.device == values.device == scales.device):
        raise ValueError("quantized_logits: x and the weight's values and scales must be on the same device")
    if values.dtype != torch.int8 or scales.dtype != torch.float32 or scales.shape != values.shape[:1] or values.shape[0] < 1:
        raise ValueError("quantized_logits: the weight must be int8 values (V, H) and float32 scales (V), as quantize_weight gives them")
    logit_scale = float(logit_scale)
    if not (_lib.F32_ZERO < logit_scale < _lib.F32_INF):
        raise ValueError(f"logit_scale must be positive and finite in float32, got {logit_scale}")
    dtype = x.dtype if dtype is None else dtype
    _lib.dtype_code(dtype)
    return _op_quantized_logits(x.detach(), values, scales.contiguous(), logit_scale, dtype)
