"""Selections from rows of logits: the top logits of a teacher's row, which ``linear_distillation`` learns from, and tokens drawn
from a model's rows.  (No counterpart in the reference.)

Both go by one order of a row: value descending, equal values by column.  Neither is differentiable.
"""
from __future__ import annotations

import ctypes
import numbers
from typing import Optional

import torch

from . import _lib
from .ops import _on_device, _ptr, _stream


def _rows_of(logits, what):
    if not logits.is_cuda:
        raise RuntimeError(f"{what} needs its tensors on an AMD GPU (device type 'cuda' under ROCm); there is no CPU path")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must have shape (..., V) with V >= 1, got {tuple(logits.shape)}")
    _lib.dtype_code(logits.dtype)
    rows = logits.detach().reshape(-1, logits.shape[-1])
    return rows if rows.stride(1) == 1 or rows.shape[1] == 1 else rows.contiguous()


@torch.library.custom_op("lce_amd::top_logits", mutates_args=(), device_types="cuda")
def _op_top_logits(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _top_logits(logits, k)


@_op_top_logits.register_fake
def _(logits, k):
    shape = logits.shape[:-1]
    return (logits.new_empty((*shape, k)), logits.new_empty((*shape, k), dtype=torch.int64),
            logits.new_empty(shape, dtype=torch.float32))


def _here(t):
    """Whether t lies on the current device (whose calls the host extension, csrc/lce_host.cpp, takes)."""
    return t.is_cuda and t.device.index == torch._C._cuda_getDevice()


def _top_logits(logits, k):
    if _here(logits):
        done = _lib.host().top_logits(logits, k, _stream(logits.device))
        if done is not None and len(done) == 2:
            _lib.raise_for_status(*done)
        if done is not None:
            return done
    rows = _rows_of(logits, "top_logits")
    N, V = rows.shape
    shape, dev = logits.shape[:-1], rows.device
    values = torch.empty((*shape, k), dtype=rows.dtype, device=dev)
    index = torch.empty((*shape, k), dtype=torch.int64, device=dev)
    lse = torch.empty(shape, dtype=torch.float32, device=dev)
    with _on_device(dev):
        rc = _lib.load().lce_top_logits(_ptr(rows), _lib.dtype_code(rows.dtype), N, V, rows.stride(0), k, _ptr(values), _ptr(index),
                                        _ptr(lse), _stream(dev))
    _lib.raise_for_status(rc, "top_logits")
    return values, index, lse


def top_logits(logits, k: int):
    """The ``k`` largest logits of each row, in order, with their columns and the row's logsumexp.

    Args:
        logits: (..., V) bfloat16, float16 or float32, any row stride.
        k: a whole number, 1 <= k <= min(V, 1024).

    Returns ``(values, index, lse)``: (..., k) in the logits' type, (..., k) torch.long and (...) float32.  Equal logits come by
    column, NaN before all; ``values - lse[..., None]`` are log-probabilities.  ``index`` and ``values`` are what
    ``linear_distillation`` takes; a column of -inf (masked) that gets among the k is no target there.
    """
    if logits.dim() < 1 or not 1 <= k <= min(logits.shape[-1], _lib.MAX_TARGETS) or k != int(k):
        raise ValueError(f"top_logits: k must be in 1 ... min(V, {_lib.MAX_TARGETS}), got {k} for logits of shape {tuple(logits.shape)}")
    k = int(k)
    if torch.compiler.is_compiling():
        return _op_top_logits(logits.detach(), k)
    return _top_logits(logits, k)


# What a setting may be once it has been rounded to float32 (top_k: a whole number): as the definition and lce.h have it.
_FINE = {
    "temperature": lambda v: -_lib.F32_ZERO <= v < _lib.F32_INF,
    "top_k": lambda v: 0 <= v < 2 ** 63 and v == int(v),
    "top_p": lambda v: _lib.F32_ZERO < v <= 1.0 + 2.0 ** -24,
    "min_p": lambda v: -_lib.F32_ZERO <= v <= 1.0 + 2.0 ** -24,
}


def _check_numbers(temperature, top_k, top_p, min_p):
    for value, name in ((temperature, "temperature"), (top_k, "top_k"), (top_p, "top_p"), (min_p, "min_p")):
        if isinstance(value, torch.Tensor):
            continue
        if not (isinstance(value, (int, float)) or isinstance(value, numbers.Real)):
            raise ValueError(f"sample_logits: {name} must be a number or a tensor, got {type(value).__name__}")
        if not _FINE[name](value):
            raise ValueError(f"sample_logits: {name} = {value} is out of range")


def _number_or_rows(value, name, shape, device, dtype):
    """(number, None), or (a number that is not looked at, a tensor with one entry a row)."""
    if isinstance(value, torch.Tensor):
        if value.device != device:
            raise ValueError(f"sample_logits: {name} is on {value.device}, the logits on {device}")
        if value.shape != shape and value.dim() != 0:
            raise ValueError(f"sample_logits: {name} has shape {tuple(value.shape)}, the rows {tuple(shape)}")
        if value.is_floating_point() != dtype.is_floating_point or value.is_complex():
            raise ValueError(f"sample_logits: {name} cannot be {value.dtype}")
        return 1, value.detach().to(dtype).expand(shape).contiguous()
    return float(value) if dtype.is_floating_point else int(value), None


# (A tensor in the place of a number: settings by row.  What is a number stays one, so that the library chooses its kernel by it.)
@torch.library.custom_op("lce_amd::sample_logits", mutates_args=(), device_types="cuda")
def _op_sample_logits(logits: torch.Tensor, u: torch.Tensor, temperature_rows: Optional[torch.Tensor] = None,
                      top_k_rows: Optional[torch.Tensor] = None, top_p_rows: Optional[torch.Tensor] = None,
                      min_p_rows: Optional[torch.Tensor] = None, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                      min_p: float = 0.0) -> torch.Tensor:
    return _sample_logits(logits, u, temperature if temperature_rows is None else temperature_rows, top_k if top_k_rows is None else top_k_rows,
                          top_p if top_p_rows is None else top_p_rows, min_p if min_p_rows is None else min_p_rows)


@_op_sample_logits.register_fake
def _(logits, u, temperature_rows=None, top_k_rows=None, top_p_rows=None, min_p_rows=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return logits.new_empty(logits.shape[:-1], dtype=torch.int64)


def _sample_logits(logits, u, temperature, top_k, top_p, min_p):
    if isinstance(u, torch.Tensor) and _here(logits):
        tokens = _lib.host().sample_logits(logits, u, temperature, top_k, top_p, min_p, _stream(logits.device))
        if tokens is not None:
            return tokens
    _check_numbers(temperature, top_k, top_p, min_p)
    rows = _rows_of(logits, "sample_logits")
    N, V = rows.shape
    shape, dev = logits.shape[:-1], rows.device
    if not isinstance(u, torch.Tensor) or u.dtype != torch.float32 or u.shape != shape or u.device != dev:
        raise ValueError("sample_logits: u must be a float32 tensor with one number for each row, on the logits' device")
    u = u.detach().contiguous()
    t, t_rows = _number_or_rows(temperature, "temperature", shape, dev, torch.float32)
    k, k_rows = _number_or_rows(top_k, "top_k", shape, dev, torch.int64)
    p, p_rows = _number_or_rows(top_p, "top_p", shape, dev, torch.float32)
    m, m_rows = _number_or_rows(min_p, "min_p", shape, dev, torch.float32)
    s = _lib.LceSampling(t, p, m, k, _ptr(t_rows), _ptr(p_rows), _ptr(m_rows), _ptr(k_rows))
    tokens = torch.empty(shape, dtype=torch.int64, device=dev)
    with _on_device(dev):
        rc = _lib.load().lce_sample(_ptr(rows), _lib.dtype_code(rows.dtype), N, V, rows.stride(0), _ptr(u), ctypes.byref(s), _ptr(tokens),
                                    _stream(dev))
    _lib.raise_for_status(rc, "sample_logits")
    return tokens


def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for each row of logits, from given random numbers.

    With ``w = exp((z - max z) / temperature)``, in the row's order: ``top_k`` keeps the first k columns, ``top_p`` those
    before which less than ``top_p`` of the weight that ``top_k`` left has gathered, ``min_p`` those of at least ``min_p`` times
    the largest weight -- each the first column at least.  The token is the first column, of what all keep, with which more than
    ``u`` times the whole weight has gathered.  Weights are whole multiples of ``2 ** -min(50, 62 - ceil(log2(V)))``, summed in 64 bits: the
    token does not depend on how many rows there are.

    Args:
        logits: (..., V) bfloat16, float16 or float32, any row stride; -inf masks a column.
        u: (...) float32 in [0, 1), e.g. ``torch.rand``: the same numbers draw the same tokens.
        temperature: positive, or 0 for the first column of the order (the largest logit).
        top_k: 0 keeps all.  top_p: 1 keeps all.  min_p: 0 keeps all.

    Each setting is a number (rounded to float32; a whole one for top_k), or a tensor (...) on the logits' device with one for every row
    (in which, without a check, top_k <= 0, top_p >= 1 and min_p <= 0 keep all, top_p <= 0 and min_p > 1 keep one column and a temperature
    that is not positive stands for 0).
    Returns torch.long tokens (...); -1 for a row that is masked altogether or has a NaN.
    """
    if torch.compiler.is_compiling():
        _check_numbers(temperature, top_k, top_p, min_p)
        settings = (temperature, top_k, top_p, min_p)
        rows = [v.detach() if isinstance(v, torch.Tensor) else None for v in settings]
        t, k, p, m = (default if isinstance(v, torch.Tensor) else v for v, default in zip(settings, (1.0, 0, 1.0, 0.0)))
        return _op_sample_logits(logits.detach(), u, *rows, float(t), int(k), float(p), float(m))
    return _sample_logits(logits, u, temperature, top_k, top_p, min_p)
