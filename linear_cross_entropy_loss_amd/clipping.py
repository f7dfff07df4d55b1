"""Clipping of many tensors' gradients by their common norm, on the device and without waiting for it.  (No counterpart in the reference.)"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _on_device, _ptr, _stream


def _dense(t):
    return t.layout == torch.strided and torch.ops.aten.is_non_overlapping_and_dense(t)


def _check(grads, out, max_norm, divisor):
    if not max_norm > _lib.F32_ZERO:
        raise ValueError(f"clip_gradients: max_norm must be positive in float32, got {max_norm}")
    if len(out) != len(grads):
        raise ValueError(f"clip_gradients: {len(grads)} gradients and {len(out)} outputs")
    for g, o in zip(grads, out):
        if not isinstance(g, torch.Tensor) or not isinstance(o, torch.Tensor):
            raise ValueError("clip_gradients: gradients and outputs must be tensors")
        if not g.is_cuda:
            raise RuntimeError("clip_gradients needs its tensors on an AMD GPU (device type 'cuda' under ROCm); there is no CPU path")
        if g.layout != torch.strided or o.layout != torch.strided:
            raise ValueError("clip_gradients: sparse gradients are not supported")
        _lib.dtype_code(g.dtype)
        if o.device != grads[0].device or g.device != grads[0].device:
            raise ValueError("clip_gradients: all tensors must be on the same device")
        if o.shape != g.shape or (o.dtype != g.dtype and o.dtype != torch.float32):
            raise ValueError(f"clip_gradients: a gradient of shape {tuple(g.shape)} and {g.dtype} cannot go to {tuple(o.shape)} and {o.dtype}")
        if o.is_inference() and not torch.is_inference_mode_enabled():
            raise RuntimeError("clip_gradients: tensors of inference mode cannot be changed outside it")
        if g.numel() > 0 and not (g.data_ptr() and o.data_ptr()):
            raise ValueError("clip_gradients: tensors that have no memory of their own (sharded ones, wrappers of others) are not supported: "
                             "hand over what they hold here")
    # (of dense tensors the library looks for shared memory; of others, two that begin with the same number are seen here)
    if len({o.data_ptr() for o in out if o.numel() > 0}) != sum(o.numel() > 0 for o in out):
        raise ValueError("clip_gradients: tensors that are written share memory")
    if isinstance(divisor, torch.Tensor):
        if divisor.dtype != torch.float32 or divisor.numel() != 1 or (grads and divisor.device != grads[0].device):
            raise ValueError("clip_gradients: divisor must be a number, or a float32 tensor with one on the gradients' device")
    elif not _lib.F32_ZERO < divisor < _lib.F32_INF:
        raise ValueError(f"clip_gradients: divisor must be positive and finite in float32, got {divisor}")


def _raise(rc, what):
    _lib.raise_for_status(rc, what + ": tensors that are written share memory, or" if rc == _lib.LCE_EINVAL_ARG else what)


@torch.compiler.disable
@torch.no_grad()
def clip_gradients(grads, max_norm, divisor=1.0, out=None):
    """Scales many tensors, together, to a norm of at most ``max_norm``, and returns the norm that they had: a float32 scalar on
    their device.

    With ``norm = sqrt(sum of all squares) / divisor`` every element becomes ``g * min(1, max_norm / norm) / divisor``.  A norm that
    is not finite (an overflow of float16), or beyond float32, leaves ``min(...)`` at 1: look at the norm before the step is taken.

    Args:
        grads: a tensor or an iterable of them: bfloat16, float16 and float32, mixed at will, on one device.  None is passed over.
            The norm is that of these tensors: nothing is added up over processes.
        max_norm: positive; infinity scales by the divisor alone.
        divisor: the factor that the loss was multiplied by (a loss scale, a number of accumulated steps): a positive number, or a
            float32 tensor with one.
        out: tensors in the gradients' place to write to, of their dtype or float32 (an optimizer's copies), no two sharing memory.
            Default: the gradients themselves, which are left alone where nothing changes.

    Squares are summed in float64, in the same order for the same list.
    """
    if isinstance(grads, torch.Tensor):
        grads, out = [grads], None if out is None else [out]
    grads = list(grads)
    out = grads if out is None else list(out)
    if len(out) == len(grads):
        kept = [i for i, g in enumerate(grads) if g is not None]
        grads, out = [grads[i] for i in kept], [out[i] for i in kept]
    max_norm = float(max_norm)
    divisor = divisor if isinstance(divisor, torch.Tensor) else float(divisor)
    by_ptr = isinstance(divisor, torch.Tensor)
    if grads and max_norm > _lib.F32_ZERO and isinstance(grads[0], torch.Tensor) and grads[0].is_cuda and (
            grads[0].device.index == torch._C._cuda_getDevice()) and (by_ptr or _lib.F32_ZERO < divisor < _lib.F32_INF):
        done = _lib.host().clip(grads, out, max_norm, 1.0 if by_ptr else divisor, divisor if by_ptr else None, _stream(grads[0].device))
        if isinstance(done, torch.Tensor):
            return done
        if done is not None:
            _raise(*done)
    _check(grads, out, max_norm, divisor)
    if not grads:
        raise ValueError("clip_gradients: there are no gradients")
    dev = grads[0].device
    late = []  # (outputs that are not written in place)
    with _on_device(dev):
        tasks = (_lib.LceTensor * len(grads))()
        held = []
        for task, g, o in zip(tasks, grads, out):
            to = o
            if not _dense(o) or g.stride() != o.stride():
                to = torch.empty(o.shape, dtype=o.dtype, device=dev)
                late.append((o, to))
                g = g.contiguous() if o is not g else to.copy_(g)
            held.append((g, to))
            task.grad, task.out, task.n = g.data_ptr(), to.data_ptr(), g.numel()
            task.dtype, task.out_dtype = _lib.dtype_code(g.dtype), _lib.dtype_code(to.dtype)
        b = ctypes.c_size_t(0)
        lib = _lib.load()
        _lib.raise_for_status(lib.lce_clip_workspace_bytes(tasks, len(tasks), ctypes.byref(b)), "clip_gradients")
        ws = torch.empty(b.value, dtype=torch.uint8, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        rc = lib.lce_clip(tasks, len(tasks), max_norm, 1.0 if by_ptr else divisor, _ptr(divisor) if by_ptr else None, _ptr(norm), _ptr(ws),
                          b.value, _stream(dev))
        _raise(rc, "clip_gradients")
        for o, to in late:
            o.copy_(to)
        torch.autograd.graph.increment_version(out)  # (written behind autograd's back)
        del ws, held
    return norm
