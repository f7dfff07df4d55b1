"""Distillation at the output layer: the loss of a student's hidden states against a teacher's top logits.

``linear_distillation`` stands beside ``linear_cross_entropy`` (ops.py) and runs on the same kernels, with K targets a row in
the place of one label: the logits do not reach memory, and where a gradient is wanted it is computed along with the
loss and multiplied by the upstream gradient in the backward.  (No counterpart in the reference.)
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib, ops
from .ops import _on_device, _ptr, _stream

_NO_LABEL = -1  # lce_soft_targets' label of a row without a target


def _check_inputs(x, At, index, logits):
    if not (x.is_cuda and At.is_cuda and index.is_cuda and logits.is_cuda):
        raise RuntimeError(
            "linear_distillation needs its tensors on an AMD GPU (device type 'cuda' under ROCm); there is no CPU path")
    if not (x.device == At.device == index.device == logits.device):
        raise ValueError("x, weight, index and logits must be on the same device")
    if At.dim() != 2:
        raise ValueError("weight must be 2-D with shape (in_features, out_features)")
    if At.shape[0] != x.shape[-1]:
        raise ValueError(f"weight has in_features={At.shape[0]}, input has {x.shape[-1]}")
    if index.dtype != torch.int64:
        raise ValueError("index must be a torch.long tensor")
    _lib.dtype_code(logits.dtype)
    if index.shape != logits.shape or index.dim() < 1 or index.shape[:-1] != x.shape[:-1]:
        raise ValueError(
            f"index and logits must have shape (..., K) with one row per row of x: got {tuple(index.shape)}, "
            f"{tuple(logits.shape)} and x of shape {tuple(x.shape)}")
    if not 1 <= index.shape[-1] <= _lib.MAX_TARGETS:
        raise ValueError(f"a row has {index.shape[-1]} targets: 1 to {_lib.MAX_TARGETS} are supported")


def _check_numbers(temperature, logit_scale):
    if not (_lib.F32_ZERO < temperature < _lib.F32_INF):
        raise ValueError(f"temperature must be positive and finite in float32, got {temperature}")
    if not (0.0 < logit_scale < math.inf):
        raise ValueError(f"logit_scale must be positive and finite, got {logit_scale}")
    if not (_lib.F32_ZERO < logit_scale / temperature < _lib.F32_INF):
        raise ValueError(f"logit_scale / temperature must be positive and finite in float32, got {logit_scale} / {temperature}")


def _rows_of(t):
    """(rows, K) view whose rows are contiguous (their stride is free)."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _targets(index, logits, V, temperature):
    """(columns, probabilities, labels) of lce_soft_targets."""
    index, logits = _rows_of(index), _rows_of(logits)
    N, K = index.shape
    dev = index.device
    columns = torch.empty((N, K), dtype=torch.int32, device=dev)
    q = torch.empty((N, K), dtype=torch.float32, device=dev)
    y = torch.empty(N, dtype=torch.int64, device=dev)
    with _on_device(dev):
        rc = _lib.load().lce_soft_targets(N, K, V, _ptr(index), index.stride(0), _ptr(logits), _lib.dtype_code(logits.dtype),
                                          logits.stride(0), temperature, _ptr(columns), _ptr(q), _ptr(y), _stream(dev))
    _lib.raise_for_status(rc, "linear_distillation")
    return columns, q, y


def _views(x_in, At):
    """The matrices that the kernels read and the weight's layout, as ops._problem_views gives them."""
    ops._check_dtypes(x_in, At)
    x = ops._aligned_rows(x_in.reshape(-1, x_in.shape[-1]))
    layout = ops._weight_layout(At, x.dtype)
    return x, ops._weight_rows(At, layout), layout


def _run(x, w, layout, targets, scale, N_chunk_size, pack, route, need_dx, need_dw, grad_output):
    """lce_distill.  Returns (loss, dx, dw); `grad_output`: a device scalar, None for 1."""
    columns, q, y = targets
    N, H = x.shape
    vh = layout == _lib.W_VH
    V = w.shape[0] if vh else w.shape[1]
    w_cols = H if vh else V
    grads = need_dx or need_dw
    lib, dev = _lib.load(), x.device
    with _on_device(dev):
        prob = _lib.make_problem(
            N, H, V, x.stride(0), w.stride(0), ops._dx_cols(H, x.dtype), ops._padded_cols(w_cols, w.dtype), x.dtype, w.dtype,
            x.dtype, w.dtype, _NO_LABEL, scale, 0.0, N_chunk_size, False, 0, pack, 0, layout,
            (_lib.ROUTE_TWO_PASS if route == 0 else _lib.ROUTE_ONE_PASS if route == 2 else _lib.ROUTE_AUTO)
            | (_lib.ROUTE_EXACT_SUMS if ops.exact_dw_sums.get() else 0)
            | (_lib.ROUTE_KEEP_LOGITS if x.dtype == torch.float32 else 0))
        nbytes = _lib.distill_workspace_bytes(prob, columns.shape[1], grads)  # (checks the problem)
        dx, dw = ops._alloc_grads(x, w, layout, N, H, V, need_dx, need_dw)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        lse = torch.empty(N, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        n_valid = torch.empty(1, dtype=torch.int64, device=dev)
        g = _lib.unit_gradient() if grad_output is None else _ptr(grad_output)
        rc = lib.lce_distill(ctypes.byref(prob), columns.shape[1], _ptr(columns), _ptr(q), _ptr(y), _ptr(x), _ptr(w), g, _ptr(lse),
                             _ptr(loss), _ptr(n_valid), _ptr(dx), _ptr(dw), _ptr(ws), nbytes, _stream(dev))
        _lib.raise_for_status(rc, "lce_distill")
        del ws
    return loss, dx, dw


def _native(x, At, index, logits, temperature, scale, N_chunk_size, pack, route, need_dx, need_dw):
    """All of the forward by the host extension (csrc/lce_host.cpp), which returns the same bits; None: no ordinary call, or one that
    has a warning to give."""
    if x.device.index != torch._C._cuda_getDevice():
        return None
    done = _lib.host().distill(x, At, index, logits, temperature, scale, N_chunk_size, pack, route, bool(ops.exact_dw_sums.get()), need_dx,
                               need_dw, "weight" in ops._copy_warned, _stream(x.device))
    if done is not None and len(done) == 2:
        _lib.raise_for_status(*done)
    return done


class LinearDistillationImplementation(torch.autograd.Function):
    """Autograd Function behind ``linear_distillation``; gradients for ``x`` and ``At`` only (the teacher is a constant)."""

    @staticmethod
    def forward(ctx, x_in, At, index, logits, temperature, logit_scale, N_chunk_size, grad_mode):
        x_in = ops._autocast_x(x_in, At)
        need_dx, need_dw = grad_mode and ctx.needs_input_grad[0], grad_mode and ctx.needs_input_grad[1]
        cfg = (logit_scale / temperature, N_chunk_size, ops._pack_mode(), ops._route_mode())
        native = _native(x_in, At, index, logits, temperature, *cfg, need_dx, need_dw)
        if native is not None:
            loss, dx, dw, pre, x, w, layout, *targets = native
        else:
            with _on_device(x_in.device):
                x, w, layout = _views(x_in, At)
                targets = _targets(index, logits, At.shape[1], temperature)
                pre = None
                if (need_dx or need_dw) and x.dtype == torch.float16:
                    pre = ops._stand_in_gradient(x, targets[2], _NO_LABEL)
                loss, dx, dw = _run(x, w, layout, targets, *cfg, need_dx, need_dw, pre)
        ctx.lce_grads = [dx, dw, pre]  # for the first backward; dropped there
        if need_dx or need_dw:
            ctx.save_for_backward(x, w, *targets)
        ctx.lce_cfg = (layout, cfg)
        ctx.x_shape = x_in.shape
        return loss

    @staticmethod
    def backward(ctx, grad_output):
        x, w, *targets = ctx.saved_tensors
        layout, cfg = ctx.lce_cfg
        grads, ctx.lce_grads = ctx.lce_grads, None
        if grads is not None:
            dx, dw, pre = grads
            ops._scale_grads(dx, dw, grad_output, pre)
        else:  # a later backward over the same graph: the first one's gradients were handed out
            with _on_device(x.device):
                g = ops._device_scalar(grad_output, x.device)
                _, dx, dw = _run(x, w, layout, targets, *cfg, ctx.needs_input_grad[0], ctx.needs_input_grad[1], g)
        dx, dw = ops._finish_grads(dx, dw, layout)
        if dx is not None:
            dx = dx.view(ctx.x_shape)
        return dx, dw, None, None, None, None, None, None


# The same for torch.compile / torch.export, as ops.py does it for the loss against labels: an opaque operator that returns the
# gradients along with the loss, and an autograd formula that multiplies the upstream gradient in.
@torch.library.custom_op("lce_amd::distill", mutates_args=(), device_types="cuda")
def _op_distill(x: torch.Tensor, At: torch.Tensor, index: torch.Tensor, logits: torch.Tensor, temperature: float, logit_scale: float,
                N_chunk_size: int, need_dx: bool, need_dw: bool, pack_rows_mode: int = 0, route: int = 1
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    with _on_device(x.device):
        x2, w, layout = _views(x, At)
        targets = _targets(index, logits, At.shape[1], temperature)
        pre = ops._stand_in_gradient(x2, targets[2], _NO_LABEL)
        loss, dx, dw = _run(x2, w, layout, targets, logit_scale / temperature, N_chunk_size, pack_rows_mode, route, need_dx, need_dw, pre)
        dx, dw = ops._finish_grads(dx, dw, layout)
    dx = dx.view(x.shape) if dx is not None else x.new_empty((0,))
    return loss, dx, dw if dw is not None else At.new_empty((0,)), pre


@_op_distill.register_fake
def _(x, At, index, logits, temperature, logit_scale, N_chunk_size, need_dx, need_dw, pack_rows_mode=0, route=1):
    dx, dw = ops._fake_grads(x, At, need_dx, need_dw)
    return x.new_empty((), dtype=torch.float32), dx, dw, x.new_empty((1,), dtype=torch.float32)


def _setup_context(ctx, inputs, output):
    _, dx, dw, pre = output
    ctx.save_for_backward(dx, dw, pre)


def _autograd(ctx, grad_loss, grad_dx, grad_dw, grad_pre):
    dx, dw, pre = ctx.saved_tensors
    factor = grad_loss.reshape(1).to(torch.float32) / pre
    gx = ops._op_scale(dx, factor) if ctx.needs_input_grad[0] else None
    gw = ops._op_scale(dw, factor) if ctx.needs_input_grad[1] else None
    return gx, gw, None, None, None, None, None, None, None, None, None


_op_distill.register_autograd(_autograd, setup_context=_setup_context)


def linear_distillation(x, At, index, logits, temperature: float = 1.0, logit_scale: float = 1.0, N_chunk_size: int = 4096):
    """Mean over the rows of KL(teacher || student), both at ``temperature``, the teacher known by its top logits.

    The student's logits are ``logit_scale * x @ At`` over all columns of ``At``; they are not formed in memory.  The teacher's
    distribution is the softmax of the logits that a row of ``logits`` holds, at the columns that ``index`` names, over those
    columns (``top_logits`` makes both).  At a temperature other than 1 the gradients shrink with its square: multiply the
    loss by ``temperature ** 2`` to weigh it against a loss on labels.

    Args:
        x: hidden states (..., H): bfloat16, float16 or float32.
        At: weight (H, V) with the strides that ``linear_cross_entropy`` takes: of x's dtype, or float32 under 16-bit x.
        index: (..., K) columns, torch.long, 1 <= K <= 1024, 2^30 of them at most.  A negative one, whatever its logit, is no
            target; one of V and above makes the loss NaN.  A column may be named twice: its probabilities add up.
        logits: (..., K) the teacher's logits there: bfloat16, float16 or float32.  -inf is no target, NaN and +inf make the loss NaN.
        temperature: divides both sides' logits.
        N_chunk_size: as of ``LinearCrossEntropyLoss``.

    float32 tensors are multiplied as pairs of bfloat16 (16 bits of mantissa), as by ``linear_cross_entropy``; 16-bit gradients come from a
    softmax minus target that was rounded to the type.

    Rows without a target (prompts, padding) have no gradient and do not count in the mean; no row with one at all gives NaN
    and zero gradients, as a batch without labels does.  Returns the loss (float32); gradients go to ``x`` and ``At``.
    """
    _check_inputs(x, At, index, logits)
    temperature, logit_scale = float(temperature), float(logit_scale)
    _check_numbers(temperature, logit_scale)
    if not torch.compiler.is_compiling():
        return LinearDistillationImplementation.apply(x, At, index.detach(), logits.detach(), temperature, logit_scale, int(N_chunk_size),
                                                      torch.is_grad_enabled())
    x = ops._autocast_x(x, At)
    need = torch.is_grad_enabled()
    return _op_distill(x, At, index, logits.detach(), temperature, logit_scale, int(N_chunk_size), need and x.requires_grad,
                       need and At.requires_grad, ops._pack_mode(), ops._route_mode())[0]
