"""Logits and log-probabilities of given tokens at the output layer, differentiable row by row.

``linear_token_logits`` stands beside ``linear_cross_entropy`` (ops.py) where the mean over the tokens is not the loss: policy
gradients and preference losses, scores under a frozen model, a vocabulary in pieces.  It runs on the same kernels, the logits of the
other columns do not reach memory, and the backward, which is told the upstream gradient of every row, recomputes them.  (No
counterpart in the reference.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from .ops import _on_device, _ptr, _stream


def _check_inputs(x, At, tokens):
    if not (x.is_cuda and At.is_cuda and tokens.is_cuda):
        raise RuntimeError(
            "linear_token_logits needs its tensors on an AMD GPU (device type 'cuda' under ROCm); there is no CPU path")
    if not (x.device == At.device == tokens.device):
        raise ValueError("x, weight and tokens must be on the same device")
    if At.dim() != 2:
        raise ValueError("weight must be 2-D with shape (in_features, out_features)")
    if x.dim() < 1 or At.shape[0] != x.shape[-1]:
        raise ValueError(f"weight has in_features={At.shape[0]}, input has {x.shape[-1] if x.dim() else 'no dimension'}")
    if tokens.dtype != torch.int64:
        raise ValueError("tokens must be a torch.long tensor")
    if tokens.shape != x.shape[:-1]:
        raise ValueError(f"tokens must have one entry per row of x: got {tuple(tokens.shape)} and x of shape {tuple(x.shape)}")


def _check_numbers(V, vocab_start, vocab_size, logit_scale):
    if not (_lib.F32_ZERO < logit_scale < _lib.F32_INF):
        raise ValueError(f"logit_scale must be positive and finite in float32, got {logit_scale}")
    if not 0 <= vocab_start <= vocab_size - V:
        raise ValueError(f"columns {vocab_start} ... {vocab_start + V - 1} do not lie in a vocabulary of {vocab_size}")


def _problem(x, w, layout, V, ignore_index, logit_scale, N_chunk_size, pack):
    N, H = x.shape
    w_cols = H if layout == _lib.W_VH else V
    return _lib.make_problem(
        N, H, V, x.stride(0), w.stride(0), ops._dx_cols(H, x.dtype), ops._padded_cols(w_cols, w.dtype), x.dtype, w.dtype, x.dtype, w.dtype,
        ignore_index, logit_scale, 0.0, N_chunk_size, False, 0, pack, 0, layout)


def _forward(x_in, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size, pack):
    """(logits, lse) and what the backward reads: the views x and w, w's layout, the labels with their ignore_index."""
    ops._check_dtypes(x_in, At)
    V, dev = At.shape[1], x_in.device
    if dev.index == torch._C._cuda_getDevice():
        done = _lib.host().token_logits(x_in, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size, pack,
                                        "weight" in ops._copy_warned, _stream(dev))
        if done is not None and len(done) == 2:
            _lib.raise_for_status(*done)
        if done is not None:
            return done
    with _on_device(dev):
        x = ops._aligned_rows(x_in.reshape(-1, x_in.shape[-1]))
        layout = ops._weight_layout(At, x.dtype)
        w = ops._weight_rows(At, layout)
        N = x.shape[0]
        logits = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        lse = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        labels = tokens.reshape(-1).contiguous()
        if N == 0:
            return logits, lse, x, w, layout, labels, ignore_index
        other = ignore_index
        if vocab_size != V:  # (one piece of several: its own columns are counted from 0)
            given, labels = labels, torch.empty_like(labels)
            rc = _lib.load().lce_token_labels(_ptr(given), N, ignore_index, vocab_start, V, vocab_size, _ptr(labels), _stream(dev))
            _lib.raise_for_status(rc, "linear_token_logits")
            ignore_index, other = -1, V
        prob = _problem(x, w, layout, V, ignore_index, logit_scale, N_chunk_size, pack)
        nbytes = _lib.token_logits_workspace_bytes(prob, False)  # (checks the problem)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = _lib.load().lce_token_logits(ctypes.byref(prob), _ptr(x), _ptr(w), _ptr(labels), other, _ptr(logits), _ptr(lse), None, _ptr(ws), nbytes,
                                          _stream(dev))
        _lib.raise_for_status(rc, "linear_token_logits")
        del ws
    return logits, lse, x, w, layout, labels, ignore_index


def _backward(x, w, layout, labels, logits, lse, g_logits, g_lse, ignore_index, logit_scale, N_chunk_size, pack, need_dx, need_dw):
    """(dx, dw): dx (N, H), dw (H, V) as the weight is stored; None where it is not needed."""
    N, H = x.shape
    V = w.shape[0] if layout == _lib.W_VH else w.shape[1]
    dev = x.device
    if dev.index == torch._C._cuda_getDevice():
        done = _lib.host().token_logits_backward(x, w, layout, labels, logits, lse, g_logits, g_lse, ignore_index, logit_scale, N_chunk_size, pack,
                                                 need_dx, need_dw, _stream(dev))
        if done is not None:
            if len(done) == 3:
                _lib.raise_for_status(*done[:2])
            dx, dw = done
            return dx, dw.t() if layout == _lib.W_VH and dw is not None else dw
    with _on_device(dev):
        dx, dw = ops._alloc_grads(x, w, layout, N, H, V, need_dx, need_dw)
        if N == 0:
            dw = dw.zero_() if need_dw else None
        else:
            prob = _problem(x, w, layout, V, ignore_index, logit_scale, N_chunk_size, pack)
            nbytes = _lib.token_logits_workspace_bytes(prob, True)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            rows = [t.detach().to(device=dev, dtype=torch.float32).reshape(-1).contiguous() for t in (logits, lse, g_logits, g_lse)]
            rc = _lib.load().lce_token_logits_backward(ctypes.byref(prob), _ptr(x), _ptr(w), _ptr(labels), *map(_ptr, rows), None, _ptr(dx), _ptr(dw),
                                                       _ptr(ws), nbytes, _stream(dev))
            _lib.raise_for_status(rc, "linear_token_logits")
            del ws
    return ops._finish_grads(dx, dw, layout)


class TokenLogitsImplementation(torch.autograd.Function):
    """Autograd Function behind ``linear_token_logits``; gradients for ``x`` and ``At``."""

    @staticmethod
    def forward(ctx, x_in, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size):
        x_in = ops._autocast_x(x_in, At)
        pack = ops._pack_mode()
        logits, lse, x, w, layout, labels, ignore = _forward(x_in, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size,
                                                             pack)
        ctx.save_for_backward(x, w, labels, logits, lse)
        ctx.lce_cfg = (layout, ignore, logit_scale, N_chunk_size, pack)
        ctx.x_shape = x_in.shape
        return logits, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logits, g_lse):
        x, w, labels, logits, lse = ctx.saved_tensors
        x, w = ops._aligned_rows(x), ops._aligned_rows(w)  # (hooks on saved tensors may bring them back with other strides)
        layout, ignore, logit_scale, N_chunk_size, pack = ctx.lce_cfg
        dx, dw = _backward(x, w, layout, labels, logits, lse, g_logits, g_lse, ignore, logit_scale, N_chunk_size, pack,
                           ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx.view(ctx.x_shape) if dx is not None else None, dw, None, None, None, None, None, None


# The same for torch.compile / torch.export: two opaque operators (ops.py).
@torch.library.custom_op("lce_amd::token_logits", mutates_args=(), device_types="cuda")
def _op_token_logits(x: torch.Tensor, At: torch.Tensor, tokens: torch.Tensor, ignore_index: int, logit_scale: float, N_chunk_size: int,
                     vocab_start: int, vocab_size: int, pack_rows_mode: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    return _forward(x, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size, pack_rows_mode)[:2]


@_op_token_logits.register_fake
def _(x, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size, pack_rows_mode=0):
    return x.new_empty(tokens.shape, dtype=torch.float32), x.new_empty(tokens.shape, dtype=torch.float32)


@torch.library.custom_op("lce_amd::token_logits_backward", mutates_args=(), device_types="cuda")
def _op_token_logits_backward(x: torch.Tensor, At: torch.Tensor, tokens: torch.Tensor, logits: torch.Tensor, lse: torch.Tensor,
                              g_logits: torch.Tensor, g_lse: torch.Tensor, ignore_index: int, logit_scale: float, N_chunk_size: int,
                              vocab_start: int, vocab_size: int, need_dx: bool, need_dw: bool, pack_rows_mode: int = 0
                              ) -> tuple[torch.Tensor, torch.Tensor]:
    V = At.shape[1]
    with _on_device(x.device):
        x2 = ops._aligned_rows(x.reshape(-1, x.shape[-1]))
        layout = ops._weight_layout(At, x2.dtype)
        w = ops._weight_rows(At, layout)
        labels = tokens.reshape(-1).contiguous()
        if vocab_size != V and labels.numel():
            given, labels = labels, torch.empty_like(labels)
            rc = _lib.load().lce_token_labels(_ptr(given), given.numel(), ignore_index, vocab_start, V, vocab_size, _ptr(labels),
                                              _stream(x.device))
            _lib.raise_for_status(rc, "linear_token_logits")
            ignore_index = -1
    dx, dw = _backward(x2, w, layout, labels, logits, lse, g_logits, g_lse, ignore_index, logit_scale, N_chunk_size, pack_rows_mode, need_dx,
                       need_dw)
    dx = dx.view(x.shape) if dx is not None else x.new_empty((0,))
    return dx, dw if dw is not None else At.new_empty((0,))


@_op_token_logits_backward.register_fake
def _(x, At, tokens, logits, lse, g_logits, g_lse, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size, need_dx, need_dw,
      pack_rows_mode=0):
    return ops._fake_grads(x, At, need_dx, need_dw)


def _setup_context(ctx, inputs, output):
    x, At, tokens, *ctx.lce_cfg = inputs
    ctx.save_for_backward(x, At, tokens, *output)


def _autograd(ctx, g_logits, g_lse):
    x, At, tokens, logits, lse = ctx.saved_tensors
    *cfg, pack = ctx.lce_cfg
    need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    dx, dw = _op_token_logits_backward(x, At, tokens, logits, lse, g_logits, g_lse, *cfg, need_dx, need_dw, pack)
    return (dx if need_dx else None, dw if need_dw else None) + (None,) * 7


_op_token_logits.register_autograd(_autograd, setup_context=_setup_context)


def linear_token_logits(x, At, tokens, ignore_index: int = -100, logit_scale: float = 1.0, N_chunk_size: int = 4096,
                        vocab_start: int = 0, vocab_size=None):
    """The logit of each row's token and the logsumexp of the row's logits: ``(logits, lse)``, float32, of the shape of ``tokens``.

    The logits are ``logit_scale * x @ At`` over all columns of ``At``; they are not formed in memory.  ``logits - lse`` is the tokens'
    log-probability.  Both results are differentiable, with any upstream gradient in every row; the backward evaluates the logits
    again, in the scratch that ``N_chunk_size`` allows.

    Args:
        x: hidden states (..., H): bfloat16, float16 or float32.
        At: weight (H, V) with the strides that ``linear_cross_entropy`` takes: of x's dtype, or float32 under 16-bit x.
        tokens: (...) torch.long.
        ignore_index: a token that marks a row as not wanted (prompts, padding): it is not computed, both results are 0 and
            it has no gradient, whatever the upstream gradient is there.  (What x holds there is to be finite: where few rows
            are marked they stay in the products, times zero.)
        N_chunk_size: as of ``LinearCrossEntropyLoss``.
        vocab_start, vocab_size: where ``At`` is one piece of a vocabulary, the token that its first column stands for and the number
            of all tokens.  A token of another piece has a logit of 0 here, so that the sum of the pieces' logits and the
            ``logsumexp`` of their lse are those of the whole.

    A token that is none (negative or beyond the vocabulary, and not ``ignore_index``) has a NaN logit.  Arithmetic as of
    ``linear_cross_entropy``: 16-bit gradients come from a dz that was rounded to the type, float32 tensors are multiplied as
    pairs of float16 under one power of two for each of x, weight and dz, and hold 22 bits (``linear_cross_entropy``: pairs of
    bfloat16, 16 bits) or 2^-39 of the largest element there (as long as that is at least 2^-106, and the product of any two of x's, the
    weight's and the upstream gradients' at least 2^-92: below, steps grow beside the elements); float16's dz is held to 2^-38 of the largest row's
    upstream gradient.
    The gradients are not differentiable in their turn.
    """
    compiling = torch.compiler.is_compiling()
    if At.dim() != 2:
        _check_inputs(x, At, tokens)
    V, ignore_index, logit_scale = At.shape[-1], int(ignore_index), float(logit_scale)
    vocab_start = int(vocab_start)
    vocab_size = vocab_start + V if vocab_size is None else int(vocab_size)
    if not compiling and x.is_cuda and x.device.index == torch._C._cuda_getDevice() and not torch.is_autocast_enabled("cuda") and (
            _lib.F32_ZERO < logit_scale < _lib.F32_INF) and 0 <= vocab_start <= vocab_size - V:
        done = _lib.host().differentiable_token_logits(x, At, tokens, ignore_index, logit_scale, int(N_chunk_size), vocab_start, vocab_size,
                                                       ops._pack_mode(), "weight" in ops._copy_warned, _stream(x.device))
        if done is not None and len(done) == 3:
            _lib.raise_for_status(*done[:2])
        if done is not None:
            return done
    _check_inputs(x, At, tokens)
    _check_numbers(V, vocab_start, vocab_size, logit_scale)
    if not compiling:
        return TokenLogitsImplementation.apply(x, At, tokens, ignore_index, logit_scale, int(N_chunk_size), vocab_start, vocab_size)
    return _op_token_logits(ops._autocast_x(x, At), At, tokens, ignore_index, logit_scale, int(N_chunk_size), vocab_start, vocab_size,
                            ops._pack_mode())
