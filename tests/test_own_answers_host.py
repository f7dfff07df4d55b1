"""CPU-side checks of what a model needs that is trained on its own answers (lce_token_logits, lce_quantize_*, lce_int8_logits, lce_clip): what
they refuse, what scratch they plan, and the Python surface.  Every call here is refused before a device is asked for, or has no rows."""
import ctypes
import math
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = ctypes.create_string_buffer(1 << 16)
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256  # memory of the host: nothing here may get as far as a kernel
BIG = 1 << 60


@pytest.fixture(scope="module")
def lib():
    from linear_cross_entropy_loss_amd import _lib
    from linear_cross_entropy_loss_amd.build import build

    build(force=False)
    return _lib.load()


def _prob(**kw):
    from linear_cross_entropy_loss_amd import _lib

    d = dict(N=512, H=256, V=4096, ldx=256, ldw=4096, lddx=256, lddw=4096, x_dtype=torch.bfloat16, w_dtype=torch.bfloat16,
             dx_dtype=torch.bfloat16, dw_dtype=torch.bfloat16, ignore_index=-100, logit_scale=1.0, z_reg=0.0, n_chunk=4096,
             monitoring=False)
    d.update(kw)
    return _lib.make_problem(**d)


SHAPE, DTYPE, ARG, WORKSPACE = -1, -2, -3, -4


def test_struct_of_a_tensor_matches_the_header():
    from linear_cross_entropy_loss_amd import _lib

    header = open(os.path.join(ROOT, "include", "lce.h")).read()
    body = re.search(r"typedef struct lce_tensor \{(.*?)\} lce_tensor;", header, flags=re.S).group(1)
    names = re.findall(r"(\w+);", body)
    assert names == [n for n, _ in _lib.LceTensor._fields_] and ctypes.sizeof(_lib.LceTensor) == 32


@pytest.mark.parametrize("kw, status", [(dict(N=0), SHAPE), (dict(H=0), SHAPE), (dict(n_chunk=0), SHAPE), (dict(ldx=255), ARG), (dict(z_reg=0.1), ARG),
                                        (dict(monitoring=True), ARG), (dict(phases=1), ARG), (dict(logit_scale=0.0), ARG),
                                        (dict(logit_scale=math.inf), ARG), (dict(logit_scale=math.nan), ARG),
                                        (dict(w_dtype=torch.float16, dw_dtype=torch.float16), DTYPE)])
def test_token_logits_problems(lib, kw, status):
    f, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    p = ctypes.byref(_prob(**kw))
    assert lib.lce_token_logits_workspace_bytes(p, ctypes.byref(f), ctypes.byref(b)) == status
    assert lib.lce_token_logits(p, PTR, PTR, PTR, 0, PTR, PTR, None, PTR, BIG, None) == status
    assert lib.lce_token_logits_backward(p, *[PTR] * 7, None, PTR, PTR, PTR, BIG, None) == status


def test_token_logits_arguments(lib):
    p = ctypes.byref(_prob())
    f, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.lce_token_logits_workspace_bytes(p, ctypes.byref(f), ctypes.byref(b)) == 0
    good = [PTR, PTR, PTR, 0, PTR, PTR, None, PTR]
    for i in (0, 1, 2, 4, 5):
        assert lib.lce_token_logits(p, *[None if i == j else g for j, g in enumerate(good)], BIG, None) == ARG, i
    assert lib.lce_token_logits(p, *good[:-1], None, BIG, None) == WORKSPACE
    assert lib.lce_token_logits(p, *good, f.value - 1, None) == WORKSPACE
    for i in range(7):
        assert lib.lce_token_logits_backward(p, *[None if i == j else PTR for j in range(7)], None, PTR, PTR, PTR, BIG, None) == ARG, i
    assert lib.lce_token_logits_backward(p, *[PTR] * 7, None, None, None, PTR, BIG, None) == ARG
    assert lib.lce_token_logits_backward(p, *[PTR] * 7, None, PTR, PTR, PTR, b.value - 1, None) == WORKSPACE
    # the backward stages dz within the scratch bound of the loss (N_chunk_size * V * 4) wherever the narrowest split fits
    for N, H, V, chunk in ((16384, 768, 50264, 4096), (4096, 64, 32768, 1024)):
        q = _prob(N=N, H=H, V=V, ldx=H, ldw=V, lddx=H, lddw=V, n_chunk=chunk)
        assert lib.lce_token_logits_workspace_bytes(ctypes.byref(q), None, ctypes.byref(b)) == 0
        assert b.value <= chunk * V * 4 + N * 12 + 4096


@pytest.mark.parametrize("N, start, V, size", [(-1, 0, 5, 5), (1, -1, 5, 9), (1, 0, 0, 5), (1, 5, 5, 9), (1, 0, 6, 5), (1, 0, (1 << 30) + 1, 1 << 40),
                                               (1, 1 << 62, 5, (1 << 62) + 4)])
def test_token_labels_sizes(lib, N, start, V, size):
    assert lib.lce_token_labels(PTR, N, -100, start, V, size, PTR, None) == SHAPE


def test_token_labels_arguments(lib):
    assert lib.lce_token_labels(None, 1, -100, 0, 5, 5, PTR, None) == ARG
    assert lib.lce_token_labels(PTR, 1, -100, 0, 5, 5, None, None) == ARG
    assert lib.lce_token_labels(None, 0, -100, 0, 5, 5, None, None) == 0


@pytest.mark.parametrize("call, rows, cols", [("lce_quantize_rows", 5, 100), ("lce_quantize_columns", 100, 5)])
def test_quantize(lib, call, rows, cols):
    f = getattr(lib, call)
    ok = dict(src=PTR, dtype=0, rows=rows, cols=cols, ld=cols, q=PTR, ldq=112, scales=PTR)

    def run(**kw):
        return f(*{**ok, **kw}.values(), None)

    depth, others = ("cols", "rows") if call == "lce_quantize_rows" else ("rows", "cols")
    assert run(dtype=3) == run(dtype=-1) == DTYPE
    for bad in ({depth: 0}, {others: 0}, {depth: (1 << 17) + 1, "ldq": 1 << 18}, {others: (1 << 30) + 1}, {depth: -5}, {others: -5}):
        assert run(**bad) == SHAPE, bad
    for bad in (dict(src=None), dict(q=None), dict(scales=None), dict(q=PTR + 8), dict(ldq=96), dict(ldq=104), dict(ld=-1), dict(src=PTR + 1),
                dict(src=PTR + 2, dtype=2), dict(ldq=1 << 19)):
        assert run(**bad) == ARG, bad


def test_int8_logits(lib):
    b = ctypes.c_size_t(0)
    assert lib.lce_int8_logits_workspace_bytes(7, 100, 50, ctypes.byref(b)) == 0 and b.value >= 7 * 112 + 28
    ok = dict(x=PTR, x_dtype=0, N=7, H=100, V=50, ldx=100, w=PTR, ldw=112, w_scales=PTR, scale=1.0, out=PTR, out_dtype=2, ldo=50, ws=PTR, ws_bytes=b.value)

    def run(**kw):
        return lib.lce_int8_logits(*{**ok, **kw}.values(), None)

    for bad in (dict(N=-1), dict(H=0), dict(H=(1 << 17) + 1), dict(V=0), dict(V=(1 << 30) + 1), dict(N=(1 << 30) + 1), dict(N=1 << 25, V=1 << 25)):
        assert run(**bad) == SHAPE, bad
    assert run(x_dtype=3) == run(out_dtype=7) == DTYPE
    for bad in (dict(x=None), dict(w=None), dict(w_scales=None), dict(out=None), dict(ldx=-1), dict(ldo=49), dict(w=PTR + 4), dict(ldw=104),
                dict(ldw=96), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(out=PTR + 2), dict(x=PTR + 1),
                dict(w_scales=PTR + 2)):
        assert run(**bad) == ARG, bad
    assert run(ws=None) == run(ws_bytes=b.value - 1) == run(ws=PTR + 8) == WORKSPACE
    assert run(N=0) == 0
    assert lib.lce_int8_logits_workspace_bytes(7, 100, 50, None) == ARG


def test_clip(lib):
    from linear_cross_entropy_loss_amd import _lib

    def tensors(*specs):
        return (_lib.LceTensor * max(1, len(specs)))(*[_lib.LceTensor(*s) for s in specs])

    b = ctypes.c_size_t(0)
    good = (PTR, PTR, 10, 0, 0)

    def run(*specs, max_norm=1.0, divisor=1.0, norm=PTR, ws=PTR, ws_bytes=BIG, count=None):
        return lib.lce_clip(tensors(*specs), len(specs) if count is None else count, max_norm, divisor, None, norm, ws, ws_bytes, None)

    assert lib.lce_clip_workspace_bytes(tensors(good), 1, ctypes.byref(b)) == 0 and b.value >= 8
    assert lib.lce_clip_workspace_bytes(tensors(good), 1, None) == ARG
    assert run(good, count=-1) == run((PTR, PTR, -1, 0, 0)) == run((PTR, PTR, (1 << 40) + 1, 0, 0)) == SHAPE
    assert run((PTR, PTR, 10, 3, 3)) == run((PTR, PTR + 64, 10, 0, 1)) == run((PTR, PTR + 64, 10, 2, 0)) == DTYPE
    for bad in ((None, PTR, 10, 0, 0), (PTR, None, 10, 0, 0), (PTR + 1, PTR + 1, 10, 0, 0), (PTR + 2, PTR + 2, 10, 2, 2), (PTR, PTR, 10, 0, 2)):
        assert run(bad) == ARG, bad
    for bad in (dict(max_norm=0.0), dict(max_norm=-1.0), dict(max_norm=math.nan), dict(divisor=0.0), dict(divisor=math.nan), dict(divisor=math.inf),
                dict(norm=None)):
        assert run(good, **bad) == ARG, bad
    assert run(good, ws=None) == run(good, ws_bytes=b.value - 1) == run(good, ws=PTR + 8) == WORKSPACE
    # memory that two outputs share, or an output and another's input
    a = PTR
    for pair in (((a, a, 10, 0, 0), (a, a, 10, 0, 0)), ((a, a, 10, 0, 0), (a + 18, a + 18, 10, 0, 0)), ((a, a + 100, 10, 0, 2), (a + 200, a + 138, 10, 0, 0)),
                 ((a, a + 100, 10, 0, 0), (a + 110, a + 300, 10, 0, 0)), ((a, a + 2, 10, 0, 0), (a + 400, a + 400, 10, 0, 0)),
                 ((a + 300, a + 400, 10, 0, 0), (a, a, 200, 0, 0))):
        assert run(*pair) == ARG, pair


def test_python_surface_refuses_on_the_cpu():
    from linear_cross_entropy_loss_amd import Quantized, clip_gradients, linear_token_logits, quantize_rows, quantize_weight, quantized_logits

    x, w, t = torch.zeros(3, 8), torch.zeros(8, 5), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: linear_token_logits(x, w, t), lambda: quantize_rows(x), lambda: quantize_weight(w),
                 lambda: quantized_logits(x, Quantized(torch.zeros(5, 8, dtype=torch.int8), torch.zeros(5))), lambda: clip_gradients([x], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_clip_gradients_arguments():
    from linear_cross_entropy_loss_amd import clip_gradients

    x = torch.zeros(3)
    for bad in (dict(max_norm=0.0), dict(max_norm=1e-50), dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, out=[])):
        with pytest.raises(ValueError):
            clip_gradients([x], **bad)
    with pytest.raises(ValueError, match="no gradients"):
        clip_gradients([], 1.0)
    with pytest.raises(ValueError, match="no gradients"):
        clip_gradients([None, None], 1.0)
    with pytest.raises(ValueError, match="must be tensors"):
        clip_gradients([3.0], 1.0)


def test_names():
    import linear_cross_entropy_loss_amd as pkg

    for name in ("linear_token_logits", "quantize_rows", "quantize_weight", "quantized_logits", "Quantized", "clip_gradients"):
        assert name in pkg.__all__ and getattr(pkg, name).__doc__
