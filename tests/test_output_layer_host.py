"""CPU-side checks of the operators around the output layer (lce_soft_targets, lce_distill, lce_top_logits, lce_sample): what they
refuse, what scratch they plan, and the Python surface.  Every call here is refused before a device is asked for, or has no rows."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32 = 0, 1, 2
BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256  # memory of the host: nothing here may get as far as a kernel


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


def _codes():
    from linear_cross_entropy_loss_amd import _lib

    assert [_lib.dtype_code(t) for t in (torch.bfloat16, torch.float16, torch.float32)] == [BF16, F16, F32]
    return _lib


def test_version_and_limit(lib):
    header = open(os.path.join(ROOT, "include", "lce.h")).read()
    assert lib.lce_version() >= 1000
    assert int(re.search(r"#define LCE_MAX_TARGETS (\d+)", header).group(1)) == _codes().MAX_TARGETS == 1024


def test_sampling_struct_matches_the_header():
    from linear_cross_entropy_loss_amd import _lib

    header = open(os.path.join(ROOT, "include", "lce.h")).read()
    body = re.search(r"typedef struct lce_sampling \{(.*?)\} lce_sampling;", header, flags=re.S).group(1)
    fields = re.findall(r"^\s*(const \w+\*|\w+)\s+(\w+);", body, flags=re.M)
    ctype = {"float": ctypes.c_float, "int64_t": ctypes.c_int64}
    assert [(n, ctype.get(t, ctypes.c_void_p)) for t, n in fields] == list(_lib.LceSampling._fields_)
    assert ctypes.sizeof(_lib.LceSampling) == 4 * 4 + 8 + 4 * 8  # (three floats and the padding before the int64)


def _soft(lib, N=4, K=8, V=100, index=PTR, ld_index=8, logits=PTR, dtype=BF16, ld=8, temperature=1.0, columns=PTR, q=PTR, y=PTR):
    return lib.lce_soft_targets(N, K, V, index, ld_index, logits, dtype, ld, temperature, columns, q, y, None)


def test_soft_targets_refusals(lib):
    L = _codes()
    for bad in (dict(N=0), dict(N=(1 << 30) + 1), dict(V=0), dict(V=(1 << 30) + 1), dict(K=0), dict(K=1025), dict(K=-1),
                dict(N=1 << 29, K=4), dict(N=(1 << 20) + 1, K=1024)):
        assert _soft(lib, **bad) == L.LCE_EINVAL_SHAPE, bad
    for bad in (3, -1):
        assert _soft(lib, dtype=bad) == L.LCE_EINVAL_DTYPE
    for bad in (dict(index=None), dict(logits=None), dict(columns=None), dict(q=None), dict(y=None), dict(ld_index=-1), dict(ld=-8),
                dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan"))):
        assert _soft(lib, **bad) == L.LCE_EINVAL_ARG, bad


def _distill(lib, p, K=8, index=PTR, q=PTR, y=PTR, x=PTR, w=PTR, g=PTR, lse=PTR, loss=PTR, n_valid=PTR, dx=PTR, dw=PTR, ws=PTR, size=0):
    return lib.lce_distill(ctypes.byref(p), K, index, q, y, x, w, g, lse, loss, n_valid, dx, dw, ws, size, None)


def test_distill_refusals(lib):
    L = _codes()
    for bad in (0, 1025, -3):
        assert _distill(lib, _prob(), K=bad) == L.LCE_EINVAL_SHAPE
    assert _distill(lib, _prob(N=(1 << 20) + 1), K=1024) == L.LCE_EINVAL_SHAPE
    assert _distill(lib, _prob(N=0)) == L.LCE_EINVAL_SHAPE
    for bad in (dict(index=None), dict(q=None), dict(y=None), dict(x=None), dict(w=None), dict(g=None), dict(lse=None), dict(loss=None),
                dict(n_valid=None), dict(x=PTR + 2), dict(w=PTR + 8), dict(dx=PTR + 4), dict(dw=PTR + 4)):
        assert _distill(lib, _prob(), **bad) == L.LCE_EINVAL_ARG, bad
    for bad in (dict(monitoring=True), dict(z_reg=1e-4), dict(logit_scale=0.0), dict(logit_scale=float("inf")),
                dict(logit_scale=float("nan")), dict(ldx=250)):
        assert _distill(lib, _prob(**bad)) == L.LCE_EINVAL_ARG, bad
    assert _distill(lib, _prob(x_dtype=torch.float32)) == L.LCE_EINVAL_DTYPE
    with_phases = _prob()
    with_phases.phases = 1
    assert _distill(lib, with_phases) == L.LCE_EINVAL_ARG
    # too little scratch, none, and scratch off its boundary
    need = _codes().distill_workspace_bytes(_prob(), 8, True)
    assert _distill(lib, _prob(), size=need - 1) == L.LCE_EWORKSPACE
    assert _distill(lib, _prob(), ws=None, size=need) == L.LCE_EWORKSPACE
    assert _distill(lib, _prob(), ws=PTR + 4, size=need) == L.LCE_EWORKSPACE


def test_a_caller_cannot_ask_for_the_inner_route(lib):
    """The kernels know a distillation by a bit of `route` that only the library sets."""
    L = _codes()
    for bit in range(8, 31):
        p = _prob(route=1 << bit)
        assert lib.lce_check_problem(ctypes.byref(p)) == L.LCE_EINVAL_ARG, bit
        assert _distill(lib, p) == L.LCE_EINVAL_ARG, bit


@pytest.mark.parametrize("route", [0, 1, 2])
@pytest.mark.parametrize("N,H,V,K", [(1, 8, 8, 1), (500, 264, 5000, 7), (512, 256, 4096, 1024), (16384, 2048, 131072, 32)])
def test_distill_workspace(lib, N, H, V, K, route):
    """At least the loss's scratch of the same problem and the 4 bytes an entry; no more with one direction, and a plan without
    gradients no larger than one with them."""
    L = _codes()
    dims = dict(N=N, H=H, V=V, ldx=H, ldw=V, lddx=H, lddw=V)
    p = _prob(**dims, route=route)
    with_grads, without = L.distill_workspace_bytes(p, K, True), L.distill_workspace_bytes(p, K, False)
    assert without <= with_grads and without >= 4 * N * K
    assert with_grads >= 4 * N * K
    assert L.distill_workspace_bytes(p, min(K + 1, 1024), True) >= with_grads
    size = ctypes.c_size_t()
    for bad in (0, 1025):
        assert lib.lce_distill_workspace_bytes(ctypes.byref(p), bad, 1, ctypes.byref(size)) == L.LCE_EINVAL_SHAPE
    assert lib.lce_distill_workspace_bytes(ctypes.byref(p), K, 1, None) == L.LCE_EINVAL_ARG
    assert lib.lce_distill_workspace_bytes(None, K, 1, ctypes.byref(size)) == L.LCE_EINVAL_ARG
    assert lib.lce_distill_workspace_bytes(ctypes.byref(_prob(**dims, monitoring=True)), K, 1, ctypes.byref(size)) == L.LCE_EINVAL_ARG
    assert lib.lce_distill_workspace_bytes(ctypes.byref(_prob(**dims, z_reg=1e-4)), K, 1, ctypes.byref(size)) == L.LCE_EINVAL_ARG


def _top(lib, logits=PTR, dtype=BF16, rows=4, cols=100, ld=100, k=8, values=PTR, index=PTR, lse=PTR):
    return lib.lce_top_logits(logits, dtype, rows, cols, ld, k, values, index, lse, None)


LOGITS_SHAPES = (dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=(1 << 30) + 1))
LOGITS_ARGS = (dict(logits=None), dict(ld=-1), dict(logits=PTR + 1), dict(logits=PTR + 2, dtype=F32))


def test_top_logits_refusals(lib):
    L = _codes()
    for bad in (*LOGITS_SHAPES, dict(k=0), dict(k=-1), dict(k=101), dict(k=1025, cols=5000)):
        assert _top(lib, **bad) == L.LCE_EINVAL_SHAPE, bad
    for bad in (*LOGITS_ARGS, dict(values=None), dict(index=None)):
        assert _top(lib, **bad) == L.LCE_EINVAL_ARG, bad
    assert _top(lib, dtype=7) == L.LCE_EINVAL_DTYPE
    assert _top(lib, rows=0, logits=None, values=None, index=None, lse=None) == L.LCE_OK


def _sample(lib, logits=PTR, dtype=BF16, rows=4, cols=100, ld=100, u=PTR, token=PTR, settings=True, **s):
    from linear_cross_entropy_loss_amd import _lib

    d = dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, temperature_rows=None, top_p_rows=None, min_p_rows=None, top_k_rows=None)
    d.update(s)
    arg = ctypes.byref(_lib.LceSampling(**d)) if settings else None
    return lib.lce_sample(logits, dtype, rows, cols, ld, u, arg, token, None)


def test_sample_refusals(lib):
    L = _codes()
    nan, inf = float("nan"), float("inf")
    for bad in LOGITS_SHAPES:
        assert _sample(lib, **bad) == L.LCE_EINVAL_SHAPE, bad
    for bad in (*LOGITS_ARGS, dict(u=None), dict(token=None), dict(settings=False), dict(temperature=-1.0), dict(temperature=inf),
                dict(temperature=nan), dict(top_p=0.0), dict(top_p=-0.5), dict(top_p=1.5), dict(top_p=nan), dict(min_p=-0.1),
                dict(min_p=1.1), dict(min_p=nan), dict(top_k=-1)):
        assert _sample(lib, **bad) == L.LCE_EINVAL_ARG, bad
    assert _sample(lib, dtype=-1) == L.LCE_EINVAL_DTYPE
    # no rows: the settings are looked at all the same, the tensors are not
    none = dict(rows=0, logits=None, u=None, token=None)
    assert _sample(lib, **none) == L.LCE_OK
    assert _sample(lib, **none, top_p=2.0) == L.LCE_EINVAL_ARG
    # numbers in whose place a row's are taken are not looked at
    assert _sample(lib, **none, temperature=nan, top_p=nan, min_p=nan, top_k=-1, temperature_rows=PTR, top_p_rows=PTR, min_p_rows=PTR,
                   top_k_rows=PTR) == L.LCE_OK


def test_python_has_no_cpu_path():
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss, linear_distillation, sample_logits, top_logits

    z, index = torch.randn(4, 10), torch.zeros(4, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        top_logits(z, 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sample_logits(z, torch.rand(4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_distillation(torch.randn(4, 8), torch.randn(8, 10), index, z[:, :3])
    with pytest.raises(RuntimeError, match="no CPU path"):
        LinearCrossEntropyLoss(8, 10).distill(torch.randn(4, 8), index, z[:, :3])


@pytest.mark.parametrize("k", [0, -1, 11, 1025])
def test_python_refuses_k_before_all_else(k):
    from linear_cross_entropy_loss_amd import top_logits

    with pytest.raises(ValueError, match="k must be in 1"):
        top_logits(torch.randn(4, 10), k)
    with pytest.raises(ValueError, match="k must be in 1"):
        top_logits(torch.tensor(1.0), 1)
