"""Logits of given tokens where calls go wrong easily: rows that are not wanted, more than one slab, float32 in its less usual forms, and
what is refused.  Inputs, oracle and tolerances are those of test_token_logits_gpu.py."""
import ctypes
import math

import pytest
import torch

from test_token_logits_gpu import BF16, F16, F32, IGNORE, check, make, oracle

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]


@pytest.fixture(params=["always", "never"])
def packing(request):
    from linear_cross_entropy_loss_amd import _lib, ops

    token = ops.pack_rows.set(_lib.PACK_ALWAYS if request.param == "always" else _lib.PACK_NEVER)
    yield request.param
    ops.pack_rows.reset(token)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("N, H, V", [(100, 64, 500), (100, 200, 500), (130, 33, 515), (2100, 320, 20001)])
def test_upstream_gradients_of_ignored_rows_are_not_looked_at(N, H, V, dtype, packing):
    from linear_cross_entropy_loss_amd import linear_token_logits

    print(f"token_logits {N} {H} {V} {dtype} packing {packing}", flush=True)
    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(N, H, V, dtype, seed=7, drop=0.5))
    gone = tokens == IGNORE
    got = []
    for fill in (0.0, math.nan, math.inf, -math.inf, 3e38):
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = linear_token_logits(xs, ws, tokens, IGNORE)
        got.append(torch.autograd.grad(out, (xs, ws), (g_logits.masked_fill(gone, fill), g_lse.masked_fill(gone, fill))))
    assert (got[0][0][gone] == 0).all() and got[0][1].isfinite().all()
    for dx, dw in got[1:]:
        assert torch.equal(dx, got[0][0]) and torch.equal(dw, got[0][1])


def test_objective_that_is_nan_on_padding():
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss

    module = LinearCrossEntropyLoss(200, 700, device="cuda", dtype=BF16, ignore_index=-1)
    x = torch.randn(4, 30, 200, device="cuda", dtype=BF16, requires_grad=True)
    tokens = torch.randint(0, 700, (4, 30), device="cuda")
    tokens[:, 20:] = -1
    advantage = torch.randn(4, 30, device="cuda")
    advantage[:, 20:] = math.nan
    module.log_probs(x, tokens).backward(advantage.nan_to_num(0.0))
    want = x.grad.clone(), module.weight.grad.clone()
    x.grad = module.weight.grad = None
    module.log_probs(x, tokens).backward(advantage)
    assert torch.equal(x.grad, want[0]) and torch.equal(module.weight.grad, want[1])


def test_a_launch_that_fails_names_its_error():
    """The library's own functions stand aside for two that return LCE_EHIP, as a failed launch does."""
    from linear_cross_entropy_loss_amd import _lib, linear_token_logits

    host, lib = _lib.host(), _lib.load()
    table = {name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _lib.EXPORTS}
    vp, i64, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    forward = ctypes.CFUNCTYPE(ctypes.c_int, vp, vp, vp, vp, i64, vp, vp, vp, vp, size, vp)(lambda *_: _lib.LCE_EHIP)
    backward = ctypes.CFUNCTYPE(ctypes.c_int, *[vp] * 12, size, vp)(lambda *_: _lib.LCE_EHIP)
    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(40, 64, 300, BF16, seed=9))
    x.requires_grad_(True)
    text = f"linear_token_logits: {lib.lce_strerror(_lib.LCE_EHIP).decode()}: "
    out = linear_token_logits(x, w, tokens, IGNORE)
    try:
        host.bind({**table, "lce_token_logits": ctypes.cast(forward, vp).value, "lce_token_logits_backward": ctypes.cast(backward, vp).value})
        with pytest.raises(RuntimeError) as failed:
            linear_token_logits(x, w, tokens, IGNORE)
        assert str(failed.value).startswith(text)
        with pytest.raises(RuntimeError) as failed:
            torch.autograd.grad(out, x, (g_logits, g_lse), retain_graph=True)
        assert str(failed.value).startswith(text)
    finally:
        host.bind(table)
    torch.autograd.grad(out, x, (g_logits, g_lse))
