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


@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_slabs_of_other_types(dtype, packing):
    from linear_cross_entropy_loss_amd import _lib
    from linear_cross_entropy_loss_amd.token_logits import _problem

    N, H, V, n_chunk = 3000, 256, 8192, 512
    inputs = make(N, H, V, dtype, seed=3)
    prob = _problem(inputs[0], inputs[1], _lib.W_HV, V, IGNORE, 1.0, n_chunk, 0)
    # (less than a dz of all columns takes: there is more than one slab)
    assert _lib.token_logits_workspace_bytes(prob, True) < N * V * dtype.itemsize
    check(inputs, n_chunk=n_chunk, scale=0.7)


@pytest.mark.parametrize("N, H, V", [(1, 64, 1000), (40, 64, 999), (130, 33, 515), (2100, 320, 20000)])
def test_float32_tied_weight(N, H, V):
    check(make(N, H, V, F32, seed=9), tied=True)
    check(make(N, H, V, F32, seed=9, pieces=2), tied=True, first=V, size=2 * V)


@pytest.mark.parametrize("rows", [(), (1,), (1, 1, 1), (5, 1)])
def test_rows_of_any_shape(rows):
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(5, 72, 300, BF16, seed=2, drop=0.0))
    n = math.prod(rows)
    leaf = x[:n].reshape(*rows, 72).requires_grad_(True)
    logits, lse = linear_token_logits(leaf, w, tokens[:n].view(rows))
    assert logits.shape == lse.shape == torch.Size(rows)
    (dx,) = torch.autograd.grad((logits, lse), leaf, (g_logits[:n].view(rows), g_lse[:n].view(rows)))
    flat = x[:n].clone().requires_grad_(True)
    out = linear_token_logits(flat, w, tokens[:n])
    (want,) = torch.autograd.grad(out, flat, (g_logits[:n], g_lse[:n]))
    assert torch.equal(logits.view(-1), out[0]) and torch.equal(lse.view(-1), out[1])
    assert dx.shape == leaf.shape and torch.equal(dx.view(-1, 72), want)


@pytest.mark.parametrize("size, w_size", [(2.0 ** -44, 2.0 ** 42), (2.0 ** -70, 2.0 ** 68), (2.0 ** -100, 2.0 ** 98), (2.0 ** 60, 2.0 ** -62),
                                          (2.0 ** -60, 2.0 ** -20), (2.0 ** -20, 2.0 ** -60)])
def test_float32_numbers_of_any_size(size, w_size):
    """Pairs are off by 2^-23 of a number or, as the largest of a tensor is multiplied to at least 2^13 and the lower number of a pair is a
    multiple of 2^-24, by 2^-38 of the largest: in each number of x, which a logit has |w| times over and dW |dz| times, and in each of w."""
    from linear_cross_entropy_loss_amd import linear_token_logits

    N, H, V = 70, 136, 600
    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(N, H, V, F32, seed=21))
    x, w = (x * size).requires_grad_(True), (w * w_size).requires_grad_(True)
    print(f"token_logits float32 x of {size} w of {w_size}", flush=True)
    logits, lse = linear_token_logits(x, w, tokens, IGNORE)
    dx, dw = torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse))
    want, (mag, mag_dx, mag_dw, w_sum, x_sum) = oracle(x.detach(), w.detach(), tokens, g_logits, g_lse, 1.0, 0)
    xd, wd = x.detach().double().abs(), w.detach().double().abs()
    tol_z = ((H + 2) * 2.0 ** -24 + 2.0 ** -21) * mag + 2.0 ** -38 * (xd.max() * wd.sum(0).max() + wd.max() * xd.sum(1).max())
    assert ((logits.double() - want[0]).abs() <= tol_z).all()
    assert ((lse.double() - want[1]).abs() <= tol_z + 2.0 ** -18 * (1 + want[1].abs())).all()
    live = tokens != IGNORE
    up = float((g_logits.abs() + g_lse.abs())[live].max())
    p_off = 2.0 ** -15 + 4 * float(tol_z.max())  # (of a softmax: exponent and lse each off by tol_z; e^2t - 1 <= 4 t for t below 1/2)
    assert p_off < 2.0 ** -10
    # (dz has steps of 2^-38 of the largest upstream gradients, rounded up to a power of two; magnitudes of all dz: at most 2 of them a row)
    for g, r, m, terms, edge in ((dx, want[2], mag_dx, V, 2.0 ** -37 * up * w_sum[None, :] + 2.0 ** -38 * wd.max() * 2 * up),
                                 (dw, want[3], mag_dw, N, 2.0 ** -37 * up * x_sum[:, None] + 2.0 ** -38 * xd.max() * 2 * up * live.sum())):
        tol = (2.0 ** -21 + p_off + terms * 2.0 ** -24) * m + 2.0 ** -24 * r.abs() + edge
        assert ((g.double() - r).abs() <= tol).all(), float(((g.double() - r).abs() / tol).max())


def test_function_transforms_and_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwAD
    from torch.func import grad, jvp, vmap

    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, *_ = (t.cuda() for t in make(40, 64, 300, BF16, seed=9, drop=0.0))

    def total(x):
        logits, lse = linear_token_logits(x, w, tokens)
        return (logits - lse).sum()

    with pytest.raises(RuntimeError):
        grad(total)(x)
    with pytest.raises(RuntimeError):
        jvp(total, (x,), (x,))
    with pytest.raises(RuntimeError):
        vmap(lambda x: linear_token_logits(x[None], w, tokens[:1])[0])(x)
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        total(fwAD.make_dual(x, x))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("N, H, V", [(1, 200, 1000), (1, 64, 999), (16, 264, 3001), (64, 1000, 4097), (200, 2048, 5000)])
def test_float32_weight_under_few_rows(N, H, V, tied, dtype):
    check(make(N, H, V, dtype, seed=N, w_dtype=F32), tied=tied)


def test_captured_backward_of_many_tiles():
    """Packed rows and several slabs in a graph, replayed between eager steps of the same operator."""
    from linear_cross_entropy_loss_amd import linear_token_logits

    inputs = [t.cuda() for t in make(2100, 320, 20001, F32, seed=5, drop=0.4)]

    def step(x, w, tokens, g_logits, g_lse):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out = linear_token_logits(x, w, tokens, IGNORE, N_chunk_size=512)
        return tuple(t.detach() for t in out) + torch.autograd.grad(out, (x, w), (g_logits, g_lse))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*inputs)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*inputs)
    for seed in range(3):
        for t, fresh in zip(inputs, make(2100, 320, 20001, F32, seed=30 + seed, drop=0.3)):
            t.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(*inputs)))
