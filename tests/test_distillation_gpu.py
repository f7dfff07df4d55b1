"""Distillation from a teacher's top logits against its definition in 64 bits.

Tolerances.  A 16-bit gradient is a sum of products with a dz that was rounded to the type (once, or twice where the logits are
computed once: eps each, half a step of a relative eps), rounded once itself: at most 3 * eps / 2 of the 2-norm, bf16 1.2e-2,
fp16 1.5e-3 (products and their fp32 sums add 2^-24 * sqrt(terms), which is below a hundredth of that).  With the roundings of
many terms independent the 2-norm sees about a third; the full bound is asserted.  fp32 operands are pairs of bf16 with 16 bits of
mantissa: 3 * 2^-16 each side, two sides: 1e-4.  An element by itself: the largest entry's 2^-6 (bf16), 2^-9 (fp16), 2^-12 (fp32).
The loss is a mean of sums of fp32 terms of magnitude |z| <= 64: 64 * 2^-22 each, before it shrinks by averaging."""
import math

import pytest
import torch

from helpers import rel_errors

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -14}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(N, H, V, K, dtype, seed, empty=0.0, short=0.0, twice=False, w_dtype=None, t_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    w = (torch.randn(H, V, generator=g) / math.sqrt(H)).to(w_dtype or dtype)
    if twice:
        index = torch.randint(0, max(1, V // 2), (N, K), generator=g)
    else:
        index = torch.rand(N, V, generator=g).argsort(1)[:, :K] if N * V < 1 << 25 else (
            torch.randint(0, V // K, (N, K), generator=g) + torch.arange(K) * (V // K))
    logits = (4.0 * torch.randn(N, K, generator=g)).to(t_dtype)
    index[torch.rand(N, K, generator=g) < short] = -1
    index[torch.rand(N, generator=g) < empty] = -5
    return x, w, index, logits


def oracle(x, w, index, logits, T, scale, w_as=None):
    """Loss, dx, dW in 64 bits; the weight rounded to the activations' type first, as the operator documents it."""
    x, w = x.double(), w.to(w_as or w.dtype).double()
    V, c = w.shape[1], scale / T
    there = (index >= 0) & (logits != -math.inf)
    kept = there.any(1)
    q = torch.zeros(x.shape[0], V, dtype=torch.float64)
    t = torch.where(there, logits.double() / T, -math.inf)
    t = torch.where(there, torch.exp(t - torch.where(kept, t.amax(1), 0.0)[:, None]), 0.0)
    t = t / torch.where(kept, t.sum(1), 1.0)[:, None]
    q.scatter_add_(1, index.clamp(min=0), t)
    z = x @ w * c
    p = torch.log_softmax(z, 1)
    R = kept.sum()
    loss = ((torch.special.xlogy(q, q) - q * p).sum(1) * kept).sum() / R
    dz = (p.exp() - q) * (kept[:, None] * c / R) if R > 0 else torch.zeros_like(q)
    return loss, dz @ w.t(), x.t() @ dz


def check(inputs, T=1.0, scale=1.0, tied=False, n_chunk=4096, up=1.0, run=None):
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = inputs
    print(f"distill N={tuple(x.shape)} W={tuple(w.shape)} K={index.shape[-1]} {x.dtype} {w.dtype} tied={tied} T={T}", flush=True)
    ref_loss, ref_dx, ref_dw = oracle(x, w, index, logits, T, scale, x.dtype if w.dtype != x.dtype else None)
    xg = x.cuda().requires_grad_(True)
    wg = (w.t().contiguous() if tied else w).cuda().requires_grad_(True)
    call = run or linear_distillation
    loss = call(xg, wg.t() if tied else wg, index.cuda(), logits.cuda(), T, scale, n_chunk)
    (loss * up).backward()
    torch.cuda.synchronize()
    got_dw = wg.grad.t() if tied else wg.grad
    kept = ((index >= 0) & (logits != -math.inf)).any(1)
    if not kept.any():
        assert loss.isnan() and not xg.grad.any() and not wg.grad.any()
        return
    eps = EPS[x.dtype]
    terms = max(1.0, ref_loss.item())
    assert abs(loss.item() - ref_loss.item()) <= 64 * 2.0 ** -22 * terms + (1e-4 if x.dtype == F32 else 0)
    for got, ref in ((xg.grad, ref_dx * up), (got_dw, ref_dw * up)):
        assert torch.isfinite(got).all()
        if not ref.any():
            # (a vocabulary of one column: softmax - q = 0 up to exp of the difference of two fp32 logits below 8, 2^-20, of which
            # x and W entries below 8 make gradients)
            assert got.abs().max().item() <= up * 2.0 ** -17
            continue
        worst, norm = rel_errors(got, ref)
        assert norm <= 1.5 * eps and worst <= 2 * eps, (worst, norm)
    assert not xg.grad[~kept.cuda()].any()
    return loss, xg.grad, got_dw


SHAPES = [(1, 8, 1, 1), (1, 64, 2, 2), (3, 17, 33, 5), (64, 256, 1000, 8), (257, 129, 511, 64), (300, 500, 1007, 65), (128, 2048, 4096, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,H,V,K", SHAPES)
def test_small_shapes(N, H, V, K, dtype):
    check(make(N, H, V, K, dtype, seed=N + K, empty=0.2 if N > 2 else 0.0, short=0.2 if K > 2 else 0.0), up=1.0 if dtype != F16 else 512.0)


@pytest.mark.parametrize("dtype,w_dtype,tied", [(BF16, None, True), (F16, None, True), (BF16, F32, False), (F16, F32, False), (BF16, F32, True)])
def test_weight_forms(dtype, w_dtype, tied):
    x, w, index, logits = make(700, 264, 1999, 31, dtype, seed=5, empty=0.1, short=0.1, w_dtype=w_dtype)
    check((x, w, index, logits), T=1.7, scale=0.6, tied=tied, up=1.0 if dtype != F16 else 512.0)


@pytest.mark.parametrize("mode", ["one_pass", "two_pass"])
@pytest.mark.parametrize("pack", [1, 2])
@pytest.mark.parametrize("dtype,n_chunk", [(BF16, 512), (F16, 4096), (F32, 2048)])
def test_routes(mode, pack, dtype, n_chunk):
    """Either route, tokens packed away or not, one chunk or several (a bound that leaves room for a part of the rows)."""
    from linear_cross_entropy_loss_amd import ops

    routes = ops.one_pass.set("always" if mode == "one_pass" else False), ops.pack_rows.set(pack)
    try:
        check(make(1300, 256, 4100, 40, dtype, seed=11, empty=0.3, short=0.3), n_chunk=n_chunk, up=1.0 if dtype != F16 else 512.0)
    finally:
        ops.one_pass.reset(routes[0])
        ops.pack_rows.reset(routes[1])


@pytest.mark.parametrize("K", [2, 64, 100, 256, 1024])
def test_columns_named_twice(K):
    check(make(70, 64, max(3, K // 2), K, BF16, seed=K, twice=True, short=0.1))


@pytest.mark.parametrize("K", [1, 63, 64, 65, 129, 257, 513, 1023, 1024])
def test_numbers_of_targets(K):
    check(make(37, 64, 2048, K, BF16, seed=K, short=0.05 if K > 1 else 0.0), T=0.5)


@pytest.mark.parametrize("t_dtype", [BF16, F16, F32])
def test_absent_entries_hold_anything(t_dtype):
    """NaN, infinities and the type's lowest value behind a negative index; -inf and the lowest value at a column."""
    x, w, index, logits = make(64, 128, 512, 6, BF16, seed=2, t_dtype=t_dtype)
    index[:, 1] = -1
    logits[::4, 1], logits[1::4, 1], logits[2::4, 1], logits[3::4, 1] = math.nan, math.inf, -math.inf, torch.finfo(t_dtype).min
    logits[:32, 3] = -math.inf
    logits[32:, 4] = torch.finfo(t_dtype).min
    logits[5] = -math.inf  # a row that is left with nothing
    index[6] = -1
    check((x, w, index, logits))


def test_no_row_has_a_target():
    x, w, index, logits = make(40, 64, 300, 4, BF16, seed=3)
    index[:] = -1
    check((x, w, index, logits))


@pytest.mark.parametrize("what", ["index", "nan", "inf"])
def test_a_bad_entry_makes_the_loss_nan(what):
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(40, 64, 300, 4, BF16, seed=3)
    if what == "index":
        index[7, 2] = 300
    else:
        logits[7, 2] = math.nan if what == "nan" else math.inf
    assert linear_distillation(x.cuda(), w.cuda(), index.cuda(), logits.cuda()).isnan()


def test_one_target_is_a_label():
    """K = 1: the loss and the gradients of cross entropy, whatever the teacher's logit."""
    from linear_cross_entropy_loss_amd import linear_cross_entropy, linear_distillation

    x, w, index, logits = make(500, 256, 1000, 1, BF16, seed=9, empty=0.2)
    a, b = x.cuda().requires_grad_(True), x.cuda().requires_grad_(True)
    wa, wb = w.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = linear_distillation(a, wa, index.cuda(), logits.cuda())
    ref = linear_cross_entropy(b, index[:, 0].cuda().clamp(min=-1), wb, ignore_index=-1)[0]
    loss.backward()
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 64 * 2.0 ** -22
    # (the same staged dz but where fp32 sums of the target logit in another order round to the other side)
    assert rel_errors(a.grad, b.grad)[1] <= 2.0 ** -8 and rel_errors(wa.grad, wb.grad)[1] <= 2.0 ** -8


def test_strides_shapes_and_leading_dimensions():
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss

    x, w, index, logits = make(60, 96, 700, 7, BF16, seed=4, empty=0.2)
    wide_index = torch.full((60, 20), 10 ** 12)
    wide_index[:, 3:10] = index
    wide_logits = torch.full((7, 60), math.nan)
    wide_logits.copy_(logits.t())
    module = LinearCrossEntropyLoss(96, 700, device="cuda", dtype=BF16, logit_scale=0.5)

    def run(xg, wg, i, l, T, scale, n_chunk):
        module.weight = torch.nn.Parameter(wg.detach())
        module.weight.grad = None
        loss = module.distill(xg.reshape(3, 20, 96), wide_index.cuda()[:, 3:10].reshape(3, 20, 7), wide_logits.cuda().t().reshape(3, 20, 7), T)
        loss.register_hook(lambda g: None)
        loss.backward()
        wg.grad = module.weight.grad
        xg.grad, kept = None, xg.grad
        return kept, loss

    ref_loss, ref_dx, ref_dw = oracle(x, w, index, logits, 1.3, 0.5)
    xg, wg = x.cuda().requires_grad_(True), w.cuda()
    dx, loss = run(xg, wg, index, logits, 1.3, 0.5, 4096)
    assert abs(loss.item() - ref_loss.item()) <= 64 * 2.0 ** -22
    assert rel_errors(dx, ref_dx)[1] <= 1.5 * EPS[BF16] and rel_errors(wg.grad, ref_dw)[1] <= 1.5 * EPS[BF16]


def test_teacher_of_all_rows_broadcast():
    """One teacher row for all tokens, expanded; and one hidden state expanded over the tokens, whose gradient is the sum."""
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(33, 64, 200, 5, F32, seed=8)
    one_x = x[:1].cuda().requires_grad_(True)
    wg = w.cuda().requires_grad_(True)
    loss = linear_distillation(one_x.expand(33, 64), wg, index[:1].cuda().expand(33, 5), logits[:1].cuda().expand(33, 5))
    loss.backward()
    ref_loss, ref_dx, ref_dw = oracle(x[:1], w, index[:1], logits[:1], 1.0, 1.0)
    assert abs(loss.item() - ref_loss.item()) <= 1e-4
    assert rel_errors(one_x.grad, ref_dx)[1] <= 1e-4 and rel_errors(wg.grad, ref_dw)[1] <= 1e-4


def test_second_backward_over_the_same_graph():
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(300, 256, 1000, 12, F16, seed=6, empty=0.1)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = linear_distillation(xg, wg, index.cuda(), logits.cuda())
    first = torch.autograd.grad(loss, (xg, wg), torch.tensor(256.0, device="cuda"), retain_graph=True)
    first = [t.clone() for t in first]
    again = torch.autograd.grad(loss, (xg, wg), torch.tensor(256.0, device="cuda"))
    for a, b in zip(first, again):
        assert rel_errors(a, b)[1] <= 2.0 ** -10  # (a power of two multiplied in before or after the rounding)
    only = linear_distillation(xg, w.cuda(), index.cuda(), logits.cuda())
    assert torch.equal(torch.autograd.grad(only, xg, torch.tensor(256.0, device="cuda"))[0], first[0])


def test_gradient_against_differences():
    """fp32: the loss along a direction, central differences."""
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(50, 64, 300, 6, F32, seed=12, empty=0.1)
    x, w, index, logits = x.cuda(), w.cuda(), index.cuda(), logits.cuda()
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_distillation(xg, wg, index, logits, 1.5), (xg, wg))
    # along the gradient itself, h = 0.05 of the parameters' size: differences of order 1e-2 of a loss known to 1e-5
    for t, d, at in ((x, dx, 0), (w, dw, 1)):
        step = d * (0.05 * t.norm() / d.norm())
        hi = linear_distillation(*((x + step, w) if at == 0 else (x, w + step)), index, logits, 1.5)
        lo = linear_distillation(*((x - step, w) if at == 0 else (x, w - step)), index, logits, 1.5)
        along = (d * step).sum()
        assert abs((hi - lo).item() / 2 - along.item()) <= 0.02 * along.item()


def test_autocast_and_no_grad():
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(100, 64, 300, 6, F32, seed=13)
    with torch.autocast("cuda", dtype=BF16):
        xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
        loss = linear_distillation(xg, wg, index.cuda(), logits.cuda())
    loss.backward()
    ref_loss, ref_dx, ref_dw = oracle(x.to(BF16), w, index, logits, 1.0, 1.0, BF16)
    assert xg.grad.dtype == F32 and wg.grad.dtype == F32
    assert rel_errors(xg.grad, ref_dx)[1] <= 1.5 * EPS[BF16] and rel_errors(wg.grad, ref_dw)[1] <= 1.5 * EPS[BF16]
    with torch.no_grad():
        free = linear_distillation(xg, wg, index.cuda(), logits.cuda())
    assert not free.requires_grad


def test_another_stream():
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = (t.cuda() for t in make(300, 256, 2000, 12, BF16, seed=14))
    ref = linear_distillation(x, w, index, logits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = linear_distillation(x, w, index, logits)
    side.synchronize()
    assert torch.equal(ref, got)


def test_captured_and_replayed():
    """Loss and gradients of new inputs in the same buffers, replayed with eager work in between, against eager calls."""
    from linear_cross_entropy_loss_amd import linear_distillation

    N, H, V, K = 512, 256, 3000, 16
    static = [t.cuda() for t in make(N, H, V, K, BF16, seed=15, empty=0.1, short=0.1)]
    x, w = static[0].requires_grad_(True), static[1].requires_grad_(True)

    def step():
        loss = linear_distillation(x, w, static[2], static[3], 1.2)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(16, 20):
        new = [t.cuda() for t in make(N, H, V, K, BF16, seed=seed, empty=0.1, short=0.1)]
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
        ref = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


def test_compiled():
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(300, 128, 1000, 9, BF16, seed=21, empty=0.1)
    run = torch.compile(lambda a, b, i, l: 2.0 * linear_distillation(a * 1.0, b, i, l, 1.1), fullgraph=True)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = run(xg, wg, index.cuda(), logits.cuda())
    loss.backward()
    ref_loss, ref_dx, ref_dw = oracle(x, w, index, logits, 1.1, 1.0)
    assert abs(loss.item() - 2 * ref_loss.item()) <= 2 * 64 * 2.0 ** -22
    assert rel_errors(xg.grad, 2 * ref_dx)[1] <= 1.5 * EPS[BF16] and rel_errors(wg.grad, 2 * ref_dw)[1] <= 1.5 * EPS[BF16]


@pytest.mark.pack_auto
@pytest.mark.parametrize("N,H,V,K,dtype", [(4096, 768, 50257, 32, BF16), (2048, 1024, 32000, 64, F16)])
def test_model_sizes(N, H, V, K, dtype):
    """Sizes of models, both weights' layouts; the oracle runs on the GPU in 64 bits."""
    from linear_cross_entropy_loss_amd import linear_distillation

    x, w, index, logits = make(N, H, V, K, dtype, seed=31, empty=0.1, short=0.2)
    up = 512.0 if dtype == F16 else 1.0
    for tied in (False, True):
        xg = x.cuda().requires_grad_(True)
        wg = (w.t().contiguous() if tied else w).cuda().requires_grad_(True)
        loss = linear_distillation(xg, wg.t() if tied else wg, index.cuda(), logits.cuda(), 2.0)
        (loss * up).backward()
        xd, wd = x.cuda().double(), w.cuda().double()
        there = (index >= 0).cuda()
        kept = there.any(1)
        t = torch.softmax(torch.where(there, logits.cuda().double() / 2.0, -math.inf), 1)
        t = torch.where(kept[:, None], t, 0.0)
        q = torch.zeros(N, V, dtype=torch.float64, device="cuda").scatter_add_(1, index.cuda().clamp(min=0), t)
        p = torch.log_softmax(xd @ wd / 2.0, 1)
        ref = (((torch.special.xlogy(q, q) - q * p).sum(1)) * kept).sum() / kept.sum()
        dz = (p.exp() - q) * kept[:, None] * (0.5 * up / kept.sum())
        assert abs(loss.item() - ref.item()) <= 64 * 2.0 ** -22 * max(1.0, ref.item())
        assert rel_errors(xg.grad, dz @ wd.t())[1] <= 1.5 * EPS[dtype]
        assert rel_errors(wg.grad.t() if tied else wg.grad, xd.t() @ dz)[1] <= 1.5 * EPS[dtype]


@pytest.mark.parametrize("dtype,w_dtype,tied,shape", [(BF16, None, False, (300, 256, 1000)), (F16, None, True, (100, 64, 511)),
                                                      (BF16, F32, False, (65, 100, 1001)), (F32, None, False, (40, 130, 700))])
def test_host_path_gives_the_same_bits(dtype, w_dtype, tied, shape):
    """The C++ host path against the Python one, which a strided index takes."""
    from linear_cross_entropy_loss_amd import _lib, distillation, linear_distillation

    N, H, V = shape
    x, w, index, logits = make(N, H, V, 9, dtype, seed=N, empty=0.1, short=0.1, w_dtype=w_dtype)
    w = (w.t().contiguous().t() if tied else w).cuda()
    wide = torch.zeros(N, 12, dtype=torch.int64, device="cuda")
    wide[:, :9] = index.cuda()
    taken = []
    native = distillation._native
    distillation._native = lambda *a: taken.append(native(*a)) or taken[-1]
    try:
        results = []
        for i in (index.cuda(), index.cuda(), wide[:, :9]):  # (the first call may have a warning to give)
            xg, wg = x.cuda().requires_grad_(True), w.detach().requires_grad_(True)
            loss = linear_distillation(xg, wg, i, logits.cuda(), 1.5, 0.7)
            results.append((loss.detach(), *torch.autograd.grad(loss, (xg, wg))))
    finally:
        distillation._native = native
    assert taken[1] is not None and taken[2] is None
    for a, b in zip(results[1], results[2]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("w_vh", [False, True])
def test_sorted_and_unsorted_entries(w_vh):
    """Both sides of the rule by which the targets' logits are formed, columns that many rows name, small numbers of fp16."""
    for N, K, H in ((2000, 40, 72), (64, 10, 72), (600, 130, 100)):
        x, w, index, logits = make(N, H, 900, K, F16, seed=K)
        index[:, 0] = 17  # a column of every row
        index[:, 1:][index[:, 1:] == 17] = 18
        w[:, ::3] *= 2.0 ** -12  # subnormal numbers of the type among them
        check((x, w, index, logits), tied=w_vh and H % 8 == 0, up=512.0)


@pytest.mark.pack_auto
def test_refusals():
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss, linear_distillation

    x, w, index, logits = (t.cuda() for t in make(6, 16, 40, 5, BF16, seed=40))
    for bad in ((x, w[:8], index, logits), (x, w[0], index, logits), (x, w, index[:5], logits[:5]), (x, w, index, logits[:, :4]),
                (x, w, index.int(), logits), (x, w, index, logits.double()), (x, w, index, logits.long()), (x, w, index[:, :0], logits[:, :0]),
                (x, w.half(), index, logits), (x.double(), w.double(), index, logits), (x[:0], w, index[:0], logits[:0]),
                (x, w, index.repeat(1, 205)[:, :1025], logits.repeat(1, 205)[:, :1025])):
        with pytest.raises(ValueError):
            linear_distillation(*bad)
    for bad in ((x.cpu(), w, index, logits), (x, w.cpu(), index, logits), (x, w, index.cpu(), logits), (x, w, index, logits.cpu())):
        with pytest.raises(RuntimeError, match="no CPU path"):
            linear_distillation(*bad)
    for numbers in ({"temperature": 0.0}, {"temperature": -1.0}, {"temperature": math.inf}, {"temperature": math.nan}, {"temperature": 1e-60},
                    {"logit_scale": 0.0}, {"logit_scale": math.inf}, {"logit_scale": math.nan}, {"logit_scale": 1e30, "temperature": 1e-30},
                    {"N_chunk_size": 0}, {"N_chunk_size": -4}):
        with pytest.raises(ValueError):
            linear_distillation(x, w, index, logits, **numbers)
    module = LinearCrossEntropyLoss(16, 40, device="cuda", dtype=BF16)
    with pytest.raises(ValueError):
        module.distill(x, index.int(), logits)


def test_two_streams_at_once():
    from linear_cross_entropy_loss_amd import linear_distillation

    sets = [[t.cuda() for t in make(700, 256, 5000, 24, BF16, seed=41 + i, empty=0.2, twice=True)] for i in range(2)]

    def call(x, w, index, logits):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_distillation(x, w, index, logits, 1.5)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    ref = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = call(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(ref, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.pack_auto
def test_opcheck():
    from linear_cross_entropy_loss_amd import ops  # noqa: F401 (registers the operators)
    from linear_cross_entropy_loss_amd import distillation  # noqa: F401

    x, w, index, logits = (t.cuda() for t in make(10, 32, 100, 5, BF16, seed=43))
    for needs in ((True, True), (False, True), (True, False), (False, False)):
        torch.library.opcheck(torch.ops.lce_amd.distill.default, (x, w, index, logits, 1.5, 0.7, 4096, *needs),
                              test_utils=("test_schema", "test_faketensor"))


def test_beside_the_loss_on_labels():
    """Both losses on the same hidden states and weight, weighed and added, as a step would: the gradients add up."""
    from linear_cross_entropy_loss_amd import linear_cross_entropy, linear_distillation

    x, w, index, logits = (t.cuda() for t in make(200, 128, 1500, 10, BF16, seed=44, empty=0.3))
    y = torch.randint(0, 1500, (200,), device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    T = 2.0
    labels, teacher = lambda: 0.3 * linear_cross_entropy(x, y, w)[0], lambda: T * T * linear_distillation(x, w, index, logits, T)
    parts = [torch.autograd.grad(loss(), (x, w)) for loss in (labels, teacher)]
    both = torch.autograd.grad(labels() + teacher(), (x, w))
    for got, a, b in zip(both, *parts):
        assert torch.equal(got, a + b)


@pytest.mark.pack_auto
@pytest.mark.parametrize("V", [1 << 20, (1 << 20) + 8])
def test_as_many_column_groups_as_are_sorted(V):
    """A vocabulary with the most groups of columns that the sort of the entries has room for, and one more; oracle on the GPU."""
    from linear_cross_entropy_loss_amd import linear_distillation

    print(f"distill V={V}", flush=True)
    N, H, K = 64, 64, 1024
    g = torch.Generator(device="cuda").manual_seed(45)
    x = torch.randn(N, H, generator=g, device="cuda").to(BF16).requires_grad_(True)
    w = (torch.randn(H, V, generator=g, device="cuda") / 8).to(BF16).requires_grad_(True)
    index = torch.randint(0, V, (N, K), generator=g, device="cuda")
    index[:, 0] = V - 1
    logits = 4.0 * torch.randn(N, K, generator=g, device="cuda")
    loss = linear_distillation(x, w, index, logits)
    loss.backward()
    q = torch.zeros(N, V, dtype=torch.float64, device="cuda").scatter_add_(1, index, torch.softmax(logits.double(), 1))
    p = torch.log_softmax(x.detach().double() @ w.detach().double(), 1)
    ref = ((torch.special.xlogy(q, q) - q * p).sum(1)).mean()
    dz = (p.exp() - q) / N
    assert abs(loss.item() - ref.item()) <= 64 * 2.0 ** -22 * max(1.0, ref.item())
    assert rel_errors(x.grad, dz @ w.detach().double().t())[1] <= 1.5 * EPS[BF16]
    assert rel_errors(w.grad, x.detach().double().t() @ dz)[1] <= 1.5 * EPS[BF16]


@pytest.mark.pack_auto
@pytest.mark.parametrize("N,K", [(40, 6), (2048, 64)])
def test_columns_beyond_the_weight_are_not_read(N, K):
    """lce_distill given columns that lce_soft_targets would not give: they are left alone, by either way to the logits, and the labels
    of those rows make the loss NaN; without them in the labels the other rows' gradients are what they are without such entries."""
    from linear_cross_entropy_loss_amd import distillation, ops

    H, V = 64, 1003
    x, w, index, logits = (t.cuda() for t in make(N, H, V, K, BF16, seed=46))
    x2, w2, layout = distillation._views(x, w)
    columns, q, y = distillation._targets(index, logits, V, 1.0)
    cfg = (1.0, 4096, ops._pack_mode(), ops._route_mode())
    odd, q_odd = columns.clone(), q.clone()
    odd[::3, 1] = torch.tensor([V, V + 63, V + 64, 2 ** 31 - 1], dtype=torch.int32, device="cuda").repeat(N)[: odd[::3].shape[0]]
    plain, q_plain = columns.clone(), q.clone()
    plain[::3, 1] = -1
    q_odd[::3, 1] = q_plain[::3, 1] = 0.0
    print(f"columns beyond N={N} K={K}", flush=True)
    got = distillation._run(x2, w2, layout, (odd, q_odd, y), *cfg, True, True, None)
    ref = distillation._run(x2, w2, layout, (plain, q_plain, y), *cfg, True, True, None)
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and torch.isfinite(got[0])
    y = y.clone()
    y[0] = V
    assert distillation._run(x2, w2, layout, (odd, q_odd, y), *cfg, True, True, None)[0].isnan()
