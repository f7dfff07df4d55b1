"""Logits and logsumexps of given tokens, and their gradients, against the definition in 64 bits.

Tolerances, from u = finfo.eps / 2, the half step of a rounding:
* a logit is a sum of H exact products of 16-bit numbers in fp32: H 2^-24 sum |x w| (H + 2 with the factor); float32 numbers are
  multiplied as pairs of 22 bits, which leaves out 2^-22 of a product and rounds two parts at 2^-23: 2^-21 sum |x w| more;
* a logsumexp has the largest of these errors, and that of exponents and logarithms of 20 bits: 2^-18 (1 + |lse|);
* a softmax p is off by the errors of z and lse together, at most 2^-15 of itself at these sizes; dz is rounded to the type (u; pairs
  2^-23), products of it are summed in fp32 (terms 2^-24), the sum is rounded once (u of the result).  An entry of a gradient is
  therefore off by at most (u + 2^-15 + terms 2^-24) times the sum of its products' magnitudes + u of itself (pairs: 2^-21 of that sum,
  for dz, the operand and the parts left out); float16's dz and that of pairs have steps of 2^-38 of the largest row's upstream gradients at the
  least, the row's own magnitude rounded up to a power of two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
IGNORE = -100


def make(N, H, V, dtype, seed, drop=0.2, pieces=1, w_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    w = (torch.randn(H, V, generator=g) / math.sqrt(H)).to(w_dtype or dtype)
    tokens = torch.randint(0, V * pieces, (N,), generator=g)
    tokens[torch.rand(N, generator=g) < drop] = IGNORE
    g_logits, g_lse = torch.randn(N, generator=g), torch.randn(N, generator=g)
    g_lse[torch.rand(N, generator=g) < 0.1] = 0.0
    return x, w, tokens, g_logits, g_lse


def oracle(x, w, tokens, g_logits, g_lse, scale, first):
    """(logits, lse, dx, dw) and the sums of magnitudes that bound the errors of each, on the GPU in 64 bits."""
    x, w = x.double(), w.to(x.dtype).double()
    rows = tokens != IGNORE
    z = x @ w * scale
    lse = torch.logsumexp(z, 1)
    at = tokens - first
    here = rows & (at >= 0) & (at < w.shape[1])
    at = at.clamp(0, w.shape[1] - 1)[:, None]
    logits = torch.where(here, z.gather(1, at)[:, 0], 0.0)
    dz = torch.softmax(z, 1) * torch.where(rows, g_lse.double(), 0.0)[:, None]
    size = dz.abs()
    one = torch.where(here, g_logits.double(), 0.0)[:, None]
    dz.scatter_add_(1, at, one)
    size.scatter_add_(1, at, one.abs())
    return (logits, torch.where(rows, lse, 0.0), scale * dz @ w.t(), scale * x.t() @ dz), (
        scale * (x.abs() @ w.abs()).amax(1), scale * size @ w.abs().t(), scale * x.abs().t() @ size, scale * w.abs().sum(1), scale * x.abs().sum(0))


def check(inputs, scale=1.0, tied=False, n_chunk=4096, first=0, size=None, up=1.0, run=None):
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in inputs)
    g_logits, g_lse = g_logits * up, g_lse * up
    print(f"token_logits x={tuple(x.shape)} W={tuple(w.shape)} {x.dtype} {w.dtype} tied={tied} chunk={n_chunk} first={first}", flush=True)
    x.requires_grad_(True)
    leaf = (w.t().contiguous() if tied else w).requires_grad_(True)
    At = leaf.t() if tied else leaf
    run = run or linear_token_logits
    logits, lse = run(x, At, tokens, ignore_index=IGNORE, logit_scale=scale, N_chunk_size=n_chunk, vocab_start=first, vocab_size=size)
    dx, dw = torch.autograd.grad((logits, lse), (x, leaf), (g_logits, g_lse))
    assert logits.dtype == lse.dtype == F32 and dx.dtype == x.dtype and dw.dtype == w.dtype and dw.shape == leaf.shape
    got = (logits, lse, dx, dw.t() if tied else dw)
    want, (mag, mag_dx, mag_dw, w_sum, x_sum) = oracle(x.detach(), w.detach(), tokens, g_logits, g_lse, scale, first)
    H, V, N = x.shape[1], w.shape[1], x.shape[0]
    pairs = x.dtype == F32
    tol_z = ((H + 2) * 2.0 ** -24 + (2.0 ** -21 if pairs else 0)) * mag
    assert ((got[0].double() - want[0]).abs() <= tol_z).all()
    assert ((got[1].double() - want[1]).abs() <= tol_z + 2.0 ** -18 * (1 + want[1].abs())).all()
    u = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -21}[x.dtype]
    u_dw = 2.0 ** -24 if w.dtype == F32 else u
    floor = 0.0
    if x.dtype != BF16:
        live = tokens != IGNORE
        floor = 2.0 ** -38 * 2 * float((g_logits.abs() + g_lse.abs())[live].max()) if live.any() else 0.0
    for g, r, m, terms, edge, u_out in ((got[2], want[2], mag_dx, V, floor * w_sum[None, :], u), (got[3], want[3], mag_dw, N, floor * x_sum[:, None], u_dw)):
        tol = (u + 2.0 ** -15 + terms * 2.0 ** -24) * m + u_out * r.abs() + edge + (2.0 ** -25 if g.dtype == F16 else 0.0)
        worst = ((g.double() - r).abs() / tol.clamp(min=1e-300)).max()
        assert ((g.double() - r).abs() <= tol).all(), float(worst)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("N, H, V", [(1, 8, 1), (1, 64, 1000), (3, 100, 257), (64, 256, 4096), (130, 33, 515), (300, 520, 2049),
                                     (257, 128, 512), (2, 1000, 50257), (700, 64, 3000)])
def test_sizes(N, H, V, dtype):
    check(make(N, H, V, dtype, seed=N + H + V))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("pack", ["always", "never"])
def test_persistent_tiles_and_packing(dtype, pack):
    from linear_cross_entropy_loss_amd import _lib, ops

    token = ops.pack_rows.set(_lib.PACK_ALWAYS if pack == "always" else _lib.PACK_NEVER)
    try:
        check(make(2100, 320, 20001, dtype, seed=5, drop=0.4), scale=0.7)
    finally:
        ops.pack_rows.reset(token)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("N, H, V", [(40, 64, 999), (2100, 320, 20000)])
def test_tied_weight(N, H, V, dtype):
    check(make(N, H, V, dtype, seed=9), tied=True)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_float32_weight(dtype):
    check(make(600, 264, 3001, dtype, seed=2, w_dtype=F32))


def test_slabs_within_a_tight_bound():
    check(make(3000, 256, 8192, BF16, seed=3), n_chunk=512)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_pieces_of_a_vocabulary_make_the_whole(dtype):
    from linear_cross_entropy_loss_amd import linear_token_logits

    N, H, V, pieces = 200, 136, 700, 3
    x, w, tokens, g_logits, g_lse = make(N, H, V * pieces, dtype, seed=4)
    for p in range(pieces):
        check((x, w[:, p * V:(p + 1) * V].contiguous(), tokens, g_logits, g_lse), first=p * V, size=V * pieces)
    x, w, tokens = x.cuda(), w.cuda(), tokens.cuda()
    parts = [linear_token_logits(x, w[:, p * V:(p + 1) * V].contiguous(), tokens, IGNORE, vocab_start=p * V, vocab_size=V * pieces)
             for p in range(pieces)]
    logits, lse = linear_token_logits(x, w, tokens, IGNORE)
    live = tokens != IGNORE
    # (the same products in the same order; the joined lse is rounded at 24 bits a few times more)
    assert torch.equal(sum(a for a, _ in parts), logits)
    joined = torch.logsumexp(torch.stack([b for _, b in parts]), 0)
    assert ((joined - lse).abs()[live] <= 2.0 ** -17 * (1 + lse.abs()[live])).all()


@pytest.mark.parametrize("up", [2.0 ** -100, 2.0 ** 30])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_upstream_gradients_of_any_size(dtype, up):
    check(make(150, 72, 333, dtype, seed=6), up=up)


@pytest.mark.parametrize("up", [2.0 ** -12, 2.0 ** 7])
def test_upstream_gradients_of_any_size_in_float16(up):
    check(make(150, 72, 333, F16, seed=6), up=up)


def test_ignored_rows_count_for_nothing():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(100, 64, 500, F16, seed=7, drop=0.5))
    gone = tokens == IGNORE
    g_logits[gone], g_lse[gone] = math.nan, math.inf
    got = []
    for bad in (False, True):
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        a, b = (g_logits, g_lse) if bad else (torch.where(gone, 0.0, g_logits), torch.where(gone, 0.0, g_lse))
        logits, lse = linear_token_logits(xs, ws, tokens, IGNORE)
        assert (logits[gone] == 0).all() and (lse[gone] == 0).all()
        got.append(torch.autograd.grad((logits, lse), (xs, ws), (a, b)))
    assert (got[0][0][gone] == 0).all()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_no_row_at_all_and_only_ignored_ones():
    from linear_cross_entropy_loss_amd import linear_token_logits

    w = torch.randn(64, 500, device="cuda", dtype=BF16).requires_grad_(True)
    x = torch.zeros(2, 0, 64, device="cuda", dtype=BF16).requires_grad_(True)
    logits, lse = linear_token_logits(x, w, torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    assert logits.shape == lse.shape == (2, 0)
    dx, dw = torch.autograd.grad(logits.sum() + lse.sum(), (x, w))
    assert dx.shape == x.shape and dw.shape == w.shape and (dw == 0).all()
    x = torch.randn(5, 64, device="cuda", dtype=BF16).requires_grad_(True)
    logits, lse = linear_token_logits(x, w, torch.full((5,), IGNORE, device="cuda"))
    dx, dw = torch.autograd.grad((logits, lse), (x, w), (torch.ones(5).cuda(), torch.ones(5).cuda()))
    assert (logits == 0).all() and (lse == 0).all() and (dx == 0).all() and (dw == 0).all()


def test_tokens_that_are_none_give_nan():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, *_ = (t.cuda() for t in make(8, 64, 500, BF16, seed=8, drop=0.0))
    tokens[1], tokens[2], tokens[3] = 500, -1, -7
    logits, lse = linear_token_logits(x, w, tokens)
    assert logits.isnan().tolist() == [False, True, True, True] + 4 * [False] and lse.isfinite().all()
    logits, _ = linear_token_logits(x, w, tokens, vocab_start=100, vocab_size=600)
    assert logits.isnan().tolist() == [False, False, True, True] + 4 * [False]


def test_gradients_against_differences():
    """Central differences of the operator itself along random directions, in float32 (pairs): with steps of d the difference quotient
    is off by the third derivative's d^2 / 6 and by the results' errors, 2^-16 of magnitudes below 8 over d."""
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(20, 32, 100, F32, seed=10))
    x.requires_grad_(True), w.requires_grad_(True)

    def value(x, w):
        logits, lse = linear_token_logits(x, w, tokens, IGNORE)
        return (logits.double() @ g_logits.double() + lse.double() @ g_lse.double())

    dx, dw = torch.autograd.grad(value(x, w), (x, w))
    g = torch.Generator(device="cuda").manual_seed(1)
    d = 2.0 ** -5
    for leaf, grad in ((x, dx), (w, dw)):
        way = torch.randn(leaf.shape, generator=g, device="cuda")
        way /= way.norm()
        a, b = (value(x + d * way, w), value(x - d * way, w)) if leaf is x else (value(x, w + d * way), value(x, w - d * way))
        quotient = float((a - b) / (2 * d))
        there = float((grad.double() * way.double()).sum())
        assert abs(quotient - there) <= 20 * (d * d + 2.0 ** -16 * 8 / d), (quotient, there)


def test_shapes_strides_and_one_gradient_only():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(60, 48, 321, BF16, seed=11))
    logits, lse = linear_token_logits(x, w, tokens, IGNORE)
    wide = torch.randn(48, 800, device="cuda").to(BF16)
    wide[:, 64:385] = w
    xs = torch.randn(60, 96, device="cuda").to(BF16)
    xs[:, ::2] = x
    a, b = linear_token_logits(xs[:, ::2].view(3, 20, 48), wide[:, 64:385], tokens.view(3, 20), IGNORE)
    assert torch.equal(a.view(-1), logits) and torch.equal(b.view(-1), lse)
    xl = x.clone().requires_grad_(True)
    wl = w.clone().requires_grad_(True)
    both = torch.autograd.grad(linear_token_logits(xl, wl, tokens, IGNORE), (xl, wl), (g_logits, g_lse))
    only_x, = torch.autograd.grad(linear_token_logits(xl, w, tokens, IGNORE), xl, (g_logits, g_lse))
    only_w, = torch.autograd.grad(linear_token_logits(x, wl, tokens, IGNORE), wl, (g_logits, g_lse))
    assert torch.equal(both[0], only_x) and torch.equal(both[1], only_w)
    one, = torch.autograd.grad(linear_token_logits(xl, w, tokens, IGNORE)[1].sum(), xl)  # (the logits' gradient is absent)
    two, = torch.autograd.grad(linear_token_logits(xl, w, tokens, IGNORE), xl, (torch.zeros(60).cuda(), torch.ones(60).cuda()))
    assert torch.equal(one, two)
    with torch.no_grad():
        assert not linear_token_logits(xl, wl, tokens, IGNORE)[0].requires_grad


def test_backward_twice_autocast_and_compiled():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(70, 40, 300, F32, seed=12))
    x.requires_grad_(True), w.requires_grad_(True)
    logits, lse = linear_token_logits(x, w, tokens, IGNORE)
    first = torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse), retain_graph=True)
    second = torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.autocast("cuda", dtype=BF16):
        logits, lse = linear_token_logits(x, w, tokens, IGNORE)
    want = linear_token_logits(x.detach().to(BF16), w.detach(), tokens, IGNORE)
    assert torch.equal(logits, want[0]) and torch.equal(lse, want[1])
    dx, dw = torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse))
    assert dx.dtype == dw.dtype == F32
    inputs = make(90, 64, 400, BF16, seed=13)
    check(inputs)

    def call(x, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size):
        return linear_token_logits(x, At, tokens, ignore_index, logit_scale, N_chunk_size, vocab_start, vocab_size)

    torch._dynamo.reset()
    check(inputs, run=torch.compile(call, backend="aot_eager"))
    check(inputs, run=torch.compile(call, backend="aot_eager"), first=100, size=900)
    torch._dynamo.reset()


def test_module_and_policy_gradient():
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss

    torch.manual_seed(0)
    module = LinearCrossEntropyLoss(64, 700, device="cuda", dtype=BF16, ignore_index=-1, logit_scale=0.5)
    x = torch.randn(2, 30, 64, device="cuda", dtype=BF16, requires_grad=True)
    tokens = torch.randint(-1, 700, (2, 30), device="cuda")
    logp = module.log_probs(x, tokens)
    z = torch.log_softmax(0.5 * x.detach().double() @ module.weight.detach().double(), -1)
    want = torch.where(tokens >= 0, z.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], 0.0)
    assert (logp.double() - want).abs().max() <= 2.0 ** -17 * 16
    # with an upstream gradient of -1/n in every row it is the loss against labels
    n = int((tokens >= 0).sum())
    (-logp.sum() / n).backward()
    dx, dw = x.grad.clone(), module.weight.grad.clone()
    x.grad = module.weight.grad = None
    module(x, tokens).backward()
    for a, b in ((dx, x.grad), (dw, module.weight.grad)):
        # (two roundings of dz to the type and one of each result)
        assert (a.double() - b.double()).norm() <= 4 * 2.0 ** -8 * b.double().norm()


def test_captured_and_replayed():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, g_logits, g_lse = (t.cuda() for t in make(200, 128, 1000, F16, seed=14))

    def step(x, w):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        logits, lse = linear_token_logits(x, w, tokens, IGNORE)
        return (logits.detach(), lse.detach()) + torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w)
    for seed in range(3):
        fresh = make(200, 128, 1000, F16, seed=20 + seed)
        for t, f in zip((x, w, tokens, g_logits, g_lse), fresh):
            t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        want = step(x, w)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_float32_holds_more_than_16_bits():
    """By norms, in which the independent errors of the products average out: those of pairs are 2^-22, those of a softmax under logits of
    up to 8, that are rounded at 2^-21, below 2^-20: 2^-19 in all.  (Pairs of bfloat16: 2^-17.8.)  A large number in a row
    that is not wanted does not count, and a weight of 2^5 makes the smallest step of the others 2^-34: nothing changes."""
    from linear_cross_entropy_loss_amd import linear_token_logits

    N, H, V = 700, 512, 5000
    for outlier in (None, 2.0 ** 12):
        x, w, tokens, g_logits, g_lse = make(N, H, V, F32, seed=5)
        if outlier:
            x[3, 5], tokens[3] = outlier, IGNORE  # (of a row that is not wanted)
            w[7, 11] = outlier * 2.0 ** -7
            x[:, 7] = 0.0
        x, w, tokens, g_logits, g_lse = (t.cuda() for t in (x, w, tokens, g_logits, g_lse))
        x.requires_grad_(True)
        w.requires_grad_(True)
        print(f"token_logits float32 outlier {outlier}", flush=True)
        logits, lse = linear_token_logits(x, w, tokens, ignore_index=IGNORE)
        dx, dw = torch.autograd.grad((logits, lse), (x, w), (g_logits, g_lse))
        want, _ = oracle(x.detach(), w.detach(), tokens, g_logits, g_lse, 1.0, 0)
        if outlier:  # (the column of dx that the large weight makes)
            assert float((dx[:, 7].double() - want[2][:, 7]).norm() / want[2][:, 7].norm()) <= 2.0 ** -19
        for g, r in ((dx, want[2]), (dw, want[3])):
            assert float((g.double() - r).norm() / r.norm()) <= 2.0 ** -19


def test_second_derivatives_are_refused():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, *_ = (t.cuda() for t in make(40, 64, 300, BF16, seed=9))
    x.requires_grad_(True)
    logits, lse = linear_token_logits(x, w, tokens, ignore_index=IGNORE)
    (dx,) = torch.autograd.grad((logits - lse).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()


@pytest.mark.pack_auto
@pytest.mark.parametrize("dtype, w_dtype", [(BF16, None), (F16, None), (BF16, F32)], ids=str)
@pytest.mark.parametrize("N, H, V, drop", [(3000, 128, 17000, 0.5), (1300, 64, 9001, 0.0), (5000, 40, 777, 0.1)])
def test_few_hidden_indices(N, H, V, drop, dtype, w_dtype):
    """Without a stage of dz, and where many rows are dropped on packed ones."""
    check(make(N, H, V, dtype, seed=N, drop=drop, w_dtype=w_dtype))
    check(make(N, H, V, dtype, seed=N, drop=drop, w_dtype=w_dtype), tied=True, scale=0.5)
    if w_dtype is None:
        check(make(N, H, V, dtype, seed=N, drop=drop, pieces=2), first=V, size=2 * V)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("N, H, V", [(37, 67, 131), (40, 64, 512)])
def test_saved_tensors_kept_on_the_host(N, H, V, tied):
    """Rows that were copied to wider ones come back dense."""
    from linear_cross_entropy_loss_amd import linear_token_logits

    def run(*args, **kw):
        with torch.autograd.graph.save_on_cpu():
            return linear_token_logits(*args, **kw)

    check(make(N, H, V, BF16, seed=11), run=run, tied=tied)
    with torch.autocast("cuda", dtype=BF16):  # (the Function in Python)
        check(make(N, H, V, BF16, seed=11), run=run, tied=tied)


def test_upstream_gradients_that_are_missing_or_expanded():
    from linear_cross_entropy_loss_amd import linear_token_logits

    x, w, tokens, *_ = (t.cuda() for t in make(60, 72, 500, BF16, seed=13))
    x.requires_grad_(True)
    w.requires_grad_(True)
    logits, lse = linear_token_logits(x.view(3, 20, 72), w, tokens.view(3, 20), ignore_index=IGNORE)
    zero, one = torch.zeros_like(lse), torch.ones_like(lse)
    for got, up in ((logits.sum(), (one, zero)), (lse.sum(), (zero, one)), ((logits - lse).mean(), (one / 60, -one / 60))):
        a = torch.autograd.grad(got, (x, w), retain_graph=True)
        b = torch.autograd.grad((logits, lse), (x, w), up, retain_graph=True)
        assert all(torch.equal(i, j) for i, j in zip(a, b))
    with pytest.raises(RuntimeError):  # (changed between the passes)
        x.data_ptr()
        with torch.no_grad():
            x.add_(1)
        torch.autograd.grad(lse.sum(), x)


@pytest.mark.pack_auto  # (the recomputation may run in a thread of autograd's, which has the library's own choice)
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_under_a_checkpoint(reentrant):
    from torch.utils.checkpoint import checkpoint

    from linear_cross_entropy_loss_amd import linear_token_logits

    def run(x, At, tokens, **kw):
        return checkpoint(lambda a, b: linear_token_logits(a, b, tokens, **kw), x, At, use_reentrant=reentrant)

    inputs = make(50, 72, 600, BF16, seed=17)
    if not reentrant:
        check(inputs, run=run)
        return
    x, w, tokens, g_logits, g_lse = (t.cuda() for t in inputs)  # (that one gives gradients to leaves only)
    grads = []
    for f in (run, linear_token_logits):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w)]
        torch.autograd.backward(f(*leaves, tokens, ignore_index=IGNORE), (g_logits, g_lse))
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.pack_auto  # (a setting of packing is a thread's own)
def test_calls_from_several_threads_and_streams():
    """Forward and backward of four threads at once, each on a stream of its own: what each gives alone."""
    import threading

    from linear_cross_entropy_loss_amd import linear_token_logits

    sizes = [(64, 256, 4096), (300, 128, 5000), (513, 72, 999), (128, 512, 9000)]
    cases = [tuple(t.cuda() for t in make(*s, BF16, seed=i)) for i, s in enumerate(sizes)]

    def step(x, w, tokens, g_logits, g_lse):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out = linear_token_logits(x, w, tokens, ignore_index=IGNORE)
        return (*out, *torch.autograd.grad(out, (x, w), (g_logits, g_lse)))

    alone = [[t.detach().clone() for t in step(*c)] for c in cases]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = step(*cases[i])
            stream.synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, alone[i])):
            failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
