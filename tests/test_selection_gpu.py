"""top_logits and sample_logits against their definitions: a stable sort in 64 bits, its weights and their sums.

Columns are compared exactly.  The kernels' sums are fixed point with 45 binary places or more (62 - log2 V, at most 50) under the largest
weight of 1, the oracle's are doubles: they agree on a token unless u * sum lies within V * 2^-46 (2^-29 at V = 131072) of a
border, about one row in 10^8 of the inputs below, whose seeds are fixed.  lse: an fp32 exponential of d = z - max is off by 2^-24 |d| relative,
and the mean of |d| over the softmax is at most log V <= 12.5: 2^-20.4 of the sum if all err to one side; sums of a thread's 136 terms and
the final rounding add 2^-23 each as errors go: 2^-20 * max(1, |lse|)."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(N, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(N, V, generator=g)).to(dtype)


def ref_top(z, k):
    key = z.double() + 0.0
    # (NaN above +inf: two sorts, the second by whether it is one)
    cols = torch.sort(torch.where(key.isnan(), math.inf, key), dim=1, descending=True, stable=True).indices
    nan = z.isnan().gather(1, cols).to(torch.uint8)
    cols = cols.gather(1, torch.sort(nan, dim=1, descending=True, stable=True).indices)[:, :k]
    return z.gather(1, cols), cols, torch.logsumexp(z.double(), 1)


def ref_sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    z = z.double() + 0.0
    N, V = z.shape

    def column(v):
        return torch.as_tensor(v).to(F32).double().expand(N).reshape(N, 1)

    temperature, top_k, top_p, min_p = map(column, (temperature, top_k, top_p, min_p))
    order = torch.sort(z, dim=1, descending=True, stable=True)
    zs = order.values
    greedy = ~(temperature > 0)
    d = torch.where(zs == zs[:, :1], 0.0, zs - zs[:, :1])
    w = torch.exp(d / torch.where(greedy, 1.0, temperature))
    place = torch.arange(V)
    w = torch.where((top_k <= 0) | (place < top_k), w, 0.0)
    before = torch.cumsum(w, 1) - w
    stays = (place == 0) | ((~(top_p < 1) | (before < top_p * w.sum(1, keepdim=True))) & (~(min_p > 0) | (w >= min_p)) & ~greedy)
    w = torch.where(stays, w, 0.0)
    upto = torch.cumsum(w, 1)
    first = (upto > u.double().reshape(N, 1) * upto[:, -1:]).to(torch.uint8).argmax(1, keepdim=True)
    token = order.indices.gather(1, first)[:, 0]
    return torch.where(z.isnan().any(1) | (z == -math.inf).all(1), -1, token)


def check_top(z, k, zg=None):
    from linear_cross_entropy_loss_amd import top_logits

    print(f"top {tuple(z.shape)} {z.dtype} k={k}", flush=True)
    values, index, lse = top_logits(z.cuda() if zg is None else zg, k)
    ref_values, ref_index, ref_lse = ref_top(z, k)
    assert values.dtype == z.dtype and index.dtype == torch.int64 and lse.dtype == F32
    assert torch.equal(index.cpu(), ref_index)
    assert torch.equal(values.cpu().nan_to_num(nan=12345.0), ref_values.nan_to_num(nan=12345.0))
    ok = torch.isfinite(ref_lse)
    assert ((lse.cpu().double() - ref_lse).abs()[ok] <= 2.0 ** -20 * ref_lse.abs().clamp(min=1.0)[ok]).all()
    odd = lse.cpu()[~ok].double()
    assert torch.equal(odd.isnan(), ref_lse[~ok].isnan()) and torch.equal(odd[~odd.isnan()], ref_lse[~ok][~odd.isnan()])


def check_sample(z, u, zg=None, **settings):
    from linear_cross_entropy_loss_amd import sample_logits

    print(f"sample {tuple(z.shape)} {z.dtype} { {k: v for k, v in settings.items() if not isinstance(v, torch.Tensor)} }", flush=True)
    got = sample_logits(z.cuda() if zg is None else zg, u.cuda(),
                        **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
    ref = ref_sample(z, u, **settings)
    assert got.dtype == torch.int64
    assert torch.equal(got.cpu(), ref), (got.cpu()[got.cpu() != ref][:5], ref[got.cpu() != ref][:5])


SIZES = [(1, 1), (1, 2), (5, 3), (3, 63), (4, 64), (4, 65), (3, 1000), (7, 1001), (2, 8193), (5, 32000), (3, 50257), (2, 131072), (1, 262147)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", SIZES)
def test_top_sizes(N, V, dtype):
    z = rows(N, V, dtype, seed=V)
    for k in sorted({1, 2, 7, 64, 65, 1000, 1024, V}):
        if k <= min(V, 1024):
            check_top(z, k)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", SIZES)
def test_sample_sizes(N, V, dtype):
    z = rows(N, V, dtype, seed=V + 1)
    u = torch.rand(N, generator=torch.Generator().manual_seed(V))
    check_sample(z, u)
    check_sample(z, u, temperature=0.0)
    check_sample(z, u, temperature=0.7, top_p=0.9)
    check_sample(z, u, temperature=1.5, top_k=40)
    check_sample(z, u, temperature=0.9, top_k=2000, top_p=0.97, min_p=0.001)
    check_sample(z, u, min_p=0.05)
    check_sample(z, u, top_k=1)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_settings_by_row(dtype):
    N, V = 96, 5003
    z = rows(N, V, dtype, seed=3, spread=3.0)
    g = torch.Generator().manual_seed(4)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (N,), generator=g)]  # noqa: E731
    nan, inf = math.nan, math.inf
    check_sample(z, torch.rand(N, generator=g), temperature=pick([0.0, -1.0, nan, 0.3, 1.0, 4.0, 1e-3, 1e4, inf]),
                 top_k=pick([0, -3, 1, 2, 50, 5002, 5003, 9999]), top_p=pick([1.0, 2.0, nan, 0.9, 0.5, 1e-6, 0.0, -1.0]),
                 min_p=pick([0.0, -1.0, nan, 0.01, 0.3, 1.0, 2.0]))
    check_sample(z, torch.rand(N, generator=g), temperature=torch.tensor(0.8), top_k=torch.tensor(30, dtype=torch.int32), top_p=0.8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_numbers_at_the_ends(dtype):
    """u = 0 takes the first column, u next to 1 the last that stays; numbers outside and NaN take the nearest."""
    z = rows(8, 700, dtype, seed=5)
    u = torch.tensor([0.0, 2.0 ** -149, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, math.nan, 0.5])
    for settings in ({}, {"top_k": 10}, {"top_p": 0.5}, {"min_p": 0.2}):
        from linear_cross_entropy_loss_amd import sample_logits

        got = sample_logits(z.cuda(), u.cuda(), **settings).cpu()
        ref = ref_sample(z, u.nan_to_num(nan=0.0).clamp(0.0, 1 - 2.0 ** -24), **settings)
        assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_equal_values(dtype):
    """Rows of one value, of two, of zeros of both signs: order by column, and borders that are exact."""
    V = 4096
    z = torch.zeros(6, V, dtype=dtype)
    z[1, ::2] = -0.0
    z[2, 1000:] = -1.0
    z[3] = torch.finfo(dtype).min
    z[4] = -3.5
    z[4, 17] = 5.0
    z[5, ::3] = 2.0
    for k in (1, 5, 1000, 1024):
        check_top(z, k)
    u = torch.tensor([0.0, 0.25, 0.9, 0.5, 0.75, 0.125])
    check_sample(z, u)
    check_sample(z, u, top_p=0.5)
    check_sample(z, u, top_k=1000)
    check_sample(z, u, top_k=100, top_p=0.25, min_p=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_columns(dtype):
    """-inf, the type's lowest value, +inf and NaN; rows that are masked altogether."""
    low = torch.finfo(dtype).min
    z = rows(10, 2000, dtype, seed=6)
    z[0, 5:] = -math.inf
    z[1] = -math.inf
    z[2, 100:] = low
    z[3] = low
    z[3, 7] = -math.inf
    z[4, 9] = math.inf
    z[5, [9, 1999]] = math.inf
    z[5, :5] = -math.inf
    z[6, 1234] = math.nan
    z[7] = math.nan
    z[8, 3] = -math.inf
    z[8, 4] = low
    for k in (1, 4, 6, 100, 1024):
        check_top(z, k)
    u = torch.rand(10, generator=torch.Generator().manual_seed(7))
    for settings in ({}, {"temperature": 0.0}, {"top_k": 8}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_k": 1500, "top_p": 0.99}):
        check_sample(z, u, **settings)


@pytest.mark.parametrize("value", [-10000.0, 0.0, 1.0])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_one_value_in_most_columns(dtype, value):
    """A mask of an ordinary number over more than 65535 columns."""
    z = torch.full((3, 140001), value, dtype=dtype)
    few = rows(3, 200, dtype, seed=8)
    z[:, 70000:70200] = few
    z[2, :] = value
    for k in (3, 150, 300, 1024):
        check_top(z, k)
    u = torch.tensor([0.3, 0.99, 0.5])
    check_sample(z, u)
    check_sample(z, u, top_p=0.9)
    check_sample(z, u, top_k=300)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_far_apart_values(dtype):
    """The whole range of the type: subnormal numbers, both signs, differences that overflow the type."""
    big = torch.finfo(dtype).max
    g = torch.Generator().manual_seed(9)
    z = (torch.randn(4, 3001, generator=g, dtype=torch.float64) * torch.exp(torch.randn(4, 3001, generator=g, dtype=torch.float64) * 20)).clamp(
        -big, big).to(dtype)
    z[2] = z[2] * torch.finfo(dtype).tiny
    z[3, 0], z[3, 1] = big, -big
    for k in (1, 64, 500):
        check_top(z, k)
    u = torch.rand(4, generator=g)
    check_sample(z, u)
    check_sample(z, u, temperature=3.0, top_p=0.8)
    check_sample(z, u, top_k=77)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strides_and_boundaries(dtype, offset):
    """Rows at any element boundary, with NaN before and behind them; transposed logits; an expanded row; leading dimensions."""
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    N, V = 6, 1003
    z = rows(N, V, dtype, seed=10)
    wide = torch.full((N, V + 10), math.nan, dtype=dtype)
    wide[:, offset:offset + V] = z
    zg = wide.cuda()[:, offset:offset + V]
    u = torch.rand(N, generator=torch.Generator().manual_seed(11))
    check_top(z, 20, zg)
    check_sample(z, u, zg, top_p=0.9)
    check_top(z, 20, z.t().contiguous().cuda().t())
    check_sample(z, u, z.t().contiguous().cuda().t())
    one = z[:1].cuda().expand(N, V)
    check_top(z[:1].expand(N, V), 5, one)
    check_sample(z[:1].expand(N, V), u, one)
    values, index, lse = top_logits(z.cuda().reshape(2, 3, V), 4)
    assert values.shape == index.shape == (2, 3, 4) and lse.shape == (2, 3)
    tokens = sample_logits(z.cuda().reshape(2, 3, V), u.cuda().reshape(2, 3), top_k=torch.full((2, 3), 5, device="cuda"))
    assert torch.equal(tokens.cpu().reshape(-1), ref_sample(z, u, top_k=5))
    single = sample_logits(z[0].cuda(), u[0].cuda())
    assert single.shape == () and single.item() == ref_sample(z[:1], u[:1]).item()


def test_no_rows():
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    values, index, lse = top_logits(torch.empty(0, 100, device="cuda"), 3)
    assert values.shape == (0, 3) and index.shape == (0, 3) and lse.shape == (0,)
    assert sample_logits(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)


def test_refusals():
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    z, u = torch.zeros(4, 50, device="cuda"), torch.zeros(4, device="cuda")
    for k in (0, -1, 51, 1025):
        with pytest.raises(ValueError):
            top_logits(z, k)
    with pytest.raises(ValueError):
        top_logits(torch.zeros(4, 2000, device="cuda"), 1025)
    for bad in (torch.zeros(4, 0, device="cuda"), torch.zeros((), device="cuda"), z.double(), z.long()):
        with pytest.raises(ValueError):
            top_logits(bad, 1)
        with pytest.raises(ValueError):
            sample_logits(bad, u)
    for settings in ({"temperature": -1.0}, {"temperature": math.inf}, {"temperature": math.nan}, {"top_k": -1}, {"top_p": 0.0}, {"top_p": 1.1},
                     {"top_p": math.nan}, {"min_p": -0.1}, {"min_p": 1.5}, {"top_k": torch.ones(3, dtype=torch.int64, device="cuda")},
                     {"top_k": torch.ones(4, device="cuda")}, {"top_p": torch.ones(4, dtype=torch.int64, device="cuda")},
                     {"min_p": torch.ones(4)}):
        with pytest.raises(ValueError):
            sample_logits(z, u, **settings)
    for bad_u in (u[:3], u.double(), u.cpu(), 0.5):
        with pytest.raises(ValueError):
            sample_logits(z, bad_u)


def test_frequencies():
    """2^16 numbers at equal distances: every token as often as its probability says, to one."""
    from linear_cross_entropy_loss_amd import sample_logits

    z = rows(1, 300, BF16, seed=12)
    n = 1 << 16
    u = (torch.arange(n, dtype=torch.float64) / n).float()
    got = sample_logits(z.cuda().expand(n, 300), u.cuda())
    counts = torch.bincount(got.cpu(), minlength=300).double()
    assert (counts - torch.softmax(z[0].double(), 0) * n).abs().max() <= 1.0 + 1e-6


def test_streams_graphs_and_compiled():
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    z, u = rows(16, 5001, BF16, seed=13).cuda(), torch.rand(16, generator=torch.Generator().manual_seed(14)).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = sample_logits(z, u, top_p=0.9)
        top = top_logits(z, 10)
    side.synchronize()
    assert torch.equal(got, sample_logits(z, u, top_p=0.9))
    assert all(torch.equal(a, b) for a, b in zip(top, top_logits(z, 10)))
    static_z, static_u = z.clone(), u.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens = sample_logits(static_z, static_u, 0.8, 100, 0.95, 0.01)
        values, index, lse = top_logits(static_z, 7)
    for seed in range(4):
        static_z.copy_(rows(16, 5001, BF16, seed=20 + seed))
        static_u.copy_(torch.rand(16, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens.cpu(), ref_sample(static_z.cpu(), static_u.cpu(), 0.8, 100, 0.95, 0.01))
        assert torch.equal(index.cpu(), ref_top(static_z.cpu(), 7)[1])
    run = torch.compile(lambda a, b: (sample_logits(a, b, temperature=0.9, top_p=0.8) + 1, top_logits(a, 5)[1]), fullgraph=True)
    tokens, index = run(z, u)
    assert torch.equal(tokens.cpu() - 1, ref_sample(z.cpu(), u.cpu(), 0.9, 0, 0.8)) and torch.equal(index.cpu(), ref_top(z.cpu(), 5)[1])


def test_distillation_on_policy():
    """A run of all of them: the student answers, the teacher's top logits of the answer are kept, loss and gradients; twice with
    the same numbers, and the loss is that of the definition."""
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss, sample_logits, top_logits

    torch.manual_seed(15)
    H, V, N, K = 64, 1003, 40, 16
    embed = torch.randn(V, H, device="cuda", dtype=BF16)
    student = LinearCrossEntropyLoss(H, V, device="cuda", dtype=BF16)
    teacher = (torch.randn(H, V, device="cuda") / 4).to(BF16)
    numbers = torch.rand(8, N, device="cuda")

    def step():
        student.weight.grad = None
        tokens = torch.zeros(N, dtype=torch.long, device="cuda")
        xs = []
        for u in numbers:
            xs.append(torch.tanh(embed[tokens]))
            tokens = sample_logits((xs[-1] @ student.weight).detach(), u, temperature=0.9, top_p=0.95)
        x = torch.stack(xs).requires_grad_(True)
        values, index, lse = top_logits(x.detach() @ teacher, K)
        index[:, tokens == 0] = -1
        loss = student.distill(x, index, values, temperature=1.5)
        loss.backward()
        return loss.detach(), x.grad, student.weight.grad, (x.detach(), index, values)

    first, again = step(), step()
    assert all(torch.equal(a, b) for a, b in zip(first[:3], again[:3]))
    x, index, values = (t.cpu() for t in first[3])
    kept = (index >= 0).all(-1)
    q = torch.softmax(values[kept].double() / 1.5, -1)
    p = torch.log_softmax(x[kept].double() @ student.weight.detach().cpu().double() / 1.5, -1)
    ref = (torch.special.xlogy(q, q) - q * p.gather(-1, index[kept])).sum(-1).mean()
    assert abs(first[0].item() - ref.item()) <= 64 * 2.0 ** -22 * max(1.0, ref.item())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", [(3001, 1009), (1100, 20011), (600, 33003)])
def test_more_rows_than_workgroups(N, V, dtype):
    """A workgroup takes rows one after another, and neighbours are done in different ways: ordinary, all equal, masked, with a NaN, with
    infinities, one column alone."""
    z = rows(N, V, dtype, seed=16)
    kind = torch.randint(0, 8, (N,), generator=torch.Generator().manual_seed(17))
    z[kind == 0] = 1.5
    z[kind == 1] = -math.inf
    z[kind == 2, V // 2] = math.nan
    z[kind == 3, V // 3] = math.inf
    z[kind == 4, 5:] = -math.inf
    u = torch.rand(N, generator=torch.Generator().manual_seed(18))
    check_top(z, 20)
    check_sample(z, u)
    check_sample(z, u, top_p=0.7)
    check_sample(z, u, temperature=0.9, top_k=33)
    g = torch.Generator().manual_seed(19)
    check_sample(z, u, temperature=torch.rand(N, generator=g), top_k=torch.randint(-1, 60, (N,), generator=g),
                 top_p=torch.rand(N, generator=g) * 1.2, min_p=torch.rand(N, generator=g) * 0.1)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_long_lists(dtype):
    """More than the way by maxima takes, and rows of fewer columns than threads."""
    for N, V in ((5, 5003), (3, 40000)):
        z, u = rows(N, V, dtype, seed=20), torch.rand(N, generator=torch.Generator().manual_seed(21))
        for k in (511, 512, 513, 1000, 1024):
            check_top(z, k)
            check_sample(z, u, top_k=k, temperature=3.0)
        check_sample(z, u, top_k=3000, temperature=5.0, top_p=0.9, min_p=0.01)
    z, u = rows(4, 700, dtype, seed=22), torch.rand(4, generator=torch.Generator().manual_seed(23))
    for k in (300, 512, 699, 700):
        check_top(z, k)
        check_sample(z, u, top_k=k)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [1000, 9000, 40000])
def test_temperatures(V, dtype):
    """From the largest column alone to the same weight for all; at 1e-3 of V = 40000 values between 2 and 8 more than one column counts."""
    z = rows(6, V, dtype, seed=24)
    u = torch.rand(6, generator=torch.Generator().manual_seed(25))
    for t in (1e-38, 1e-6, 1e-3, 0.1, 30.0, 1e6, 1e30, 3e38):
        check_sample(z, u, temperature=t)
        check_sample(z, u, temperature=t, top_p=0.37)
        check_sample(z, u, temperature=t, min_p=0.8, top_k=V // 2)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_values_close_together(dtype):
    """Thousands of different values within a few bins of the weight, and as many equal ones beside them."""
    V = 15000
    g = torch.Generator().manual_seed(26)
    near = (1.0 + torch.rand(4, V, generator=g) / 300).to(dtype)
    near[1, ::2] = 1.0
    near[2, :100] += 3
    near[3, 5000:] -= 40
    u = torch.rand(4, generator=g)
    for settings in ({}, {"top_p": 0.5}, {"top_k": 4000}, {"min_p": 0.999}, {"temperature": 0.001, "top_p": 0.6}):
        check_sample(near, u, **settings)
    check_top(near, 100)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_row_of_millions(dtype):
    V = (1 << 22) + 5
    z, u = rows(1, V, dtype, seed=27), torch.tensor([0.8125])
    check_top(z, 1024)
    check_top(z, 10)
    check_sample(z, u, top_p=0.9)
    check_sample(z, u, top_k=50)


def test_two_streams_and_two_threads_at_once():
    import threading

    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    sets = [(rows(300, 33000, BF16, seed=28 + i).cuda(), torch.rand(300, device="cuda")) for i in range(2)]
    sets.append((rows(300, 9000, F32, seed=30).cuda(), torch.rand(300, device="cuda")))
    call = lambda z, u: (sample_logits(z, u, 0.9, 0, 0.9), sample_logits(z, u, top_k=40), *top_logits(z, 30))
    ref = [call(*s) for s in sets]
    torch.cuda.synchronize()
    got = [None] * len(sets)

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                got[i] = call(*sets[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(ref, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_gradient_and_opcheck():
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    z, u = rows(4, 300, BF16, seed=31).cuda().requires_grad_(True), torch.rand(4, device="cuda")
    values, _, lse = top_logits(z, 5)
    assert not values.requires_grad and not lse.requires_grad and not sample_logits(z, u).requires_grad
    z = z.detach()
    torch.library.opcheck(torch.ops.lce_amd.top_logits.default, (z, 5), test_utils=("test_schema", "test_faketensor"))
    one = torch.ones((), device="cuda")
    torch.library.opcheck(torch.ops.lce_amd.sample_logits.default, (z, u, one, torch.zeros((), dtype=torch.int64, device="cuda"), one, 0 * one),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("V", [9000, 40000])
@pytest.mark.parametrize("dtype,temperature", [(BF16, 1e38), (F16, 3000.0), (F16, 1e5), (F32, 2e38), (F16, 1.0), (BF16, 1.0)])
def test_the_lowest_number_with_a_weight(dtype, temperature, V):
    """Columns masked by the type's lowest number count like any other where the temperature leaves them a weight."""
    z = rows(6, V, dtype, seed=32)
    z[:3, V // 3:] = torch.finfo(dtype).min
    z[1, ::2] = -math.inf
    u = torch.tensor([0.1, 0.6, 0.99, 0.1, 0.6, 0.99])
    check_sample(z, u, temperature=temperature)
    check_sample(z, u, temperature=temperature, top_p=0.7)


def test_captured_long_rows():
    """The way that takes a whole compute unit's LDS, captured without a call before, two graphs replayed in turn."""
    from linear_cross_entropy_loss_amd import sample_logits

    z = [rows(40, 50257, dtype, seed=33).cuda() for dtype in (BF16, F16)]
    u = torch.rand(40, generator=torch.Generator().manual_seed(34)).cuda()
    graphs, tokens = [], []
    for one in z:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            tokens.append(sample_logits(one, u, 0.8, 0, 0.9))
    for seed in range(3):
        u.copy_(torch.rand(40, generator=torch.Generator().manual_seed(35 + seed)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for one, got in zip(z, tokens):
            assert torch.equal(got.cpu(), ref_sample(one.cpu(), u.cpu(), 0.8, 0, 0.9))
            assert torch.equal(got, sample_logits(one, u, 0.8, 0, 0.9))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_beyond_the_cache(dtype):
    """So many long rows that a workgroup takes several: what each part of them gives by itself, where it takes one."""
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    N, V = 600, 300001 if dtype == F32 else 600001
    g = torch.Generator(device="cuda").manual_seed(38)
    z = (2.0 * torch.randn(N, V, generator=g, device="cuda")).to(dtype)
    z[7] = 0.0
    z[300, 5] = math.nan
    z[500, 20:] = -math.inf
    u = torch.rand(N, generator=g, device="cuda")
    top, token = top_logits(z, 20), sample_logits(z, u, 0.9, 30)
    for i in range(0, N, 200):
        part = top_logits(z[i:i + 200], 20)
        assert torch.equal(top[1][i:i + 200], part[1])
        assert torch.equal(top[0][i:i + 200].nan_to_num(nan=9e9), part[0].nan_to_num(nan=9e9))
        assert torch.equal(top[2][i:i + 200].nan_to_num(nan=9e9), part[2].nan_to_num(nan=9e9))
        assert torch.equal(token[i:i + 200], sample_logits(z[i:i + 200], u[i:i + 200], 0.9, 30))
    check_top(z[:2].cpu(), 20)
    check_top(z[596:].cpu(), 20)
    assert torch.equal(top[1][596:].cpu(), ref_top(z[596:].cpu(), 20)[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_row_does_not_depend_on_the_others(dtype):
    """Bit for bit the same values, columns and lse alone, among few and among many rows, by either way to do a row."""
    from linear_cross_entropy_loss_amd import sample_logits, top_logits

    for V in (777, 30011):
        z, u = rows(700, V, dtype, seed=39).cuda(), torch.rand(700, generator=torch.Generator().manual_seed(40)).cuda()
        many, token = top_logits(z, 30), sample_logits(z, u, 0.7, 0, 0.9)
        for n in (1, 100):
            few = top_logits(z[:n], 30)
            assert all(torch.equal(a, b[:n]) for a, b in zip(few, many))
            assert torch.equal(sample_logits(z[:n], u[:n], 0.7, 0, 0.9), token[:n])
        assert torch.equal(top_logits(z, 700)[2], many[2])  # (by digits)
        assert torch.equal(top_logits(z[:3], 700)[2], many[2][:3])


def test_host_path_gives_the_same_and_knows_its_limits(monkeypatch):
    """What the C++ host path takes gives what Python gives; what it does not take gets there by itself."""
    from linear_cross_entropy_loss_amd import sample_logits, selection, top_logits

    z = rows(12, 301, BF16, seed=41).cuda()
    u = torch.rand(12, generator=torch.Generator().manual_seed(42)).cuda()
    g = torch.Generator().manual_seed(43)
    T, P = torch.rand(12, generator=g).cuda(), torch.rand(12, generator=g).cuda()
    K = torch.randint(0, 40, (12,), generator=g).cuda()
    wide = torch.zeros(12, 400, dtype=BF16, device="cuda")
    wide[:, 50:351] = z
    calls = [lambda: sample_logits(z, u), lambda: sample_logits(z, u, 0.7, 30, 0.9, 0.01), lambda: sample_logits(z, u, 1, 0, 1, 0),
             lambda: sample_logits(z, u, T, K, P, 0.02), lambda: sample_logits(z, u, T[0], K.int(), P[3], 0), lambda: sample_logits(
                 wide[:, 50:351], u, 0.9), lambda: sample_logits(z.reshape(3, 4, 301), u.reshape(3, 4), 0.9, K.reshape(3, 4)),
             lambda: sample_logits(z.t().contiguous().t(), u), lambda: sample_logits(z[0], u[0]), lambda: sample_logits(z[::2], u[::2], T[::2]),
             lambda: sample_logits(z.expand(2, 12, 301), u.expand(2, 12)), lambda: sample_logits(z[:, :1], u),
             lambda: torch.cat([t.reshape(-1).float() for t in top_logits(z, 9)]),
             lambda: torch.cat([t.reshape(-1).float() for t in top_logits(wide[:, 50:351], 9)]),
             lambda: torch.cat([t.reshape(-1).float() for t in top_logits(z.reshape(2, 6, 301), 9)]),
             lambda: torch.cat([t.reshape(-1).float() for t in top_logits(z[3], 2)])]
    native = [call() for call in calls]
    monkeypatch.setattr(selection, "_here", lambda t: False)
    for call, a in zip(calls, native):
        b = call()
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
    monkeypatch.undo()
    values, index, lse = top_logits(z.requires_grad_(True).reshape(2, 6, 301), 4)
    assert values.shape == index.shape == (2, 6, 4) and lse.shape == (2, 6) and values.dtype == BF16 and not values.requires_grad
    for bad in ({"temperature": "1"}, {"top_k": 1 << 70}, {"top_k": None}):
        with pytest.raises((ValueError, TypeError, OverflowError)):
            sample_logits(z, u, **bad)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,V,offset", [(3, 9001, 0), (3, 9001, 3), (300, 5003, 1), (2, 40000, 5)])
def test_fewer_large_columns_than_are_asked_for(N, V, offset, dtype):
    """Rows of which the first k reach into columns that are all equal: masked but for a few, constant, zeros of either sign, and -- float32 --
    numbers that differ in their last places alone."""
    base = rows(N, V, dtype, seed=44)
    few = torch.rand(N, V, generator=torch.Generator().manual_seed(45)) < 12 / V
    u = torch.rand(N, generator=torch.Generator().manual_seed(46))
    signs = torch.where(torch.rand(N, V, generator=torch.Generator().manual_seed(47)) < 0.5, 0.0, -0.0).to(dtype)
    close = (1.0 + torch.arange(V) % 7 * 2.0 ** -20).to(dtype).expand(N, V)
    for floor in (-math.inf, torch.finfo(dtype).min, -1e4, 0.0, 1.5, signs, close):
        z = torch.where(few, base, torch.as_tensor(floor).to(dtype))
        buffer = torch.full((N, V + 11), 7.0, dtype=dtype, device="cuda")
        zg = buffer[:, offset:offset + V]
        zg.copy_(z.cuda())
        for k in (1, 5, 32, 512):
            check_top(z, k, zg)
            check_sample(z, u, zg, top_k=k)
        check_sample(z, u, zg, top_k=50, temperature=2.0, top_p=0.9)
        check_sample(z, u, zg, top_k=torch.full((N,), 40), temperature=0.5, min_p=0.01)
