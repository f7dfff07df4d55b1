"""Clipping of many tensors by their common norm against the definition in 64 bits.  The norm: squares and sums in doubles, rounded to
float32 once (2^-24; 2^-23 asserted, the doubles' own sums being off by 2^-40 at most).  An element: one fp32 factor (2^-24), one
product (2^-24), the type's half step; numbers below the type's normal range half of its smallest step."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SMALLEST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}


def check(grads, max_norm, divisor=1.0, out=None):
    from linear_cross_entropy_loss_amd import clip_gradients

    print(f"clip {[(tuple(g.shape), str(g.dtype)) for g in grads[:6]]} ... {len(grads)} max {max_norm}", flush=True)
    was = [g.double() for g in grads]
    number = float(divisor)
    norm = math.sqrt(math.fsum(float((g * g).sum()) for g in was)) / number
    factor = (min(1.0, max_norm / norm) if norm > 0 else 1.0) / number
    got = clip_gradients(grads, max_norm, divisor, out)
    assert got.dtype == F32 and got.shape == ()
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, o in zip(was, out if out is not None else grads):
        half = torch.finfo(o.dtype).eps / 2
        assert ((o.double() - g * factor).abs() <= (2.0 ** -23 + half) * (g * factor).abs() + SMALLEST[o.dtype]).all()
    return got


def make(shapes, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    types = dtype if isinstance(dtype, list) else [dtype] * len(shapes)
    return [(torch.randn(s, generator=g, device="cuda") * size).to(t) for s, t in zip(shapes, types)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("n", [1, 7, 8, 255, 8191, 8192, 8193, 100001, 1 << 22])
def test_one_tensor(n, dtype):
    check(make([(n,)], dtype, n), 0.5)
    check(make([(n,)], dtype, n), 1e6)


@pytest.mark.parametrize("count", [2, 120, 121, 300])
def test_many_tensors_of_all_types(count):
    shapes = [(1 + (37 * i) % 9000,) for i in range(count)]
    types = [(BF16, F16, F32)[i % 3] for i in range(count)]
    check(make(shapes, types, count), 3.0)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_to_other_tensors(dtype, max_norm):
    grads = make([(300, 70), (9001,), (), (0,), (20000,)], dtype, 1)
    kept = [g.clone() for g in grads]
    for to in (F32, dtype):
        out = [torch.full(g.shape, 5.0, dtype=to, device="cuda") for g in grads]
        check(grads, max_norm, out=out)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))


def test_divisor():
    check(make([(3000,), (77, 5)], F16, 2, size=100.0), 1.0, divisor=4096.0)
    check(make([(3000,), (77, 5)], F16, 2, size=100.0), 1.0, divisor=torch.tensor(4096.0, device="cuda"))
    check(make([(3000,), (77, 5)], F32, 2), math.inf, divisor=8.0)


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e18, 1e30])
def test_squares_beyond_float32(size):
    check(make([(10000,), (33,)], F32, 3, size=size), size)
    check(make([(10000,), (33,)], BF16, 3, size=size), size)


def test_addresses_and_strides_of_any_kind():
    room = torch.randn(50001, device="cuda")
    check([room.clone()[1:40000], room.clone().to(BF16)[3:30000], room.clone().to(F16)[1:]], 1.0)
    square = torch.randn(200, 300, device="cuda")
    check([square.clone().t(), square.clone()[:, ::2], square.clone()[5:, 7:], square.clone().to(BF16).t()[::3]], 1.0)
    around = torch.full((200, 300), 9.0, device="cuda")
    part = around[20:40, 30:60]
    check([part], 1.0)
    around[20:40, 30:60] = 9.0
    assert (around == 9.0).all()


def test_the_ends_of_a_tensor():
    for n in (1, 8192, 8200, 30000):
        room = torch.full((n + 64,), 3.0, device="cuda", dtype=BF16)
        check([room[32:n + 32]], 1.0)
        assert (room[:32] == 3.0).all() and (room[n + 32:] == 3.0).all()


def test_zeros_nan_and_infinities():
    from linear_cross_entropy_loss_amd import clip_gradients

    zeros = [torch.zeros(100, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(clip_gradients(zeros, 1.0)) == 0.0 and (zeros[0] == 0).all()
    for bad in (math.nan, math.inf):
        g = make([(9000,), (50,)], F16, 4)
        g[1][3] = bad
        was = [t.clone() for t in g]
        norm = float(clip_gradients(g, 1.0, divisor=2.0))
        assert not math.isfinite(norm)
        for a, b in zip(g, was):
            # (half of a number below 2^-13 is rounded to a multiple of 2^-24: off by up to 2^-25, and twice that here)
            assert torch.equal(a.isfinite(), b.isfinite())
            assert ((a.float() * 2).nan_to_num() - b.float().nan_to_num()).abs().max() <= 2 * SMALLEST[F16]


def test_the_order_of_sums_is_fixed_and_versions_count():
    from linear_cross_entropy_loss_amd import clip_gradients

    g = make([(1 << 21,), (1 << 20,), (5,)], BF16, 5)
    norms = {float(clip_gradients([t.clone() for t in g], 1.0)) for _ in range(5)}
    assert len(norms) == 1
    leaf = torch.randn(5, device="cuda", requires_grad=True)
    t = leaf * 1.0
    y = (t * t).sum()
    clip_gradients([t.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_captured_step_replayed():
    from linear_cross_entropy_loss_amd import clip_gradients

    given = make([(5000,), (300, 40)], BF16, 6)
    work = [g.clone() for g in given]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clip_gradients(work, 1.0)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for w, g in zip(work, given):
            w.copy_(g)
        norm = clip_gradients(work, 1.0)
    for size in (1.0, 0.001, 7.0):
        for g, f in zip(given, make([(5000,), (300, 40)], BF16, 7, size=size)):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        eager = [g.clone() for g in given]
        assert torch.equal(norm, clip_gradients(eager, 1.0)) and all(torch.equal(a, b) for a, b in zip(work, eager))


def test_two_streams_at_once():
    from linear_cross_entropy_loss_amd import clip_gradients

    sets = [make([(100000,), (333,)], F32, 8 + i, size=10.0) for i in range(2)]
    want = [[t.clone() for t in s] for s in sets]
    norms = [clip_gradients(s, 1.0) for s in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            got.append(clip_gradients(s, 1.0))
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(got), torch.stack(norms))
    assert all(torch.equal(a, b) for s, w in zip(sets, want) for a, b in zip(s, w))


def test_offsets_past_32_bits():
    from linear_cross_entropy_loss_amd import clip_gradients

    n = (1 << 31) + 12345
    g = torch.full((n,), 2.0 ** -8, dtype=BF16, device="cuda")
    g[-1] = 3.0
    print(f"clip {n}", flush=True)
    norm = math.sqrt((n - 1) * 2.0 ** -16 + 9.0)
    got = clip_gradients(g, 0.5)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for at, was in ((0, 2.0 ** -8), (n - 2, 2.0 ** -8), (n - 1, 3.0)):
        want = was * 0.5 / norm
        assert abs(float(g[at]) - want) <= (2.0 ** -23 + 2.0 ** -8) * want
    assert torch.equal(g[:-1].min(), g[:-1].max())
