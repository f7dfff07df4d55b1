"""Numbers of 8 bits and logits from them, against their definitions.  The whole numbers are equal: they are the nearest to a quotient of two
numbers of the type, which 64 bits decide (127 t and (k + 1/2) max |t| have at most 32 bits).  A logit is one exact sum times three fp32
numbers, two of them rounded: four roundings of 2^-24 (the sum's, two products', the scales' product) and one of 2^-24 in each scale, then the
type's half step: 8 * 2^-24 + finfo.eps / 2."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def whole(t):
    """(q, scale) of the rows of t in 64 bits."""
    t = t.double()
    top = t.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, torch.round(t * 127.0 / torch.where(top > 0, top, 1.0)), 0.0)
    return q, top[..., 0] / 127.0


def check_numbers(got, t):
    q, s = whole(t)
    assert got.values.dtype == torch.int8 and got.scales.dtype == F32
    assert got.values.shape == t.shape and got.scales.shape == t.shape[:-1]
    assert torch.equal(got.values.double(), q)
    assert ((got.scales.double() - s).abs() <= 2.0 ** -24 * s + 2.0 ** -150).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 4096), (3, 7), (65, 100), (130, 1000), (17, 8195), (2, 131072), (1000, 64)])
def test_rows(rows, cols, dtype):
    from linear_cross_entropy_loss_amd import quantize_rows

    print(f"quantize_rows {rows} {cols} {dtype}", flush=True)
    t = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols)).to(dtype).cuda()
    check_numbers(quantize_rows(t), t)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("H, V", [(1, 1), (7, 3), (64, 1000), (100, 65), (500, 4099), (2048, 300), (129, 64), (8195, 130)])
def test_columns(H, V, dtype):
    from linear_cross_entropy_loss_amd import quantize_weight

    print(f"quantize_weight {H} {V} {dtype}", flush=True)
    At = torch.randn(H, V, generator=torch.Generator().manual_seed(H + V)).to(dtype).cuda()
    got = quantize_weight(At)
    check_numbers(got, At.t())
    tied = quantize_weight(At.t().contiguous().t())  # (stored (V, H))
    assert torch.equal(tied.values, got.values) and torch.equal(tied.scales, got.scales)
    wide = torch.randn(H, V + 9, device="cuda").to(dtype)
    wide[:, 3:V + 3] = At
    cut = quantize_weight(wide[:, 3:V + 3])  # (rows at any element boundary)
    assert torch.equal(cut.values, got.values) and torch.equal(cut.scales, got.scales)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_ties_go_to_the_even_number(dtype):
    from linear_cross_entropy_loss_amd import quantize_rows, quantize_weight

    # a largest magnitude of 127 * 2^e: every half is a number of the type
    steps = torch.arange(-254, 255).double() / 2
    t = torch.cat([steps, torch.tensor([127.0], dtype=torch.float64)]).mul(2.0 ** -6).to(dtype).cuda().repeat(3, 1)
    check_numbers(quantize_rows(t), t)
    check_numbers(quantize_weight(t.t().contiguous()), t)


def test_float32_numbers_next_to_a_border():
    from linear_cross_entropy_loss_amd import quantize_rows

    g = torch.Generator().manual_seed(3)
    top = torch.rand(64, 1, generator=g, dtype=torch.float64).add_(0.5).float()
    border = ((torch.randint(0, 127, (64, 500), generator=g).double() + 0.5) * top.double() / 127.0).float()
    near = [border, torch.nextafter(border, torch.tensor(0.0)), torch.nextafter(border, torch.tensor(9.0))]
    t = torch.cat(near + [-border, top], 1).cuda()
    check_numbers(quantize_rows(t), t)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_the_smallest_and_the_largest_numbers(dtype):
    from linear_cross_entropy_loss_amd import quantize_rows

    t = torch.randn(6, 200, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    t = (t * torch.tensor([1e-40, 1e-38, 1e-31, 1e-29, 1e37, 8e37], dtype=torch.float64)[:, None]).to(dtype).cuda()
    check_numbers(quantize_rows(t), t)


def test_rows_of_zeros_nan_and_infinities():
    from linear_cross_entropy_loss_amd import quantize_rows, quantize_weight, quantized_logits

    t = torch.randn(6, 100, device="cuda", dtype=BF16)
    t[1] = 0
    t[2, 50], t[3, 99], t[4, 0] = math.nan, math.inf, -math.inf
    for got in (quantize_rows(t), quantize_weight(t.t().contiguous())):
        assert got.scales.isnan().tolist() == [False, False, True, True, True, False]
        assert got.scales[1] == 0 and (got.values[1:5] == 0).all()
        x = torch.randn(4, 100, device="cuda", dtype=BF16)
        z = quantized_logits(x, got)
        assert z.isnan().all(0).tolist() == got.scales.isnan().tolist() and (z[:, 1] == 0).all()
    z = quantized_logits(t, quantize_weight(torch.randn(100, 30, device="cuda", dtype=BF16)))
    assert z.isnan().all(1).tolist() == [False, False, True, True, True, False] and z[[0, 1, 5]].isfinite().all()


def check_logits(N, H, V, dtype, out=None, scale=1.0, seed=0):
    from linear_cross_entropy_loss_amd import quantize_weight, quantized_logits

    print(f"quantized_logits {N} {H} {V} {dtype} {out}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(seed + N + H + V)
    x = torch.randn(N, H, generator=g, device="cuda").to(dtype)
    At = (torch.randn(H, V, generator=g, device="cuda") / math.sqrt(H)).to(dtype)
    weight = quantize_weight(At)
    z = quantized_logits(x, weight, scale, out)
    assert z.shape == (N, V) and z.dtype == (out or dtype) and z.is_contiguous()
    (qx, sx), (qw, sw) = whole(x), whole(At.t())
    want = (qx @ qw.t()) * sx[:, None] * sw * scale
    half = torch.finfo(z.dtype).eps / 2
    assert ((z.double() - want).abs() <= (8 * 2.0 ** -24 + half) * want.abs() + (2.0 ** -25 if z.dtype == F16 else 0)).all()
    return x, weight, z


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("N, H, V", [(1, 1, 1), (1, 2048, 5000), (1, 100, 257), (2, 8192, 300), (5, 130, 1001), (16, 64, 1000), (17, 1024, 4097),
                                     (31, 777, 50257), (33, 500, 515), (64, 256, 4096), (100, 48, 129), (129, 2000, 1000), (300, 640, 2051),
                                     (1000, 136, 333)])
def test_logits(N, H, V, dtype):
    check_logits(N, H, V, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("N, H, V", [(1500, 512, 20001), (2100, 1000, 16384), (700, 3000, 30000)])
def test_logits_of_many_tiles(N, H, V, dtype):
    check_logits(N, H, V, dtype)


@pytest.mark.parametrize("N", [1, 8, 40, 300])
def test_types_of_the_result_and_scale(N):
    for out in (BF16, F16, F32):
        check_logits(N, 200, 1111, F16, out=out, scale=0.3)


def test_largest_sums():
    """131072 products of 127 * 127 are 2114060288, and no more fits 31 bits."""
    from linear_cross_entropy_loss_amd import quantize_weight, quantized_logits

    H = 131072
    x = torch.full((3, H), 2.0, device="cuda", dtype=BF16)
    x[1] = -2.0
    z = quantized_logits(x, quantize_weight(torch.full((H, 40), 0.5, device="cuda", dtype=BF16)), dtype=F32)
    want = torch.tensor([H, -H, H], dtype=F32, device="cuda")[:, None].expand(3, 40)
    assert ((z - want).abs() <= 8 * 2.0 ** -24 * H).all()


def test_shapes_strides_and_rows_alone():
    from linear_cross_entropy_loss_amd import Quantized, quantize_weight, quantized_logits

    x, weight, z = check_logits(60, 144, 999, BF16)
    xs = torch.randn(60, 300, device="cuda").to(BF16)
    xs[:, 1:289:2] = x
    assert torch.equal(quantized_logits(xs[:, 1:289:2].view(3, 20, 144), weight).view(60, 999), z)
    xs[:, 3:147] = x
    assert torch.equal(quantized_logits(xs[:, 3:147], weight), z)
    for i in (0, 17, 59):  # a row by itself gives the same bits
        assert torch.equal(quantized_logits(x[i], weight), z[i])
    dense = Quantized(weight.values.contiguous(), weight.scales)
    assert torch.equal(quantized_logits(x, dense), z)
    odd = quantize_weight(torch.randn(45, 77, device="cuda").to(BF16))
    y = torch.randn(5, 45, device="cuda").to(BF16)
    assert torch.equal(quantized_logits(y, Quantized(odd.values.contiguous(), odd.scales)), quantized_logits(y, odd))
    assert quantized_logits(x[:0], weight).shape == (0, 999)
    assert quantized_logits(torch.empty(2, 0, 144, device="cuda", dtype=BF16), weight).shape == (2, 0, 999)
    # what lies behind the end of a row has no effect
    room = torch.full((77, 48), 99, dtype=torch.int8, device="cuda")
    room[:, :45] = odd.values
    assert torch.equal(quantized_logits(y, Quantized(room[:, :45], odd.scales)), quantized_logits(y, odd))


def test_nothing_is_written_beside_the_result():
    """Rows of a larger buffer through the C interface: the elements around them stay."""
    import ctypes

    from linear_cross_entropy_loss_amd import _lib, quantize_weight

    lib = _lib.load()
    for N, V, dtype in ((1, 333, BF16), (20, 257, F16), (40, 1001, F32), (300, 515, BF16)):
        H = 100
        x = torch.randn(N, H, device="cuda").to(dtype)
        weight = quantize_weight(torch.randn(H, V, device="cuda").to(dtype))
        room = torch.full((N + 2, V + 10), 7.0, device="cuda", dtype=dtype)
        b = ctypes.c_size_t(0)
        assert lib.lce_int8_logits_workspace_bytes(N, H, V, ctypes.byref(b)) == 0
        ws = torch.empty(b.value, dtype=torch.uint8, device="cuda")
        out = room[1:-1, 5:-5]
        rc = lib.lce_int8_logits(x.data_ptr(), _lib.dtype_code(dtype), N, H, V, H, weight.values.data_ptr(), weight.values.stride(0),
                                 weight.scales.data_ptr(), 1.0, out.data_ptr(), _lib.dtype_code(dtype), V + 10, ws.data_ptr(), b.value,
                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        kept = room.clone()
        kept[1:-1, 5:-5] = 7.0
        assert (kept == 7.0).all() and not (out == 7.0).all()


def test_compiled_and_captured():
    from linear_cross_entropy_loss_amd import quantize_weight, quantized_logits

    x, weight, z = check_logits(9, 128, 700, BF16)
    At = torch.randn(128, 700, device="cuda").to(BF16)
    torch._dynamo.reset()
    both = torch.compile(lambda x, At: quantized_logits(x, quantize_weight(At), 0.5), backend="aot_eager", fullgraph=True)
    assert torch.equal(both(x, At), quantized_logits(x, quantize_weight(At), 0.5))
    torch._dynamo.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = quantized_logits(x, quantize_weight(At))
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        At.copy_(torch.randn(At.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, quantized_logits(x, quantize_weight(At)))


def test_offsets_past_32_bits():
    """A result of more than 2^31 numbers, and a weight of more than 2^31 bytes: the rows at either end are those that are computed alone."""
    from linear_cross_entropy_loss_amd import quantize_weight, quantized_logits
    from linear_cross_entropy_loss_amd.quantization import Quantized

    x = torch.randn(17000, 64, device="cuda").to(BF16)
    w = quantize_weight(torch.randn(64, 131000, device="cuda").to(BF16))
    print("quantized_logits 17000 x 131000", flush=True)
    z = quantized_logits(x, w)
    for rows in (slice(0, 3), slice(16300, 16500), slice(16999, 17000)):
        assert torch.equal(z[rows], quantized_logits(x[rows], w))
    del z
    H, V = 16400, 131500  # (V, H) int8: 2.16e9 bytes
    for N in (1, 5, 40, 300):
        print(f"quantized_logits {N} x {H} x {V}", flush=True)
        values = torch.randint(-127, 128, (V, H), dtype=torch.int8, device="cuda")
        scales = torch.rand(V, device="cuda")
        x = torch.randn(N, H, device="cuda").to(BF16)
        z = quantized_logits(x, Quantized(values, scales), dtype=F32)
        for cols in (slice(0, 100), slice(V - 600, V)):
            assert torch.equal(z[:, cols], quantized_logits(x, Quantized(values[cols], scales[cols]), dtype=F32))


def test_many_columns_and_rows_past_32_bits():
    from linear_cross_entropy_loss_amd import quantize_rows, quantize_weight

    At = torch.empty(16400, 131500, dtype=BF16, device="cuda").normal_()
    print("quantize_weight 16400 x 131500", flush=True)
    got = quantize_weight(At)
    for cols in (slice(0, 50), slice(131000, 131500)):
        check_numbers(quantize_rows(At[:, cols].t()), At[:, cols].t())
        assert torch.equal(got.values[cols], quantize_rows(At[:, cols].t()).values)
    At = At[:, :131072]
    check_numbers(quantize_rows(At[-3:]), At[-3:])
    assert torch.equal(quantize_rows(At).values[-3:], quantize_rows(At[-3:]).values)


def test_values_that_share_rows_are_copied():
    from linear_cross_entropy_loss_amd import quantized_logits
    from linear_cross_entropy_loss_amd.quantization import Quantized

    x = torch.randn(5, 96, device="cuda").to(BF16)
    row = torch.randint(-127, 128, (1, 96), dtype=torch.int8, device="cuda")
    scales = torch.rand(70, device="cuda")
    got = quantized_logits(x, Quantized(row.expand(70, 96), scales))
    assert torch.equal(got, quantized_logits(x, Quantized(row.repeat(70, 1), scales)))
