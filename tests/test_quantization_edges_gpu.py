"""Numbers of 8 bits where calls go wrong easily: through the C interface with row strides of the caller's own choice, with more rows than one
launch takes, and with weights that were not laid out here."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def quantize(call, src, depth, others, ld, ldq):
    """lce_quantize_rows or lce_quantize_columns into rows of ldq bytes that hold 77, between two rows that stay as they are."""
    from linear_cross_entropy_loss_amd import _lib

    lib = _lib.load()
    room = torch.full((others + 2, ldq), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((others + 2,), 5.0, device="cuda")
    rows, cols = (others, depth) if call == "lce_quantize_rows" else (depth, others)
    rc = getattr(lib, call)(src.data_ptr(), _lib.dtype_code(src.dtype), rows, cols, ld, room[1:].data_ptr(), ldq, scales[1:].data_ptr(),
                            torch.cuda.current_stream().cuda_stream)
    _lib.raise_for_status(rc, call)
    assert (room[0] == 77).all() and (room[-1] == 77).all() and scales[0] == 5.0 and scales[-1] == 5.0
    return room[1:-1], scales[1:-1]


def strides(depth):
    least = -(-depth // 16) * 16
    return sorted({least, least + 16, 2 * least + 512, 4096, 9008, 1 << 18} - set(range(0, least, 16)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("rows", [3, 1500])
@pytest.mark.parametrize("cols", [1, 17, 100, 300, 700, 1000, 2100, 5000])
def test_rows_of_any_stride(rows, cols, dtype):
    from linear_cross_entropy_loss_amd import quantize_rows

    t = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols)).to(dtype).cuda()
    want = quantize_rows(t)
    for ldq in strides(cols):
        print(f"lce_quantize_rows {rows} {cols} {dtype} ldq {ldq}", flush=True)
        q, scales = quantize("lce_quantize_rows", t, cols, rows, cols, ldq)
        assert torch.equal(q[:, :cols], want.values) and torch.equal(scales, want.scales)
        assert not q[:, cols:].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("others", [5, 64, 130])
@pytest.mark.parametrize("depth", [1, 64, 100, 200, 300, 1000, 1100, 2100, 4097])
def test_columns_of_any_stride(depth, others, dtype):
    from linear_cross_entropy_loss_amd import quantize_weight

    At = torch.randn(depth, others, generator=torch.Generator().manual_seed(depth + others)).to(dtype).cuda()
    want = quantize_weight(At)
    for ldq in strides(depth):
        print(f"lce_quantize_columns {depth} {others} {dtype} ldq {ldq}", flush=True)
        q, scales = quantize("lce_quantize_columns", At, depth, others, others, ldq)
        assert torch.equal(q[:, :depth], want.values) and torch.equal(scales, want.scales)
        assert not q[:, depth:].any()


@pytest.mark.parametrize("N", [1, 5, 40, 300])
def test_values_of_rows_wider_than_the_library_takes_are_copied(N):
    from linear_cross_entropy_loss_amd import Quantized, quantize_weight, quantized_logits

    x = torch.randn(N, 100, device="cuda").to(BF16)
    weight = quantize_weight(torch.randn(100, 333, device="cuda").to(BF16))
    for ld in ((1 << 18), (1 << 18) + 16, 1 << 20):
        wide = torch.full((333, ld), 99, dtype=torch.int8, device="cuda")
        wide[:, :100] = weight.values
        assert torch.equal(quantized_logits(x, Quantized(wide[:, :100], weight.scales)), quantized_logits(x, weight))


def windows(n):
    """Rows at both ends and around every 2^21-th."""
    at = {0, n - 40} | {i - 20 for i in range(1 << 21, n - 40, 1 << 21)}
    return [slice(i, i + 40) for i in sorted(at)]


# (a launch has fewer than 2^32 threads: 16, 64 and 256 of them to a row, by its length)
@pytest.mark.parametrize("rows, cols, dtype", [((1 << 28) + 77, 8, BF16), ((1 << 26) + 77, 520, F32), ((1 << 24) + 77, 2100, F32)], ids=str)
def test_more_rows_than_a_launch_takes(rows, cols, dtype):
    """Rows that begin one number after another: a source that fits."""
    from linear_cross_entropy_loss_amd import quantize_rows

    src = torch.randn(rows + cols - 1, device="cuda", dtype=F32).to(dtype)
    ldq = -(-cols // 16) * 16
    print(f"lce_quantize_rows {rows} {cols} {dtype}", flush=True)
    q, scales = quantize("lce_quantize_rows", src, cols, rows, 1, ldq)
    for part in windows(rows):
        want = quantize_rows(src[part.start:part.stop + cols - 1].unfold(0, cols, 1))
        assert torch.equal(q[part, :cols], want.values) and torch.equal(scales[part], want.scales) and not q[part, cols:].any()


def test_more_columns_than_a_launch_takes():
    from linear_cross_entropy_loss_amd import quantize_rows

    cols = 1 << 30
    src = torch.empty(cols, device="cuda", dtype=BF16).normal_()
    print(f"lce_quantize_columns 1 {cols}", flush=True)
    q, scales = quantize("lce_quantize_columns", src, 1, cols, cols, 16)
    for part in windows(cols)[::16] + windows(cols)[-1:]:
        want = quantize_rows(src[part, None])
        assert torch.equal(q[part, :1], want.values) and torch.equal(scales[part], want.scales) and not q[part, 1:].any()
