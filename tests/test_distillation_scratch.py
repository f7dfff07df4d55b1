"""Scratch of lce_distill: what the loss plans for the same problem, 16 MiB at least for the sort of the targets, and 4 bytes an entry; and
targets that are sorted a stretch of rows at a time because they are too many for it."""
import pytest
import torch

from linear_cross_entropy_loss_amd import _lib

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _prob(N, H, V, n_chunk, dtype, w_dtype, vh, **kw):
    cols = H if vh else V
    up = lambda v, t: (v + 7) // 8 * 8 if t != F32 else (v + 3) // 4 * 4  # noqa: E731
    return _lib.make_problem(N, H, V, up(H, dtype), up(cols, w_dtype), up(H, dtype), up(cols, w_dtype), dtype, w_dtype, dtype, w_dtype, -1, 1.0,
                             0.0, n_chunk, False, w_layout=_lib.W_VH if vh else _lib.W_HV, **kw)


@pytest.mark.parametrize("pack", [_lib.PACK_AUTO, _lib.PACK_NEVER, _lib.PACK_ALWAYS])
@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_ONE_PASS, _lib.ROUTE_TWO_PASS])
@pytest.mark.parametrize("dtype,w_dtype,vh", [(BF16, BF16, False), (BF16, BF16, True), (F16, F32, False), (F32, F32, False)])
@pytest.mark.parametrize("N,H,V,K,n_chunk", [
    (65536, 64, 4096, 1024, 4096), (1 << 20, 64, 1024, 1024, 4096), (65536, 256, 4096, 128, 4096), (16384, 2048, 131072, 64, 4096),
    (1 << 18, 136, 2048, 512, 1024), (2048, 2048, 16384, 64, 4096), (40000, 1024, 1 << 20, 1024, 64), (1 << 20, 8, 2048, 1024, 64)])
def test_scratch_is_bounded(N, H, V, K, n_chunk, dtype, w_dtype, vh, route, pack):
    """No more than 12.1 GiB for (2^20, 64, 1024, K = 1024), 776 MiB for (65536, 64, 4096, K = 1024): entries by the sort's 8 bytes."""
    p = _prob(N, H, V, n_chunk, dtype, w_dtype, vh, route=route, pack_rows=pack)
    # (hidden sizes up to 128, a backward without a stage: distillation has one, as the loss where rows are packed on demand)
    staged = _prob(N, H, V, n_chunk, dtype, w_dtype, vh, route=route, pack_rows=_lib.PACK_ALWAYS if H <= 128 else pack)
    alone = _lib.forward_workspace_bytes(p)
    loss = max(alone, _lib.forward_backward_workspace_bytes(p), _lib.forward_backward_workspace_bytes(staged), n_chunk * V * 4)
    least, own = 16 << 20, 4 * N * K + 8192
    assert 4 * N * K <= _lib.distill_workspace_bytes(p, K, False) <= max(alone, least) + own
    assert 4 * N * K <= _lib.distill_workspace_bytes(p, K, True) <= max(loss, least) + own


@pytest.mark.gpu
@pytest.mark.pack_auto
@pytest.mark.parametrize("dtype,w_dtype,tied", [(BF16, None, False), (F16, None, True), (BF16, F32, False)])
def test_more_targets_than_are_sorted_at_once(dtype, w_dtype, tied):
    """2100 rows of 1024 targets, rows without any among them: two stretches, the second short; the loss alone is the same."""
    from linear_cross_entropy_loss_amd import linear_distillation
    from test_distillation_gpu import check, make

    N, H, V, K = 2100, 72, 3001, 1024
    x, w, index, logits = make(N, H, V, K, dtype, seed=5, empty=0.05, short=0.01, w_dtype=w_dtype)
    losses = []

    def run(*args):
        losses.append(linear_distillation(*args))
        return losses[0]

    up = 512.0 if dtype == F16 else 1.0
    check((x, w, index, logits), T=1.5, tied=tied, up=up, run=run)
    with torch.no_grad():
        wg = (w.t().contiguous() if tied else w).cuda()
        alone = linear_distillation(x.cuda(), wg.t() if tied else wg, index.cuda(), logits.cuda(), 1.5)
    assert abs(alone.item() - losses[0].item()) <= 64 * 2.0 ** -22 * max(1.0, alone.item())


@pytest.mark.gpu
@pytest.mark.pack_auto
def test_a_row_has_the_same_logits_in_any_stretch():
    """The loss of the rows of several stretches is the mean of the losses of parts of them that are sorted whole."""
    from linear_cross_entropy_loss_amd import linear_distillation
    from test_distillation_gpu import make

    x, w, index, logits = (t.cuda() for t in make(6000, 64, 2003, 700, BF16, seed=6))
    whole = linear_distillation(x, w, index, logits).double()
    parts = torch.stack([linear_distillation(x[i:i + 1000], w, index[i:i + 1000], logits[i:i + 1000]) for i in range(0, 6000, 1000)])
    # (sums of the same fp32 terms in doubles; each loss is rounded once)
    assert (whole - parts.double().mean()).abs() <= 2.0 ** -22 * whole
