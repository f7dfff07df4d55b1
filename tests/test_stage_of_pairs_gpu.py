"""Gradients of fp32 tensors entry by entry, on the route that stages dz as pairs: every entry of the stage counts, not their norm.

An entry of dW is a sum over the rows of x dz.  A pair has 16 bits of mantissa: each factor is off by 2^-17, the product of the lower halves
is left out, the softmax is off by what its logit is off, 2^-16 sum |x| |w| <= 2^-16 * 4 for the hidden sizes here.  Together less than
2^-13 of sum |x| |dz|; a stage entry that is missing is a whole term of 700, each about as large as another."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(x, w, q, kept):
    xd, wd = x.detach().double(), w.detach().double()
    dz = (torch.softmax(xd @ wd, 1) - q) * (kept[:, None] / kept.sum())
    return xd.t().contiguous() @ dz, xd.t().abs().contiguous() @ dz.abs(), dz @ wd.t().contiguous(), dz.abs() @ wd.t().abs().contiguous()


@pytest.mark.parametrize("N,H,V", [(725, 9, 8490), (944, 15, 4228), (1104, 6, 7164), (851, 2, 8674), (600, 9, 7639), (670, 57, 7680)])
def test_every_entry_counts(N, H, V):
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss, linear_distillation, ops

    for seed in range(8):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(N, H, generator=g, device="cuda").requires_grad_(True)
        module = LinearCrossEntropyLoss(H, V, ignore_index=-1, device="cuda")
        with torch.no_grad():
            module.weight.copy_(torch.randn(H, V, generator=g, device="cuda") / math.sqrt(H))
        index = torch.randint(0, V, (N, 3), generator=g, device="cuda")
        index[torch.rand(N, generator=g, device="cuda") < 0.1] = -1
        kept = index[:, 0] >= 0
        token = ops.one_pass.set(False)
        try:
            labels = torch.autograd.grad(module(x, index[:, 0]), (x, module.weight))
            teacher = torch.autograd.grad(linear_distillation(x, module.weight, index, torch.zeros(N, 3, device="cuda")), (x, module.weight))
        finally:
            ops.one_pass.reset(token)
        print(f"pairs N={N} H={H} V={V} seed={seed}", flush=True)
        for (dx, dw), entries in ((labels, index[:, :1]), (teacher, index)):
            q = torch.zeros(N, V, dtype=torch.float64, device="cuda").scatter_add_(
                1, entries.clamp(min=0), torch.full(entries.shape, 1.0 / entries.shape[1], dtype=torch.float64, device="cuda") * kept[:, None])
            ref_dw, most_dw, ref_dx, most_dx = _reference(x, module.weight, q, kept)
            assert ((dw.double() - ref_dw).abs() <= 2.0 ** -13 * most_dw).all()
            assert ((dx.double() - ref_dx).abs() <= 2.0 ** -13 * most_dx).all()
