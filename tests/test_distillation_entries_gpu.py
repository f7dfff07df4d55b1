"""Distillation's gradients entry by entry: targets of small probability and columns of small softmax count like any others.

With h half a step of the type (bf16 2^-8, fp16 2^-11), an entry of dW is a sum over the rows of x dz, where dz = (softmax - q) c has been rounded
twice at most (h each) and the sum once.  Softmax and q themselves are fp32: a logit is off by 2^-24 of the sums of |x| |w| and of lse that
it comes from, some 32 units of 2^-24 for logits below 16, and so is softmax, relatively; q by 8 units (a difference, an exponential, a
sum, a quotient).  That is, with a hundredth of h for products of these,
    |error| <= 2.03 h sum |x| |dz| + 1.01 h |dW| + sum |x| (2^-19 softmax + 2^-21 q) c,
and for dx alike.  fp32 tensors are pairs of bf16: 2^-17 for each of the factors and of dz, 2^-16 for the product of lower halves that is left
out, and a logit off by 2^-16 sum |x| |w| <= 2^-16 * 16; 6 * 2^-17 sum |x| |dz| and 2^-12 softmax.  fp16 numbers below its normal range are off by
2^-25 times the factor that they are staged with, 2^-10, and in dW by 2^-25."""
import math

import pytest
import torch

from test_distillation_gpu import BF16, F16, F32, make

pytestmark = pytest.mark.gpu

HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.mark.parametrize("one_pass", [False, "always"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,H,V,K", [(1, 64, 500, 7), (1, 64, 3001, 300), (5, 72, 1000, 40), (300, 40, 900, 9), (260, 136, 5000, 1024)])
def test_entries(N, H, V, K, dtype, one_pass):
    from linear_cross_entropy_loss_amd import linear_distillation, ops

    x, w, index, logits = (t.cuda() for t in make(N, H, V, K, dtype, seed=51, short=0.1 if N > 1 else 0.0))
    x.requires_grad_(True)
    w.requires_grad_(True)
    up = 512.0 if dtype == F16 else 1.0  # (a power of two: no rounding of its own)
    print(f"entries N={N} H={H} V={V} K={K} {dtype} {one_pass}", flush=True)
    token = ops.one_pass.set(one_pass)
    try:
        dx, dw = torch.autograd.grad(linear_distillation(x, w, index, logits) * up, (x, w))
    finally:
        ops.one_pass.reset(token)
    xd, wd = x.detach().double(), w.detach().double()
    there = index >= 0
    kept = there.any(1)
    c = (kept * (up / kept.sum()))[:, None]
    t = torch.where(there, logits.double(), -math.inf)
    t = torch.where(there, torch.exp(t - torch.where(kept, t.amax(1), 0.0)[:, None]), 0.0)
    q = torch.zeros(N, V, dtype=torch.float64, device="cuda").scatter_add_(1, index.clamp(min=0), t / torch.where(kept, t.sum(1), 1.0)[:, None])
    z = xd @ wd
    assert z.abs().max() < 16
    p = torch.softmax(z, 1)
    dz = (p - q) * c
    if dtype == F32:
        off, last = 6 * 2.0 ** -17 * dz.abs() + (2.0 ** -12 * p + 2.0 ** -21 * q) * c, 2.0 ** -24
    else:
        off, last = 2.03 * HALF[dtype] * dz.abs() + (2.0 ** -19 * p + 2.0 ** -21 * q) * c, 1.01 * HALF[dtype]
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    off = off + tiny * 2.0 ** -10 * c
    for got, ref, most in ((dw, xd.t().contiguous() @ dz, xd.t().abs().contiguous() @ off), (dx, dz @ wd.t().contiguous(), off @ wd.t().abs().contiguous())):
        ratio = ((got.double() - ref).abs() / (most + last * ref.abs() + tiny * up)).max().item()
        print(f"  {ratio:.3f} of what it may be off", flush=True)
        assert ratio <= 1.0
