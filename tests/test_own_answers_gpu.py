"""One step of training on a model's own answers, as the operators are used together: logits of the 8-bit weight, a token drawn from
each row, its log-probability under the weight itself, the gradients of a policy's objective, clipped."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_step(dtype):
    from linear_cross_entropy_loss_amd import LinearCrossEntropyLoss, clip_gradients, quantized_logits, sample_logits, top_logits

    torch.manual_seed(1)
    N, H, V = 300, 136, 1003
    trunk = torch.nn.Linear(40, H, device="cuda", dtype=dtype)
    head = LinearCrossEntropyLoss(H, V, device="cuda", dtype=dtype, ignore_index=-1)
    given = torch.randn(N, 40, device="cuda", dtype=dtype)
    factor = 1024.0 if dtype == torch.float16 else 1.0

    with torch.no_grad():
        logits = quantized_logits(trunk(given), head.quantize())
        tokens = sample_logits(logits, torch.rand(N, device="cuda"), temperature=0.9)
    assert ((tokens >= 0) & (tokens < V)).all()
    # (8 bits keep a logit's place: what is drawn greedily is among the first of the weight's own logits)
    exact = trunk(given).double() @ head.weight.double()
    first = sample_logits(logits, torch.rand(N, device="cuda"), temperature=0.0)
    assert torch.equal(first, top_logits(logits, 1)[1][:, 0])
    gap = exact.amax(1) - exact.gather(1, first[:, None])[:, 0]
    # a number is off by half a step, 1/254 of its row's largest: by Cauchy-Schwarz a logit by (|x| |w| over all rows and columns) twice that
    x, w = trunk(given).double(), head.weight.double()
    off = (x.abs().amax(1) / 254 * math.sqrt(H) * w.norm(dim=0).max() + x.norm(dim=1) * math.sqrt(H) * w.abs().max() / 254 * (1 + 1 / 127)
           + exact.abs().amax(1) * torch.finfo(dtype).eps)
    assert (gap <= 2 * off).all()
    tokens[:30] = -1  # (prompts)
    advantage = torch.randn(N, device="cuda")

    logp = head.log_probs(trunk(given), tokens)
    loss = -(advantage * logp).sum() / 270
    (loss * factor).backward()
    grads = [p.grad for p in (*trunk.parameters(), head.weight)]
    was = [g.double() / factor for g in grads]
    norm = clip_gradients(grads, 0.01, divisor=factor)
    want = math.sqrt(sum(float((g * g).sum()) for g in was))
    assert want > 0.01 and abs(float(norm) - want) <= 2.0 ** -23 * want
    for g, b in zip(grads, was):
        assert ((g.double() - b * (0.01 / want)).abs() <= (2.0 ** -23 + torch.finfo(dtype).eps / 2) * (b * (0.01 / want)).abs() + 2.0 ** -25).all()

    # the gradients of the definition in 64 bits
    t64 = [p.detach().double().requires_grad_(True) for p in (*trunk.parameters(), head.weight)]
    hidden = (given.double() @ t64[0].t() + t64[1])
    hidden = hidden + (trunk(given).detach().double() - hidden).detach()  # (the activations as they were rounded)
    p = torch.log_softmax(hidden @ t64[2], 1).gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    (-(advantage.double() * torch.where(tokens >= 0, p, 0.0)).sum() / 270).backward()
    for b, t in zip(was, t64):
        # (dz, dx, dW and the trunk's gradients rounded once each, and its products' operand dx)
        assert (b - t.grad).norm() <= 5 * torch.finfo(dtype).eps / 2 * t.grad.norm()
