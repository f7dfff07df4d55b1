"""Sampling and logsumexp where a border decides: a bin's border next to zero, weights next to half a place, sums of very many terms."""
import math

import pytest
import torch

from test_selection_gpu import BF16, F16, F32, check_sample

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

# The largest value and the temperature of a row whose zeros weigh 2^-(85/80) and 2^-(102/80), with 80 bins of the weight to an octave:
# top * 80 * log2(e) / T is within 2^-53 of a whole number, so that a border worked out in doubles is off zero to either side.
AT_ZERO = [(12295127 * 2.0 ** -23, 16694700 * 2.0 ** -23), (12295127 * 2.0 ** -23, 13912250 * 2.0 ** -23),
           (12295127 * 2.0 ** -13, 13912250 * 2.0 ** -13), (12295127 * 2.0 ** -40, 16694700 * 2.0 ** -40)]


@pytest.mark.parametrize("N", [1, 300])
@pytest.mark.parametrize("top,temperature", AT_ZERO)
def test_a_bin_border_at_zero(top, temperature, N):
    """Values next to zero lie closer together than differences to the largest value are known."""
    V = 9000
    z = torch.zeros(4, V)
    z[0, 1::2] = -0.0
    z[1, 100:] = -1e30 * top  # (few enough for a list)
    z[2] = 2.0 ** -80 * top * torch.randn(V, generator=torch.Generator().manual_seed(1))
    z[3, 3000:] = 2.0 ** -1.5 * top
    z[:, 5] = top
    u = torch.tensor([0.5, 0.625, 0.7, 0.9])
    for row in range(4):
        for settings in ({}, {"top_p": 0.75}, {"top_k": 3001}, {"top_k": 6001, "top_p": 0.9}, {"min_p": 0.25}):
            check_sample(z[row:row + 1].expand(N, V), u[row:row + 1].expand(N), z[row:row + 1].cuda().expand(N, V), temperature=temperature,
                         **settings)


def fixed_point_token(z, u, temperature):
    """The definition with weights as whole multiples of 2^-b, b = min(50, 62 - ceil(log2 V)), in exact sums; one row, no filter."""
    bits = min(50, 62 - math.ceil(math.log2(z.numel())))
    order = torch.sort(z.double(), descending=True, stable=True)
    w = torch.round(torch.exp((order.values - order.values[0]) / temperature) * 2.0 ** bits).long()
    upto = torch.cumsum(w, 0)
    target = min(int(u * float(upto[-1])), int(upto[-1]) - 1)
    return order.indices[(upto > target).to(torch.uint8).argmax()].item()


@pytest.mark.parametrize("N", [1, 300])
@pytest.mark.parametrize("dtype,V,u", [(F32, 1 << 20, 1 - 2.0 ** -24), (F32, 5000, 1.0), (BF16, 5000, 1.0), (F16, 12000, 1.0), (BF16, 20000, 1.0),
                                       (F16, 40000, 1.0)])
def test_weights_next_to_half_a_place(dtype, V, u, N):
    """What is above half a place counts as one, what is below as none, whichever way a row is done.  (u = 1 takes the last column with
    a weight; a million columns of half a place are 2^-22 of the whole, which a number below 1 reaches.)"""
    from linear_cross_entropy_loss_amd import sample_logits

    bits = min(50, 62 - math.ceil(math.log2(V)))
    # weights of the others by their logarithm: -(bits + 1) and 2^-11 more or less, 3e-4 of half a place
    for more in (2.0 ** -11, -(2.0 ** -11)):
        temperature = torch.tensor(64.0 * 1.4426950408889634 / (bits + 1 - more)).item()
        z = torch.full((V,), -64.0).to(dtype)
        z[V // 3] = 0.0
        got = sample_logits(z.cuda().expand(N, V), torch.full((N,), u, device="cuda"), temperature=temperature).cpu()
        print(f"{dtype} V={V} N={N} {more}: {got[0].item()}", flush=True)
        assert torch.equal(got, torch.full((N,), fixed_point_token(z, u, temperature)))


@pytest.mark.parametrize("N", [1, 300])
@pytest.mark.parametrize("dtype,V", [(BF16, (1 << 22) + 5), (F16, 1 << 23), (F32, (1 << 22) + 5), (F32, 131072), (BF16, 50257)])
def test_lse_of_long_flat_rows(dtype, V, N):
    """A term is off by 2 units of 2^-24 and |z - max| <= 2 more; an fp32 sum of at most 130 of them by 65 on top, all to one side; the rest
    is in doubles and rounded once."""
    from linear_cross_entropy_loss_amd import top_logits

    for value in (-1.0986, -0.4055, -1.9, -0.01):
        z = torch.full((1, V), value, device="cuda").to(dtype)
        z[0, 7] = 0.0
        ref = torch.logsumexp(z.double(), 1).item()
        for k in (10, 700):
            lse = top_logits(z.expand(N, V), k)[2].cpu().double()
            print(f"{dtype} V={V} N={N} k={k} {value}: off by {(lse[0].item() - ref):.2e}", flush=True)
            assert ((lse - ref).abs() <= 2.0 ** -24 * (70 + abs(ref))).all()
