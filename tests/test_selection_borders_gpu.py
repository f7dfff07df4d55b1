"""Sampling where a border decides: a bin's border next to zero."""
import pytest
import torch

from test_selection_gpu import check_sample

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
