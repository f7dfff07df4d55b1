"""Settings of sample_logits and numbers of linear_distillation: which are refused, and by what name."""
import math

import pytest
import torch

from linear_cross_entropy_loss_amd import sample_logits

BAD = [{"temperature": -1.0}, {"temperature": math.nan}, {"temperature": math.inf}, {"top_p": 0.0}, {"top_p": 1.5}, {"top_p": math.nan},
       {"min_p": -0.1}, {"min_p": 2.0}, {"min_p": math.nan}, {"top_k": -3}, {"top_k": 1 << 70}]
# numbers that are none in float32, and no whole ones
BAD_ROUNDED = [{"temperature": 1e39}, {"top_p": 1e-50}, {"top_p": 1.0 + 1e-7}, {"top_k": 2.7}, {"top_k": 0.5}, {"top_k": -0.5},
               {"top_k": math.nan}, {"top_k": math.inf}]


@pytest.mark.parametrize("settings", BAD + BAD_ROUNDED, ids=str)
def test_refused_by_name_before_all_else(settings):
    with pytest.raises(ValueError, match=next(iter(settings))):
        sample_logits(torch.zeros(4, 50), torch.zeros(4), **settings)


# (numbers that float32 rounds to one that is fine)
GOOD = [{}, {"temperature": 0.0}, {"temperature": 3.4028234e38}, {"temperature": 1e-60}, {"top_k": 50}, {"top_k": 50.0}, {"top_k": True},
        {"top_k": 2 ** 63 - 1}, {"top_p": 1.0 + 1e-9}, {"top_p": 1e-40}, {"min_p": -1e-60}, {"min_p": 1},
        {"temperature": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.01}]


@pytest.mark.parametrize("settings", GOOD, ids=str)
def test_taken(settings):
    with pytest.raises(RuntimeError, match="no CPU path"):  # (the next thing that is looked at)
        sample_logits(torch.zeros(4, 50), torch.zeros(4), **settings)


def test_the_library_takes_the_largest_numbers():
    import ctypes

    from linear_cross_entropy_loss_amd import _lib

    largest = torch.finfo(torch.float32).max
    for temperature, status in ((largest, _lib.LCE_OK), (math.inf, _lib.LCE_EINVAL_ARG)):
        s = _lib.LceSampling(temperature, 1.0, 0.0, 0, None, None, None, None)
        assert _lib.load().lce_sample(None, 0, 0, 100, 100, None, ctypes.byref(s), None, None) == status
        p = _lib.make_problem(512, 256, 4096, 256, 4096, 256, 4096, *4 * (torch.bfloat16,), -1, temperature, 0.0, 4096, False)
        size = ctypes.c_size_t()
        assert _lib.load().lce_distill_workspace_bytes(ctypes.byref(p), 8, 1, ctypes.byref(size)) == status


@pytest.mark.parametrize("temperature,scale,name", [(1e39, 1.0, "temperature"), (1e-50, 1.0, "temperature"), (1.0, 1e39, "logit_scale /"),
                                                    (1e30, 1e-30, "logit_scale /"), (1e-30, 1e30, "logit_scale /"), (1.0, math.inf, "logit_scale")])
def test_distillation_names_the_number(temperature, scale, name):
    from linear_cross_entropy_loss_amd import distillation

    with pytest.raises(ValueError, match=name):
        distillation._check_numbers(temperature, scale)
    distillation._check_numbers(1e38, 1e39)  # (what the library gets is the quotient)
    distillation._check_numbers(3.4e38, 1.0)


@pytest.mark.gpu
@pytest.mark.pack_auto
def test_the_largest_temperature():
    from test_distillation_gpu import check, make

    largest = torch.finfo(torch.float32).max
    check(make(70, 64, 300, 7, torch.bfloat16, seed=3, short=0.2), T=largest, scale=largest)
