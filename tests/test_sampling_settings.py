"""Settings of sample_logits, numbers of top_logits and linear_distillation: which are refused, eager and compiled, and that numbers
reach the library as numbers."""
import math

import pytest
import torch

from linear_cross_entropy_loss_amd import sample_logits, selection, top_logits

BAD = [{"temperature": -1.0}, {"temperature": math.nan}, {"temperature": math.inf}, {"top_p": 0.0}, {"top_p": 1.5}, {"top_p": math.nan},
       {"min_p": -0.1}, {"min_p": 2.0}, {"min_p": math.nan}, {"top_k": -3}, {"top_k": 1 << 70}]
# numbers that are none in float32, and no whole ones
BAD_ROUNDED = [{"temperature": 1e39}, {"top_p": 1e-50}, {"top_p": 1.0 + 1e-7}, {"top_k": 2.7}, {"top_k": 0.5}, {"top_k": -0.5},
               {"top_k": math.nan}, {"top_k": math.inf}]


@pytest.mark.parametrize("settings", BAD + BAD_ROUNDED, ids=str)
def test_refused_by_name_before_all_else(settings):
    with pytest.raises(ValueError, match=next(iter(settings))):
        sample_logits(torch.zeros(4, 50), torch.zeros(4), **settings)


@pytest.mark.parametrize("k", [0, 0.5, 2.7, 51, 1e30, math.nan, math.inf])
def test_top_logits_takes_whole_numbers(k):
    with pytest.raises(ValueError, match="k must be in 1"):
        top_logits(torch.zeros(4, 50), k)
    with pytest.raises(RuntimeError, match="no CPU path"):
        top_logits(torch.zeros(4, 50), 7.0)


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


@pytest.mark.parametrize("settings", BAD + BAD_ROUNDED, ids=str)
def test_compiled_refuses_the_same(settings):
    torch.compiler.reset()
    run = torch.compile(lambda z, u: sample_logits(z, u, **settings), backend="eager")
    with pytest.raises(ValueError, match=next(iter(settings))):
        run(torch.zeros(4, 50), torch.zeros(4))


def test_compiled_calls_hand_numbers_over_as_numbers(monkeypatch):
    """One operator call, no tensor made of a number; tensors by row beside numbers."""
    seen = []

    def record(*args):
        seen.append(args)
        return args[0].new_zeros(args[0].shape[:-1], dtype=torch.int64)

    monkeypatch.setattr(selection, "_op_sample_logits", torch.compiler.allow_in_graph(record))
    z, u, rows = torch.zeros(4, 50), torch.zeros(4), torch.ones(4)
    for settings in ({}, {"temperature": 0.0}, {"temperature": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.01}, {"temperature": rows, "top_k": 40}):
        torch.compiler.reset()
        seen.clear()
        torch.compile(lambda a, b: sample_logits(a, b, **settings), backend="eager", fullgraph=True)(z, u)
        by_row, numbers = seen[-1][2:6], seen[-1][6:]
        assert [isinstance(t, torch.Tensor) for t in by_row] == [settings.get("temperature") is rows, False, False, False]
        given = {**settings, "temperature": 1.0} if settings.get("temperature") is rows else settings
        assert numbers == tuple(given.get(name, default) for name, default in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))


@pytest.mark.gpu
@pytest.mark.pack_auto
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_on_the_gpu(dtype):
    """Tokens and refusals of compiled calls; greedy decoding and a short top_k take one kernel and allocate the tokens alone."""
    z = torch.randn(6, 20011, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    u = torch.rand(6, generator=torch.Generator().manual_seed(2)).cuda()
    by_row = torch.tensor([0.0, 0.5, 1.0, 1.5, 0.2, 2.0]).cuda()
    for settings in ({}, {"temperature": 0.0}, {"top_k": 30}, {"temperature": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.01}, {"top_p": 0.5},
                     {"temperature": by_row, "top_k": 40}, {"temperature": by_row[1], "top_k": 40, "top_p": by_row.clamp(0.1, 1.0)}):
        torch.compiler.reset()
        run = torch.compile(lambda a, b: sample_logits(a, b, **settings), fullgraph=True)
        assert torch.equal(run(z, u), sample_logits(z, u, **settings))
        if any(isinstance(v, torch.Tensor) for v in settings.values()):
            continue
        torch.cuda.synchronize()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            run(z, u)
            torch.cuda.synchronize()
        kernels = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA and "sample" in e.name.lower()]
        others = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA and "sample" not in e.name.lower()]
        assert len(kernels) == 1 and not others, (kernels, others)
        if settings.get("temperature") == 0.0 or settings.get("top_k"):
            assert "sample_top_kernel" in kernels[0]
    for settings in BAD + BAD_ROUNDED:
        torch.compiler.reset()
        with pytest.raises(ValueError):
            torch.compile(lambda a, b: sample_logits(a, b, **settings))(z, u)


@pytest.mark.gpu
@pytest.mark.pack_auto
def test_compiled_with_changing_numbers():
    """Numbers that are arguments of the compiled function, which it takes for symbols from the second call on."""
    torch.compiler.reset()
    z = torch.randn(4, 5000, generator=torch.Generator().manual_seed(4)).cuda()
    u = torch.rand(4, generator=torch.Generator().manual_seed(5)).cuda()
    run = torch.compile(lambda a, b, t, k, p: sample_logits(a, b, t, k, p), fullgraph=True)
    for t, k, p in ((1.0, 5, 0.9), (0.5, 6, 0.9), (0.25, 7, 0.8), (0.0, 0, 1.0), (2.0, 1000, 1.0)):
        assert torch.equal(run(z, u, t, k, p), sample_logits(z, u, t, k, p))
