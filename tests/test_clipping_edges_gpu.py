"""Clipping where calls go wrong easily: norms at the end of float32, and tensors that have no memory of their own."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.pack_auto]

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_a_norm_beyond_float32_is_infinite_and_nothing_is_clipped(dtype):
    from linear_cross_entropy_loss_amd import clip_gradients

    for to in (None, F32):
        for divisor in (1.0, torch.ones((), device="cuda")):
            g = [torch.full((9001,), 3e38, device="cuda").to(dtype), torch.full((5,), -2.0, device="cuda").to(dtype)]
            was = [t.clone() for t in g]
            out = None if to is None else [torch.zeros_like(t, dtype=to) for t in g]
            assert float(clip_gradients(g, 1.0, divisor, out)) == math.inf
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(g if out is None else out, was))
    # by the divisor alone: a norm of 2^127 and one of 2^128, which is no float32
    for divisor, clipped in ((0.5, True), (2.0 ** -2, False)):
        g = torch.full((4,), 2.0 ** 125, device="cuda", dtype=dtype)
        norm = float(clip_gradients(g, 2.0, divisor))
        assert norm == (2.0 ** 126 / divisor if clipped else math.inf)
        assert (g == (1.0 if clipped else 2.0 ** 125 / divisor)).all()


class Wrapped(torch.Tensor):
    """A tensor whose numbers are another's, as those of sharded tensors are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        inner = [a.inner if isinstance(a, Wrapped) else a for a in args]
        return func(*inner, **(kwargs or {}))


def test_tensors_without_memory_of_their_own_are_refused():
    from linear_cross_entropy_loss_amd import clip_gradients

    plain = torch.ones(10, device="cuda")
    sharded = Wrapped(torch.ones(10, device="cuda"))
    for grads, out in (([sharded], None), ([plain, sharded], None), ([plain], [sharded]), ([sharded], [plain])):
        with pytest.raises(ValueError, match="no memory of their own"):
            clip_gradients(grads, 1.0, out=out)
    assert (plain == 1).all() and (sharded.inner == 1).all()


def test_the_same_tensor_twice_is_refused():
    from linear_cross_entropy_loss_amd import clip_gradients

    a = torch.ones(20, 30, device="cuda")
    for grads in ([a, a], [a, a[:, ::2]], [a[:, ::2], a[:, ::2]], [a[:, ::2], a[::2, ::2]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_gradients(grads, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([torch.ones_like(a), torch.ones_like(a)], 1.0, out=[a.t().t(), a])
    assert (a == 1).all()
    clip_gradients([a[:, ::2], a[:, 1::2]], 1.0)  # (side by side)
    norm = math.sqrt(600.0)
    assert ((a * norm - 1).abs() <= 2.0 ** -22).all()


def test_tensors_of_inference_mode():
    """Outside that mode torch refuses to change them; so does this, before anything is written."""
    from linear_cross_entropy_loss_amd import clip_gradients

    with torch.inference_mode():
        given = torch.randn(5000, device="cuda")
        dense, strided = given.clone(), given.clone().view(50, 100)[:, ::2]
        want = [t.clone() for t in (dense, strided)]
        for t, was in zip((dense, strided), want):
            out = torch.empty_like(t)
            assert float(clip_gradients(t, 1.0)) == float(clip_gradients(was, 1.0, out=out)) > 1
            assert torch.equal(t, out)
    kept = [t.clone() for t in (dense, strided)]
    for t, was in zip((dense, strided), kept):
        with pytest.raises(RuntimeError, match="inference"):
            clip_gradients(t, 0.5)
        assert torch.equal(t, was)
        assert abs(float(clip_gradients(t, 0.5, out=torch.zeros(t.shape, device="cuda"))) - 1) <= 2.0 ** -20  # (only read)
