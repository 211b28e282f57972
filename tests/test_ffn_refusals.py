"""CPU (no GPU): tensors that the feed-forward operators cannot take for what they are, refused before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from hot_amd import ops
from hot_amd._lib import HotkError


def test_forward_derivatives_are_refused():
    x = torch.randn(3, 8)
    calls = [lambda t: ops.rms_norm(t, x[0]), lambda t: ops.rms_norm_quantized(t, x[0]), ops.quantize_rows, lambda t: ops.linear_act(t, x),
             lambda t: ops.linear_act(t, x, act='gelu')]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(HotkError, match='forward-mode'):
                call(dual)
            with torch.no_grad(), pytest.raises(HotkError, match='forward-mode'):
                call(dual)
    for call in calls:
        with pytest.raises(HotkError, match='HIP device'):        # the same tensor without one: the CPU is all that is wrong
            call(x)


class Wrapped(torch.Tensor):
    """a tensor class without memory of its own, as distributed and fake tensors are"""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f'{func} ran')


def test_tensors_that_stand_for_others_are_refused():
    x = torch.randn(3, 4, 8)
    calls = [lambda t: ops.rms_norm(t, torch.ones(8)), lambda t: ops.rms_norm_quantized(t, torch.ones(8)), ops.quantize_rows, lambda t: ops.linear_act(t, torch.ones(5, 8))]
    for call in calls:
        for taken in (lambda: call(Wrapped(x)), lambda: torch.func.vmap(call)(x), lambda: torch.func.jvp(call, (x,), (x,)),
                      lambda: torch.func.grad(lambda t: call(t).sum())(x)):
            with pytest.raises(HotkError, match='plain tensor'):
                taken()
