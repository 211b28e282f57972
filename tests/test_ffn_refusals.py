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
