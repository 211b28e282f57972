"""GPU (-m gpu): calls of the feed-forward operators that their documentation allows, or that they have to refuse, beyond the sizes
and values of test_gpu_ffn.py.  Tolerances as there: u half a step of the type, E = 2^-24 for every 32-bit operation."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_ffn import DEV, rnd

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------
# what is refused
# ------------------------------------------------------------------------------------------------
def test_forward_derivatives_are_refused():
    """a forward-mode derivative of any argument or gradient would be lost without a word"""
    from hot_amd import ops
    from hot_amd._lib import HotkError
    x, w, W, r, b = rnd(500, 6, 16), rnd(501, 16), rnd(502, 24, 16), rnd(503, 6, 16), rnd(504, 24)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(W)
    with forward_ad.dual_level():
        def d(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: ops.rms_norm(d(x), w), lambda: ops.rms_norm(x, d(w)), lambda: ops.rms_norm(x, w, d(r)), lambda: ops.rms_norm_quantized(d(x), w),
                 lambda: ops.rms_norm_quantized(x, d(w)), lambda: ops.rms_norm_quantized(x, w, d(r)), lambda: ops.quantize_rows(d(x)),
                 lambda: ops.linear_act(d(x), W), lambda: ops.linear_act(x, d(W)), lambda: ops.linear_act(x, W, d(b)),
                 lambda: ops.linear_act(x, W, b, residual=d(rnd(505, 6, 24))), lambda: ops.linear_act(d(x).requires_grad_(True), W),
                 lambda: ops.linear_act_quantized(q, d(s), wq, ws), lambda: ops.linear_act_quantized(q, s, wq, d(ws)),
                 lambda: ops.linear_act_quantized(q, s, wq, ws, d(b), out_dtype=torch.float32)]
        for i, call in enumerate(calls):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(HotkError, match='forward-mode'):
                    call()
                    raise AssertionError(f'call {i} was taken')
        leaf = x.clone().requires_grad_(True)
        for y in (ops.rms_norm(leaf, w), ops.linear_act(leaf, W, act='silu')):
            with pytest.raises(RuntimeError, match='forward-mode'):
                torch.autograd.grad(y, leaf, d(torch.ones_like(y)))
        assert torch.equal(ops.rms_norm(x, w), ops.rms_norm(leaf, w).detach())       # within the level, without a derivative: as ever


def test_tensors_that_stand_for_others_are_refused():
    """in any place: an optional operand without memory would otherwise count as none, a batched gradient as one"""
    from hot_amd import ops
    from hot_amd._lib import HotkError
    from test_ffn_refusals import Wrapped
    x, w, W, b, y = rnd(510, 6, 16), rnd(511, 16), rnd(512, 24, 16), rnd(513, 24), rnd(514, 6, 24)
    kind = torch.ones(6, dtype=torch.uint8, device=DEV)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(W)
    v = Wrapped
    calls = [lambda: ops.rms_norm(v(x), w), lambda: ops.rms_norm(x, v(w)), lambda: ops.rms_norm(x, w, v(x)), lambda: ops.rms_norm(x, w, kind=v(kind)),
             lambda: ops.rms_norm_quantized(x, w, v(x)), lambda: ops.quantize_rows(v(x)), lambda: ops.linear_act(x, v(W)),
             lambda: ops.linear_act(x, W, v(b)), lambda: ops.linear_act(x, W, residual=v(y)), lambda: ops.linear_act_quantized(v(q), s, wq, ws),
             lambda: ops.linear_act_quantized(q, v(s), wq, ws), lambda: ops.linear_act_quantized(q, s, wq, v(ws)),
             lambda: ops.linear_act_quantized(q, s, wq, ws, v(b), out_dtype=torch.float32)]
    for i, call in enumerate(calls):
        with pytest.raises(HotkError, match='plain tensor'):
            call()
            raise AssertionError(f'call {i} was taken')
    leaf = x.clone().requires_grad_(True)
    for z in (ops.rms_norm(leaf, w), ops.linear_act(leaf, W, act='silu')):
        with pytest.raises(RuntimeError, match='plain tensor'):
            torch.autograd.grad(z, leaf, torch.ones(3, *z.shape, device=DEV), is_grads_batched=True)
