"""GPU (-m gpu): calls of the feed-forward operators that their documentation allows, or that they have to refuse, beyond the sizes
and values of test_gpu_ffn.py.  Tolerances as there: u half a step of the type, E = 2^-24 for every 32-bit operation."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_ffn import DEV, E, TYPES, act64, floor_of, half_step, hold, rnd, slope64

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


# ------------------------------------------------------------------------------------------------
# activations far from zero
# ------------------------------------------------------------------------------------------------
def column(z, n, dt):
    """operands whose product is z in each of n columns, exactly: one term, times one"""
    return z.to(dt)[:, None].to(DEV), torch.ones(n, 1, dtype=dt, device=DEV)


# gelu(z) = z q, q = erfc(-z / sqrt 2) / 2.  16-bit results: q's fit to 3e-5 of itself below z = -2.6 (q < 0.0047); fp32: to 1.2e-7.
# The exponent z^2 / 2 has up to three roundings, 1.5 z^2 E of the result, and sixteen operations besides.
def gelu_tail(z, dt):
    return 1.2e-7 + (0 if dt == torch.float32 else 3e-5) + (1.5 * z * z + 16) * E


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('M', [33, 400])
def test_gelu_negative_tail(M, dt):
    """relative to its value, down to where the type ends, in both kernels and over 8-bit operands"""
    from hot_amd import ops
    x, w = column(-torch.linspace(2.6, 12.5, M), 24, dt)
    z = x.double().expand(M, 24)
    want = act64(z, 'gelu')
    hold('y', ops.linear_act(x, w, act='gelu'), want, (half_step(dt) + gelu_tail(z, dt)) * want.abs() + floor_of(dt))
    e = (-torch.linspace(2.6, 12.5, M)).to(torch.float8_e4m3fn)[:, None].to(DEV)
    z = e.double().expand(M, 24)
    want = act64(z, 'gelu')
    one = torch.ones(24, device=DEV)
    got = ops.linear_act_quantized(e, torch.ones(M, device=DEV), one[:, None].to(torch.float8_e4m3fn), one, act='gelu', out_dtype=dt)
    hold('8 bits', got, want, (half_step(dt) + gelu_tail(z, dt)) * want.abs() + floor_of(dt))


@pytest.mark.parametrize('M', [33, 400])
def test_gelu_gradient_in_the_negative_tail(M):
    """fp32: slope = q + z exp(-z^2 / 2) / sqrt(2 pi); the second term dominates and has the exponent's roundings too"""
    from hot_amd import ops
    x, w = column(-torch.linspace(2.6, 12.5, M), 1, torch.float32)
    x.requires_grad_(True)
    y = ops.linear_act(x, w, act='gelu')
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    want = slope64(z, 'gelu')
    hold('dx', dx, want, 3 * gelu_tail(z, torch.float32) * want.abs() + floor_of(torch.float32))


@pytest.mark.parametrize('M', [33, 400])
def test_tanh_gradient_far_from_zero(M):
    """fp32: the slope 1 / cosh^2 relative to its value, where 1 - tanh^2 has no digits left; the exponent 2 |z| is rounded once, and
    a dozen operations follow"""
    from hot_amd import ops
    x, w = column(torch.linspace(-40, 40, M), 1, torch.float32)
    x.requires_grad_(True)
    y = ops.linear_act(x, w, act='tanh')
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    hold('dx', dx, z.cosh() ** -2, (2 * z.abs() + 12) * E * z.cosh() ** -2 + floor_of(torch.float32))
