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


SMOOTH = ['gelu', 'tanh', 'silu']


def slope64_far(z, act):
    """slopes in 64 bits that keep their digits where the activation saturates"""
    s = torch.sigmoid(z)
    return {'gelu': lambda: slope64(z, 'gelu'), 'tanh': lambda: z.cosh() ** -2, 'silu': lambda: s * (1 + z * torch.sigmoid(-z))}[act]()


def code_error(s, dt):
    """half a step of the 16-bit code of a slope: 2^-15 from 1/16 up; below, the code is 21504 (16 |s|)^(1/n), whose half step is
    n / (2 code) of s (a tenth more for the curve within it)"""
    a, n = s.abs(), 8 if dt == torch.float16 else 16
    return torch.where(a >= 1 / 16, torch.full_like(a, 2.0 ** -15), 1.1 * a * n / (2 * 21504 * (16 * a) ** (1 / n)).clamp_min(1e-300))


def slope_error(z, s, act):
    """a 16-bit slope as computed: gelu's fit to 3e-5 of q (below |slope|, |z| > 2.6), a few operations next to an exponent that is
    rounded up to three times; where a slope crosses zero or q is large, 32-bit operations of size one"""
    return ((3e-5 if act == 'gelu' else 0) + (1.5 * z * z + 2 * z.abs() + 32) * E) * s.abs() + torch.where(z.abs() < 2.7, 1e-6, 0.)


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('act', SMOOTH)
@pytest.mark.parametrize('M', [33, 400])
def test_gradients_of_saturated_units(M, act, dt):
    """|z| up to 12: the gradient relative to its value, down to where the type ends"""
    from hot_amd import ops
    x, w = column(torch.linspace(-12, 12, M), 1, dt)
    z = x.double()
    s = slope64_far(z, act)
    for scale in (1., 256.):                       # (a scaled loss lifts what fp16 could not hold)
        leaf, b = x.clone().requires_grad_(True), torch.zeros(1, dtype=dt, device=DEV, requires_grad=True)
        y = ops.linear_act(leaf, w, b, act=act)
        dx, db = torch.autograd.grad(y, (leaf, b), torch.full_like(y, scale))
        want, off = scale * s, scale * (code_error(s, dt) + slope_error(z, s, act))
        hold('dx', dx, want, half_step(dt) * (want.abs() + off) + off + 2 * floor_of(dt))
        hold('db', db, want.sum(0), half_step(dt) * want.sum(0).abs() + off.sum(0) + (M + 8) * E * want.abs().sum(0) + floor_of(dt))


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('act,bias', [('silu', -10.), ('tanh', 6.), ('tanh', -6.), ('gelu', -4.5)])
@pytest.mark.parametrize('M,N,K', [(900, 40, 160), (4096, 64, 160)])
def test_weight_gradients_of_saturated_units(M, N, K, act, bias, dt):
    """a layer whose units sit far from zero: dx and dw are off by the roundings of dz (one, where the product is long) and of the
    result, each at most 0.58 u as a whole, and by the slope's code"""
    from hot_amd import ops
    x, w, b = rnd(520, M, K, dt=dt), rnd(521, N, K, dt=dt, scale=0.5 * K ** -0.5), torch.full((N,), bias, dtype=dt, device=DEV)
    dy = rnd(522, M, N, dt=dt, scale=1. if dt == torch.bfloat16 else 4096.)
    z = x.double() @ w.double().t() + b.double()
    s = slope64_far(z, act)
    dz = dy.double() * s
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_act(*leaves, act=act), leaves, dy)
    u = 0.58 * half_step(dt)
    code = float((dy.double() * code_error(s, dt)).norm() / dz.norm()) * 0.58 + float(((K + 8) * E * z.abs() + 1e-5).max())
    for what, got, want, roundings in (('dx', dx, dz @ w.detach().double(), 2), ('dw', dw, dz.t() @ x.detach().double(), 2), ('db', db, dz.sum(0), 1)):
        assert float((got.double() - want).norm() / want.norm()) <= (roundings * u * u + code * code) ** 0.5, what


def test_piecewise_linear_slopes_are_exact():
    from hot_amd import ops
    for dt in (torch.bfloat16, torch.float16):
        x, w = column(torch.tensor([-3., -1e-3, 0., 1e-3, 5.]), 1, dt)
        for act, low in (('relu', 0.), ('leakyrelu', 0.01)):
            leaf = x.clone().requires_grad_(True)
            dx, = torch.autograd.grad(ops.linear_act(leaf, w, act=act), leaf, torch.ones(5, 1, dtype=dt, device=DEV))
            assert torch.equal(dx[:, 0], torch.tensor([low, low, low, 1., 1.]).to(dt).to(DEV))


# ------------------------------------------------------------------------------------------------
# what saved-tensor hooks give back
# ------------------------------------------------------------------------------------------------
def kept_leaves(M, K, N, dt, clone=False):
    """operands that the forward pass copies (K no whole pieces, transposed), or takes in place"""
    return [rnd(530, M, K + 9, dt=dt)[:, 3:K + 3], rnd(531, K, N, dt=dt).t(), rnd(532, N, dt=dt), rnd(533, M, N, dt=dt)]


def kept_gradients(M, K, N, dt, mask):
    from hot_amd import ops
    x, w, b, r = [t.detach().requires_grad_(True) for t in kept_leaves(M, K, N, dt)]
    kind = (torch.arange(M, device=DEV) % 3).to(torch.uint8) if mask else None
    y = ops.linear_act(x, w, b, act='silu', residual=r)
    z, h = ops.rms_norm(x, w[0], x, kind=kind)
    return lambda: torch.autograd.grad((y, z, h), (x, w, b, r), (rnd(534, M, N, dt=dt), rnd(535, M, K, dt=dt), rnd(536, M, K, dt=dt)))


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mask', [False, True])
@pytest.mark.parametrize('M,K,N', [(3, 742, 36), (70, 37, 24), (65, 64, 40), (1100, 40, 24)])
def test_kept_tensors_in_another_layout(M, K, N, mask, dt):
    """the same values at other strides: transposed storage, every second element of a row"""
    def unpack(t):
        if t.dim() == 2 and t.size(0) > 1:
            return t.t().contiguous().t()
        return torch.stack((t, torch.zeros_like(t)), -1)[..., 0]
    want = kept_gradients(M, K, N, dt, mask)()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        got = kept_gradients(M, K, N, dt, mask)()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('change', [lambda t: t.to(torch.float64), lambda t: t[:-1], lambda t: t.cpu(), lambda t: torch.cat((t, t))])
def test_kept_tensors_that_are_others_are_refused(change):
    for which in range(7):                       # x, w, slopes of the product; stream, statistics, weight, kind of the norm
        count = [0]

        def unpack(t):
            count[0] += 1
            return change(t) if count[0] == which + 1 else t
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            gradients = kept_gradients(70, 37, 24, torch.float32, True)
            with pytest.raises(RuntimeError, match='expected|kept for the backward pass|is on'):
                gradients()
                raise AssertionError(f'tensor {which} was taken')


# ------------------------------------------------------------------------------------------------
# the precision of dz
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,N,K', [(50, 200, 130), (2000, 130, 72), (4096, 264, 136), (300, 1040, 1000)])
def test_parts_of_dz(M, N, K, dt):
    """whatever the size: in two parts the result's rounding is left (uniform in half a step, 0.58 u as a whole at most), in one
    dz's beside it (0.82 u); None is one of the two, by the size"""
    from hot_amd import ops
    x, w, b, dy = rnd(540, M, K, dt=dt), rnd(541, N, K, dt=dt, scale=K ** -0.5), rnd(542, N, dt=dt), rnd(543, M, N, dt=dt)
    dz = dy.double() * slope64(x.double() @ w.double().t() + b.double(), 'gelu')
    want = (dz @ w.double(), dz.t() @ x.double())
    x.requires_grad_(True), w.requires_grad_(True)
    got = {parts: torch.autograd.grad(ops.linear_act(x, w, b, act='gelu', dz_parts=parts), (x, w), dy) for parts in (1, 2, None)}
    for parts, most in ((1, 0.85), (2, 0.62)):
        for what, g, v in zip(('dx', 'dw'), got[parts], want):
            assert float((g.double() - v).norm() / v.norm()) <= most * half_step(dt), (what, parts)
    assert all(torch.equal(a, c) for a, c in zip(got[None], got[2 if M * N * K <= 2 ** 25 else 1]))


def test_parts_of_dz_that_do_not_matter():
    """fp32, and no activation: dz is dy itself or held in fp32"""
    from hot_amd import ops
    from hot_amd._lib import HotkError
    for dt, act in ((torch.float32, 'gelu'), (torch.bfloat16, 'none')):
        x, w, dy = rnd(544, 30, 24, dt=dt).requires_grad_(True), rnd(545, 40, 24, dt=dt).requires_grad_(True), rnd(546, 30, 40, dt=dt)
        one, two = (torch.autograd.grad(ops.linear_act(x, w, act=act, dz_parts=parts), (x, w), dy) for parts in (1, 2))
        assert all(torch.equal(a, c) for a, c in zip(one, two))
    for bad in (0, 3, -1, 1.5, 'one'):
        with pytest.raises(HotkError):
            ops.linear_act(x, w, dz_parts=bad)


# ------------------------------------------------------------------------------------------------
# gradients that nobody asked for
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('R,D', [(3, 40), (1024, 40), (1025, 40), (2100, 7), (1500, 520), (1030, 20000)])
def test_norm_gradient_of_the_rows_alone(R, D, dt):
    """a frozen weight: dx as with the weight's gradient, and no memory or launch for the latter"""
    from hot_amd import _lib, ops
    x, w, dy = rnd(550, R, D, dt=dt).requires_grad_(True), rnd(551, D, dt=dt), rnd(552, R, D, dt=dt)
    want, _ = torch.autograd.grad(ops.rms_norm(x, v := w.clone().requires_grad_(True)), (x, v), dy)
    y = ops.rms_norm(x, w)
    requested = lambda: torch.cuda.memory_stats()['requested_bytes.all.allocated']      # (blocks may be larger than asked for)
    before = requested()
    _lib.timing_begin(None)
    got, = torch.autograd.grad(y, x, dy)
    seen = _lib.timing_end()
    asked = requested() - before
    assert asked == got.numel() * got.element_size()                                    # the result and nothing else
    assert torch.equal(got, want) and set(seen) == {'hotk_rmsnorm_bwd'}


# ------------------------------------------------------------------------------------------------
# gradients past 2^31 elements: operands of -1, 0 and 1, so that every sum is a whole number below 2^24 and exact in any order
# ------------------------------------------------------------------------------------------------
def whole(seed, *size):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-1, 2, size, generator=g, device=DEV, dtype=torch.int8).to(torch.bfloat16)


ROWS, CHUNK = 1100000, 55000


def test_weight_gradient_past_32_bits():
    """dw = dy^T x with x of 2^31 elements, contracted down its columns in splits: bit for bit"""
    from hot_amd import ops
    x, V, dy = whole(560, ROWS, 2048), whole(561, 16, 2048).requires_grad_(True), whole(562, ROWS, 16)
    dV, = torch.autograd.grad(ops.linear_act(x, V), V, dy)
    want = torch.zeros(16, 2048, device=DEV, dtype=torch.float64)
    for i in range(0, ROWS, CHUNK):
        want += dy[i:i + CHUNK].double().t().contiguous() @ x[i:i + CHUNK].double()
    assert torch.equal(dV, want.to(torch.bfloat16))


def test_all_gradients_past_32_bits():
    """dy, slopes and dz of 2^31 elements each"""
    from hot_amd import ops
    x, W, b, dy = whole(563, ROWS, 24), whole(564, 2048, 24), whole(565, 2048), whole(566, ROWS, 2048)
    leaves = [t.requires_grad_(True) for t in (x, W, b)]
    dx, dW, db = torch.autograd.grad(ops.linear_act(*leaves, act='relu'), leaves, dy)
    want_w, want_b = torch.zeros(2048, 24, device=DEV, dtype=torch.float64), torch.zeros(2048, device=DEV, dtype=torch.float64)
    Wd = W.detach().double()
    for i in range(0, ROWS, CHUNK):
        xd = x.detach()[i:i + CHUNK].double()
        dz = dy[i:i + CHUNK].double() * (xd @ Wd.t().contiguous() + b.detach().double() > 0)
        want_w += dz.t().contiguous() @ xd
        want_b += dz.sum(0)
        assert torch.equal(dx[i:i + CHUNK], (dz @ Wd).to(torch.bfloat16)), i
    assert torch.equal(dW, want_w.to(torch.bfloat16)) and torch.equal(db, want_b.to(torch.bfloat16))


# ------------------------------------------------------------------------------------------------
# rows that lie far apart, rows that are too long
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M', [3, 70])
def test_short_rows_far_apart(M, dt):
    """a stride above 8 MiB is no reason to refuse rows of 40 elements"""
    from hot_amd import ops
    far = (1 << 23) // dt.itemsize + 64
    x, w, dy = rnd(570, M, 40, dt=dt), rnd(571, 5, 40, dt=dt), rnd(572, M, 24, dt=dt)
    W = rnd(573, 24, 40, dt=dt)

    def apart(t):
        big = torch.empty(t.size(0), far, dtype=dt, device=DEV)[:, 8:8 + t.size(1)]
        return big.copy_(t)
    def grads(x, W, dy):
        x, W = x.detach().requires_grad_(True), W.detach().requires_grad_(True)
        y = ops.linear_act(x, W, act='gelu')
        return (y.detach(),) + torch.autograd.grad(y, (x, W), dy)
    want = grads(x, W, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads(apart(x), W, apart(dy)), want))
    assert all(torch.equal(a, b) for a, b in zip(grads(x, apart(W), dy), want))
    dx, = torch.autograd.grad(ops.linear_act(v := x.clone().requires_grad_(True), W), v, apart(dy))      # dz is dy, in place or copied
    assert torch.equal(dx, torch.autograd.grad(ops.linear_act(v := x.clone().requires_grad_(True), W), v, dy)[0])


def test_gradients_of_too_long_results_are_refused_at_once():
    from hot_amd import ops
    from hot_amd._lib import HotkError
    N = (1 << 22) + 8
    x, w = rnd(574, 2, 1, dt=torch.bfloat16), torch.ones(N, 1, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(ops.linear_act(x, w), x.expand(2, N))
    for which in (x, w):
        which.requires_grad_(True)
        with pytest.raises(HotkError, match='8 MiB'):
            ops.linear_act(x, w)
        which.requires_grad_(False)
    b = torch.zeros(N, dtype=torch.bfloat16, device=DEV, requires_grad=True)       # the bias's alone needs no product
    db, = torch.autograd.grad(ops.linear_act(x, w, b), b, torch.ones(2, N, dtype=torch.bfloat16, device=DEV))
    assert (db == 2).all()


# ------------------------------------------------------------------------------------------------
# what is kept for the backward pass
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('K', [40, 37])
@pytest.mark.parametrize('M', [6, 200])
def test_only_what_a_gradient_needs_is_kept(M, K):
    """x is kept for the weight's gradient and the weight for x's, so the other one may change or go in between; one that is needed and
    read in place may not"""
    from hot_amd import ops
    dt = torch.bfloat16
    x0, w0, b0, dy = rnd(580, M, K, dt=dt), rnd(581, 24, K, dt=dt), rnd(582, 24, dt=dt), rnd(583, M, 24, dt=dt)
    full = [t.clone().requires_grad_(True) for t in (x0, w0, b0)]
    want = torch.autograd.grad(ops.linear_act(*full, act='gelu'), full, dy)
    for which in range(3):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x0, w0, b0))]
        y = ops.linear_act(*leaves, act='gelu')
        needed = {0: 1, 1: 0}.get(which)
        for i, t in enumerate(leaves):
            if i not in (which, needed):
                t.add_(1)
        got, = torch.autograd.grad(y, leaves[which], dy)
        assert torch.equal(got, want[which]), which
    if K % 8 == 0:
        for which, other in ((0, 1), (1, 0)):
            leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x0, w0, b0))]
            y = ops.linear_act(*leaves, act='gelu')
            leaves[other].add_(1)
            with pytest.raises(RuntimeError, match='modified by an inplace operation'):
                torch.autograd.grad(y, leaves[which], dy)


def test_rows_before_a_frozen_weight_are_not_held():
    from hot_amd import ops
    x, w = torch.zeros(1 << 20, 64, device=DEV, requires_grad=True), rnd(584, 8, 64)
    x1 = x * 1
    before = torch.cuda.memory_allocated()
    y = ops.linear_act(x1, w)
    del x1
    assert before - torch.cuda.memory_allocated() >= (1 << 28) - y.numel() * 4 - (1 << 22)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    want = w.double().sum(0)
    hold('dx', dx[:3], want.expand(3, 64), 10 * E * w.double().abs().sum(0).expand(3, 64))


@pytest.mark.parametrize('reentrant', [False, True])
def test_under_checkpointing(reentrant):
    """the forward pass run again in the backward pass, with its own kept tensors: the same gradients"""
    from torch.utils.checkpoint import checkpoint
    from hot_amd import ops
    M, K, N, dt = 70, 37, 24, torch.bfloat16

    def step(x, w, b, r):
        return ops.linear_act(ops.rms_norm(x, w[0]), w, b, act='gelu', residual=r)
    def gradients(call):
        leaves = [t.detach().clone().requires_grad_(True) for t in kept_leaves(M, K, N, dt)]
        return torch.autograd.grad(call(*leaves), leaves, rnd(590, M, N, dt=dt)) if not reentrant else backward(call, leaves)
    def backward(call, leaves):
        call(*leaves).backward(rnd(590, M, N, dt=dt))
        return [t.grad for t in leaves]
    got, want = gradients(lambda *t: checkpoint(step, *t, use_reentrant=reentrant)), gradients(step)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('parts', [1, 2])
def test_parts_of_dz_in_a_graph(parts):
    """captured forward and backward, replayed with other eager work between: each replay equals the eager result"""
    from hot_amd import ops
    dt = torch.float16
    x, w, b, dy = rnd(591, 300, 136, dt=dt), rnd(592, 264, 136, dt=dt, scale=0.1), rnd(593, 264, dt=dt), rnd(594, 300, 264, dt=dt)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.linear_act(*leaves, act='silu', dz_parts=parts)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for turn in range(3):
        x.copy_(rnd(595 + turn, 300, 136, dt=dt))
        want = [t.clone() for t in step()]
        for t in out:
            t.zero_()
        g.replay()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), turn
