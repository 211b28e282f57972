"""GPU (-m gpu): the feed-forward operators against their definition in 64 bits.

Tolerances are bounds by arithmetic, per element.  u = half a step of the type (eps / 2), E = 2^-24 for every 32-bit
operation: a sum of n terms is off by at most n E times the sum of their magnitudes, the result's one rounding adds u of its
value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn


def half_step(dt):
    return torch.finfo(dt).eps / 2


def floor_of(dt):
    """half a step at the bottom of the type's range"""
    return torch.finfo(dt).tiny * torch.finfo(dt).eps


def rnd(seed, *size, dt=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*size, generator=g) * scale).to(dt).to(DEV)


def hold(what, got, want, tol):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).max()):.3g} x the '
                           f'bound, first at {tuple(int(v) for v in bad.nonzero()[0])}')


# ------------------------------------------------------------------------------------------------
# norm
# ------------------------------------------------------------------------------------------------
CHAIN = 160     # longest chain of additions of a row's sum: 64 in a lane, 6 across lanes, 16 across waves, the mean, and the
                # products' own roundings; tests stay below 8192 elements a row


def norm64(x, w, r, eps, kept, dt):
    h = x.double() if r is None else (x.float() + r.float()).to(dt).double()
    if kept is not None:
        h = torch.where(kept, h, torch.zeros_like(h))
    inv = ((h * h).mean(-1, keepdim=True) + eps).rsqrt()
    y = h * inv * w.double()
    if kept is not None:
        y = torch.where(kept, y, torch.zeros_like(y))
    return h, inv, y


def norm_case(R, D, dt, residual, mask, seed=0):
    x, w = rnd(seed, R, D, dt=dt, scale=2.0), (1 + 0.3 * rnd(seed + 1, D)).to(dt)
    r = rnd(seed + 2, R, D, dt=dt) if residual else None
    kind = None
    if mask:
        kind = torch.randint(0, 3, (R,), generator=torch.Generator().manual_seed(seed + 3)).to(torch.uint8).to(DEV)
    return x, w, r, kind


NORM_SIZES = [(1, 1), (3, 3), (5, 7), (2, 8), (7, 9), (4, 15), (65, 33), (9, 255), (8, 256), (6, 257), (5, 1000), (3, 1001), (17, 2048),
              (3, 2049), (2, 4100), (3, 8191), (1024, 40), (1025, 40), (3000, 7), (2500, 300)]


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('R,D', NORM_SIZES)
@pytest.mark.parametrize('residual,mask', [(False, False), (True, False), (False, True), (True, True)])
def test_norm_forward_and_gradients(R, D, dt, residual, mask):
    from hot_amd import ops
    x, w, r, kind = norm_case(R, D, dt, residual, mask)
    kept = None if kind is None else (kind != 0)[:, None]
    leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
    out = ops.rms_norm(x, w, r, eps=1e-5, kind=kind)
    y, h = out if residual else (out, None)
    h64, inv, y64 = norm64(x.detach(), w.detach(), None if r is None else r.detach(), 1e-5, kept, dt)
    u = half_step(dt)
    hold('y', y.detach(), y64, (u + CHAIN * E) * y64.abs() + floor_of(dt))
    if residual:
        assert torch.equal(h.detach().double(), h64)
    dy, dh = rnd(10, R, D, dt=dt), (rnd(11, R, D, dt=dt) if residual else None)
    got = torch.autograd.grad(out, leaves, (dy, dh) if residual else dy)
    on = torch.ones(R, 1, dtype=torch.float64, device=DEV) if kept is None else kept.double()
    g = dy.double() * on * w.detach().double()
    unit = h64 * inv
    m = (g * unit).mean(-1, keepdim=True)
    dx = inv * (g - unit * m) + (dh.double() * on if residual else 0)
    size = inv * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True)) + (dh.double().abs() * on if residual else 0)
    hold('dx', got[0], dx * on, u * dx.abs() + 3 * CHAIN * E * size + floor_of(dt))
    dw = (dy.double() * on * unit).sum(0)
    hold('dw', got[1], dw, u * dw.abs() + (CHAIN + R) * E * (dy.double() * on * unit).abs().sum(0) + floor_of(dt))
    if residual:
        assert torch.equal(got[2], got[0])


def test_norm_gradient_against_differences():
    """d/dt of <y, a> + <h, b> along a direction, fp32 in and 64-bit differences of the definition"""
    from hot_amd import ops
    R, D = 6, 40
    x, w, r, _ = norm_case(R, D, torch.float32, True, False, seed=20)
    a, b = rnd(30, R, D), rnd(31, R, D)
    for t in (x, w, r):
        t.requires_grad_(True)
    got = torch.autograd.grad(ops.rms_norm(x, w, r), (x, w, r), (a, b))
    dirs = [rnd(40 + i, *t.shape) for i, t in enumerate((x, w, r))]
    along = sum(float((g.double() * d.double()).sum()) for g, d in zip(got, dirs))

    def f(t):
        xx, ww, rr = (v.detach().double() + t * d.double() for v, d in zip((x, w, r), dirs))
        h = xx + rr
        return float((h * ((h * h).mean(-1, keepdim=True) + 1e-6).rsqrt() * ww * a.double()).sum() + (h * b.double()).sum())
    step = 1e-5
    diff = (f(step) - f(-step)) / (2 * step)
    assert abs(along - diff) <= 1e-5 * max(1.0, abs(diff)), (along, diff)


@pytest.mark.parametrize('dt', TYPES)
def test_norm_masked_rows_are_not_read(dt):
    from hot_amd import ops
    R, D = 12, 100
    x, w, r, _ = norm_case(R, D, dt, True, False, seed=50)
    kind = torch.tensor([0, 1, 2, 0] * 3, dtype=torch.uint8, device=DEV)
    gone = kind == 0
    dy, dh = rnd(51, R, D, dt=dt), rnd(52, R, D, dt=dt)
    ref = None
    for fill in (0., float('nan'), float('inf'), torch.finfo(dt).min):
        xs, rs, gs, hs = (t.clone().masked_fill_(gone[:, None], fill) for t in (x, r, dy, dh))
        leaves = [t.requires_grad_(True) for t in (xs, w.clone(), rs)]
        out = ops.rms_norm(leaves[0], leaves[1], leaves[2], kind=kind)
        res = [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (gs, hs)))
        q = ops.rms_norm_quantized(xs.detach(), w, rs.detach(), kind=kind)
        res += [q[0].float(), q[1], q[2]]
        for k in (0, 1, 2, 4, 5, 7):
            assert (res[k][gone] == 0).all(), k
        assert (q[1][gone] == 2.0 ** -126).all()
        if ref is None:
            ref = res
        assert all(torch.equal(a, b) for a, b in zip(ref, res))
    nothing = ops.rms_norm(x, w, kind=torch.zeros(R, dtype=torch.uint8, device=DEV))
    assert (nothing == 0).all()
    one_kind = ops.rms_norm(x, w, kind=kind, keep=4)       # only kind 2
    assert (one_kind[kind != 2] == 0).all() and torch.equal(one_kind[kind == 2], ops.rms_norm(x, w)[kind == 2])


@pytest.mark.parametrize('dt', TYPES)
def test_norm_values_at_the_edges(dt):
    from hot_amd import ops
    D = 37
    w = torch.ones(D, dtype=dt, device=DEV)
    x = rnd(60, 4, D, dt=dt)
    x[1] = 0
    x[2, 5] = float('nan')
    x[3, 5] = float('inf')
    y = ops.rms_norm(x, w)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[0].isfinite().all()
    assert y[3, 5].isnan() and (y[3, :5] == 0).all()           # inf * 0, finite * 0
    q, s = ops.quantize_rows(x)
    assert s[1] == 2.0 ** -126 and (q[1].float() == 0).all() and s[2].isnan() and s[3].isinf() and s[0].isfinite()
    assert (q[3, :5].float() == 0).all() and q[3, 5].float().isnan()


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('R,D', [(1, 1), (3, 5), (4, 16), (33, 129), (5, 1000), (3, 1001), (9, 4096), (2, 8190)])
def test_quantize_rows(R, D, dt):
    """bit for bit: one correctly rounded division for the scale, one per element, one rounding to e4m3"""
    from hot_amd import ops
    x = rnd(70, R, D, dt=dt, scale=3.0)
    x[:, D // 2] *= 50
    q, s = ops.quantize_rows(x)
    xc = x.cpu().float()
    want_s = (xc.abs().amax(1) / 448).clamp_min(2.0 ** -126)
    assert q.dtype == E4M3 and torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().float(), (xc / want_s[:, None]).to(E4M3).float())


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('R,D,residual', [(1, 1, True), (4, 13, False), (33, 129, True), (5, 1000, True), (7, 2050, False), (2, 8191, True)])
def test_norm_quantized(R, D, dt, residual):
    from hot_amd import ops
    x, w, r, _ = norm_case(R, D, dt, residual, False, seed=80)
    out = ops.rms_norm_quantized(x, w, r)
    h64, _, y64 = norm64(x, w, r, 1e-6, None, dt)
    s64 = y64.abs().amax(1) / 448
    hold('scale', out[1], s64, (CHAIN + 2) * E * s64)
    # half a step of e4m3 relative to the value, half its smallest step near zero; y itself is off by CHAIN E
    hold('q', out[0].double() * out[1].double()[:, None], y64, (2.0 ** -4 + 4 * CHAIN * E) * y64.abs() + 2.0 ** -10 * 1.001 * s64[:, None])
    if residual:
        assert torch.equal(out[2].double(), h64)


def test_norm_rows_in_place_at_any_stride():
    from hot_amd import ops
    big = rnd(90, 9, 300, dt=torch.bfloat16)
    w = rnd(91, 101, dt=torch.bfloat16)
    for view in (big[:, 3:104], big[::2, 7:108], big[:, 100:201].unflatten(0, (3, 3)), big[:, :202:2], big[4, 5:106], big[:, 3:104].t().contiguous().t()):
        assert torch.equal(ops.rms_norm(view, w), ops.rms_norm(view.contiguous(), w))
        q, s = ops.quantize_rows(view)
        q2, s2 = ops.quantize_rows(view.contiguous())
        assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2)
    row = rnd(92, 1, 101, dt=torch.bfloat16).expand(4, 101)      # rows at stride zero, a shared leaf
    leaf = row[:1].clone().requires_grad_(True)
    y = ops.rms_norm(leaf.expand(4, 101), w)
    dy = rnd(93, 4, 101, dt=torch.bfloat16)
    g, = torch.autograd.grad(y, leaf, dy)
    parts = [torch.autograd.grad(ops.rms_norm(l, w), l, dy[i:i + 1])[0] for i in range(4) for l in [leaf.detach().clone().requires_grad_(True)]]
    total = sum(p.double() for p in parts)
    hold('shared leaf', g, total, 4 * half_step(torch.bfloat16) * sum(p.double().abs() for p in parts))


@pytest.mark.parametrize('R', [0, 1])
def test_empty_batches(R):
    from hot_amd import ops
    x, w = rnd(95, R, 24).requires_grad_(True), rnd(96, 24).requires_grad_(True)
    W, b = rnd(97, 8, 24).requires_grad_(True), rnd(98, 8).requires_grad_(True)
    y = ops.linear_act(ops.rms_norm(x, w), W, b, act='gelu')
    assert y.shape == (R, 8)
    grads = torch.autograd.grad(y, (x, w, W, b), torch.ones_like(y))
    assert [tuple(g.shape) for g in grads] == [(R, 24), (24,), (8, 24), (8,)]
    if R == 0:
        assert all((g == 0).all() for g in grads)
    q, s = ops.quantize_rows(x.detach())
    assert q.shape == (R, 24) and s.shape == (R,)
    wq, ws = ops.quantize_rows(W.detach())
    assert ops.linear_act_quantized(q, s, wq, ws, out_dtype=torch.float32).shape == (R, 8)


def test_offsets_past_32_bits():
    """more than 2^31 elements: the last rows equal the same rows in a small call"""
    from hot_amd import ops
    R, D, dt = 1100000, 2048, torch.bfloat16
    tail = slice(R - 70, R)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(R, D, generator=g, device=DEV, dtype=dt)
    w = rnd(1, D, dt=dt)
    y, h = ops.rms_norm(x, w, x)
    ys, hs = ops.rms_norm(x[tail], w, x[tail])
    assert torch.equal(y[tail], ys) and torch.equal(h[tail], hs)
    del y, h
    q, s = ops.quantize_rows(x)
    qs, ss = ops.quantize_rows(x[tail])
    assert torch.equal(q[tail].float(), qs.float()) and torch.equal(s[tail], ss)
    del q, s
    W = rnd(2, D, 24, dt=dt, scale=0.2)
    z = ops.linear_act(x[:, :24], W, act='relu', residual=x)                # read at a stride, 2^31 results
    assert torch.equal(z[tail], ops.linear_act(x[tail, :24].contiguous(), W, act='relu', residual=x[tail]))
    del z
    leaf = x[:, 24:48].detach().requires_grad_(True)
    dx, = torch.autograd.grad(ops.linear_act(leaf, W), leaf, x)
    want = x[tail].double() @ W.double()                                    # (a small call may split its sum: not bit for bit)
    hold('dx', dx[tail], want, half_step(dt) * want.abs() + (D + 8) * E * (x[tail].double().abs() @ W.double().abs()))
    V = rnd(3, 16, D, dt=dt, scale=0.02).requires_grad_(True)
    dV, = torch.autograd.grad(ops.linear_act(x, V), V, rnd(4, R, 16, dt=dt))
    ref = (rnd(4, R, 16, dt=dt)[-1000:].double().t() @ x[-1000:].double())
    part, = torch.autograd.grad(ops.linear_act(x[-1000:], V), V, rnd(4, R, 16, dt=dt)[-1000:].contiguous())
    assert dV.isfinite().all() and float((part.double() - ref).norm() / ref.norm()) < half_step(dt)


@pytest.mark.parametrize('dt', TYPES)
def test_one_tensor_in_two_places(dt):
    """the stream as its own residual, the weight as the rows: gradients add up"""
    from hot_amd import ops
    x, w = rnd(400, 30, 64, dt=dt).requires_grad_(True), rnd(401, 64, dt=dt)
    dy, dh = rnd(402, 30, 64, dt=dt), rnd(403, 30, 64, dt=dt)
    both, = torch.autograd.grad(ops.rms_norm(x, w, x), x, (dy, dh))
    a, b = x.detach().requires_grad_(True), x.detach().requires_grad_(True)
    ga, gb = torch.autograd.grad(ops.rms_norm(a, w, b), (a, b), (dy, dh))
    assert torch.equal(both, ga + gb)
    W = rnd(404, 40, 64, dt=dt).requires_grad_(True)
    dz = rnd(405, 40, 40, dt=dt)
    both, = torch.autograd.grad(ops.linear_act(W, W, act='gelu'), W, dz)
    a, b = W.detach().requires_grad_(True), W.detach().requires_grad_(True)
    ga, gb = torch.autograd.grad(ops.linear_act(a, b, act='gelu'), (a, b), dz)
    assert torch.equal(both, ga + gb)
    x.grad = None
    y, h = ops.rms_norm(x, w, x)
    y.backward(dy)                                   # only one of the two outputs has a gradient
    only_y = x.grad.clone()
    y, h = ops.rms_norm(a_ := x.detach().requires_grad_(True), w, a_)
    g2, = torch.autograd.grad((y, h), a_, (dy, torch.zeros_like(h)))
    assert torch.equal(only_y, g2)
    y, h = ops.rms_norm(x, w, x)
    g3, = torch.autograd.grad(h, x, dh)
    assert torch.equal(g3, dh + dh)


def test_calls_from_several_threads():
    """forward and backward from four threads on streams of their own"""
    import threading
    from hot_amd import ops
    p = block_params(136, 264, 90, torch.bfloat16, seed=410)
    xs = [rnd(420 + i, 90, 136, dt=torch.bfloat16) for i in range(4)]
    dy = rnd(430, 90, 136, dt=torch.bfloat16)

    def step(x):
        leaves = [t.detach().requires_grad_(True) for t in [x] + list(p.values())]
        y = block(ops, leaves[0], dict(zip(p, leaves[1:])))
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got[i] = step(xs[i])
            s.synchronize()
        except Exception as e:      # noqa: BLE001 (shown by the assertion below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_wide_rows():
    from hot_amd import ops
    for dt in TYPES:
        for D in (12000, 32768):
            x, w, r, _ = norm_case(3, D, dt, True, False, seed=99)
            for t in (x, w, r):
                t.requires_grad_(True)
            out = ops.rms_norm(x, w, r)
            h64, inv, y64 = norm64(x.detach(), w.detach(), r.detach(), 1e-6, None, dt)
            hold('y', out[0].detach(), y64, (half_step(dt) + CHAIN * E) * y64.abs() + floor_of(dt))
            dy = rnd(100, 3, D, dt=dt)
            dx, dw, _ = torch.autograd.grad(out[0], (x, w, r), dy)
            g, unit = dy.double() * w.detach().double(), h64 * inv
            want = inv * (g - unit * (g * unit).mean(-1, keepdim=True))
            size = inv * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True))
            hold('dx', dx, want, half_step(dt) * want.abs() + 3 * CHAIN * E * size + floor_of(dt))


# ------------------------------------------------------------------------------------------------
# product
# ------------------------------------------------------------------------------------------------
ACTS = ['none', 'relu', 'leakyrelu', 'gelu', 'tanh', 'silu']


def act64(z, act):
    s = torch.sigmoid(z)
    return {'none': lambda: z, 'relu': lambda: z.clamp_min(0), 'leakyrelu': lambda: torch.where(z > 0, z, 0.01 * z),
            'gelu': lambda: z * 0.5 * torch.erfc(-z / math.sqrt(2)), 'tanh': lambda: z.tanh(), 'silu': lambda: z * s}[act]()


def slope64(z, act):
    s = torch.sigmoid(z)
    return {'none': lambda: torch.ones_like(z), 'relu': lambda: (z > 0).double(),
            'leakyrelu': lambda: torch.where(z > 0, 1.0, 0.01).double(),
            'gelu': lambda: 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            'tanh': lambda: 1 - z.tanh() ** 2, 'silu': lambda: s * (1 + z * (1 - s))}[act]()


def linear_case(M, N, K, dt, bias, residual, seed=0):
    return (rnd(seed, M, K, dt=dt), rnd(seed + 1, N, K, dt=dt, scale=K ** -0.5), rnd(seed + 2, N, dt=dt) if bias else None,
            rnd(seed + 3, M, N, dt=dt) if residual else None)


def z_bounds(x, w, b, scales=None):
    """(z, how far 32-bit accumulation may be from it)"""
    xd, wd = x.double(), w.double()
    if scales is not None:
        xd, wd = xd * scales[0].double()[:, None], wd * scales[1].double()[:, None]
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, (x.size(1) + 8) * E * size


def check_forward(y, z, dz, act, r, dt):
    f = act64(z, act)
    y64 = f if r is None else f + r.double()
    # |f'| < 1.13; the functions themselves: 4e-7 of max(1, |z|) (the largest is the erf's 1.5e-7 times z / 2)
    tol = half_step(dt) * y64.abs() + 1.13 * dz + (4e-7 * z.abs().clamp_min(1) if act != 'none' else 0) + 2 * E * (f.abs() + y64.abs())
    hold('y', y, y64, tol + floor_of(dt))


SIZES = [(1, 1, 1), (1, 5, 3), (2, 3, 7), (15, 16, 8), (16, 17, 16), (17, 64, 24), (33, 65, 40), (64, 100, 65), (65, 33, 64), (100, 130, 129),
         (129, 128, 72), (130, 257, 200), (257, 31, 1000), (1, 300, 2048), (5, 64, 4096), (200, 70, 3001)]


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('M,N,K', SIZES)
def test_product_forward(M, N, K, dt):
    from hot_amd import ops
    for i, act in enumerate(ACTS):
        x, w, b, r = linear_case(M, N, K, dt, i % 2 == 0, i % 3 == 0, seed=100 + i)
        z, dz = z_bounds(x, w, b)
        check_forward(ops.linear_act(x, w, b, act=act, residual=r), z, dz, act, r, dt)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('M,N,K', [(700, 512, 72), (4100, 1030, 40), (2048, 3000, 136), (16, 4096, 64), (40, 2050, 320), (3000, 33, 520)])
def test_product_forward_many_tiles(M, N, K, dt):
    from hot_amd import ops
    x, w, b, r = linear_case(M, N, K, dt, True, True, seed=120)
    z, dz = z_bounds(x, w, b)
    check_forward(ops.linear_act(x, w, b, act='silu', residual=r), z, dz, 'silu', r, dt)


def check_gradients(x, w, b, r, act, dy, got, dt):
    M, K = x.shape
    N = w.size(0)
    u = half_step(dt)
    xd, wd, gd = x.double(), w.double(), dy.double()
    z, ez = z_bounds(x, w, b)
    s = slope64(z, act)
    # the slope: kept to 2^-15 for 16-bit types, 1e-6 of max(1, |z|) as computed, |f''| <= 1.2 times z's error; a kink within that
    # error of zero may lie on either side
    es = (0 if act in ('none', 'relu', 'leakyrelu') else (2.0 ** -15 if dt != torch.float32 else 0) + 1e-6 * z.abs().clamp_min(1) + 1.2 * ez)
    if act in ('relu', 'leakyrelu'):
        es = (z.abs() <= ez).double()
    dz = gd * s
    e32 = gd.abs() * es + 2 * E * dz.abs()                   # in 32 bits, as the bias gradient adds it
    e = e32 + u * (dz.abs() + e32) + floor_of(dt)            # as the products read it
    size = dz.abs() + e
    want = dz @ wd
    hold('dx', got['x'], want, u * want.abs() + e @ wd.abs() + (N + 8) * E * (size @ wd.abs()) + floor_of(dt))
    want = dz.t() @ xd
    hold('dw', got['w'], want, u * want.abs() + e.t() @ xd.abs() + (M + 8) * E * (size.t() @ xd.abs()) + floor_of(dt))
    if b is not None:
        want = dz.sum(0)
        hold('db', got['b'], want, u * want.abs() + e32.sum(0) + (M + 8) * E * size.sum(0) + floor_of(dt))
    if r is not None:
        assert torch.equal(got['r'], dy)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (3, 5, 7), (17, 16, 8), (33, 65, 40), (64, 64, 64), (100, 130, 129), (130, 72, 257), (300, 264, 32),
                                   (1000, 40, 24), (4099, 48, 16), (2, 1000, 136)])
def test_product_gradients(M, N, K, dt):
    from hot_amd import ops
    for i, act in enumerate(ACTS):
        x, w, b, r = linear_case(M, N, K, dt, i % 2 == 0, i % 3 == 0, seed=140 + i)
        dy = rnd(150 + i, M, N, dt=dt)
        named = {k: t.requires_grad_(True) for k, t in (('x', x), ('w', w), ('b', b), ('r', r)) if t is not None}
        y = ops.linear_act(x, w, b, act=act, residual=r)
        got = dict(zip(named, torch.autograd.grad(y, list(named.values()), dy)))
        with torch.no_grad():
            z, dz = z_bounds(x, w, b)
            check_forward(y.detach(), z, dz, act, r, dt)
            check_gradients(x, w, b, r, act, dy, got, dt)


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('M,N,K', [(50, 200, 130), (700, 24, 64), (2000, 130, 72), (64, 3000, 40)])
def test_small_gradients_carry_no_rounding_but_their_own(M, N, K, dt):
    """where the products are short dz enters them in two parts: what is left is the result's rounding (0.58 u as a whole at most,
    uniform in half a step), where one more rounding would bring 0.8"""
    from hot_amd import ops
    x, w, b, _ = linear_case(M, N, K, dt, True, False, seed=155)
    dy = rnd(156, M, N, dt=dt)
    z, _ = z_bounds(x, w, b)
    dz = dy.double() * slope64(z, 'gelu')
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(ops.linear_act(x, w, b, act='gelu'), (x, w), dy)
    for what, got, want in (('dx', dx, dz @ w.detach().double()), ('dw', dw, dz.t() @ x.detach().double())):
        assert float((got.double() - want).norm() / want.norm()) <= 0.62 * half_step(dt), what


def test_infinite_gradients_stay_infinite():
    """a gradient beyond the type's range is infinite in dz; what its rounding left is nothing, not a NaN"""
    from hot_amd import ops
    for dt in (torch.bfloat16, torch.float16):
        x, w = torch.ones(70, 8, dtype=dt, device=DEV, requires_grad=True), torch.ones(16, 8, dtype=dt, device=DEV)
        dy = torch.ones(70, 16, dtype=dt, device=DEV)
        dy[3, 5] = float('inf')
        dx, = torch.autograd.grad(ops.linear_act(x, w, act='silu'), x, dy)
        assert (dx[3] == float('inf')).all() and dx[4].isfinite().all()


@pytest.mark.parametrize('only', ['x', 'w', 'b', 'r'])
def test_product_one_gradient_at_a_time(only):
    from hot_amd import ops
    M, N, K, dt = 70, 40, 24, torch.bfloat16
    x, w, b, r = linear_case(M, N, K, dt, True, True, seed=160)
    dy = rnd(161, M, N, dt=dt)
    full = {k: t.clone().requires_grad_(True) for k, t in (('x', x), ('w', w), ('b', b), ('r', r))}
    want = dict(zip(full, torch.autograd.grad(ops.linear_act(full['x'], full['w'], full['b'], act='gelu', residual=full['r']), list(full.values()), dy)))
    one = {k: t.clone().requires_grad_(k == only) for k, t in (('x', x), ('w', w), ('b', b), ('r', r))}
    got, = torch.autograd.grad(ops.linear_act(one['x'], one['w'], one['b'], act='gelu', residual=one['r']), [one[only]], dy)
    assert torch.equal(got, want[only])


def test_product_gradient_against_differences():
    from hot_amd import ops
    M, N, K = 9, 12, 10
    for act in ('gelu', 'tanh', 'silu'):
        x, w, b, r = linear_case(M, N, K, torch.float32, True, True, seed=170)
        a = rnd(171, M, N)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        got = torch.autograd.grad(ops.linear_act(x, w, b, act=act, residual=r), leaves, a)
        dirs = [rnd(172 + i, *t.shape) for i, t in enumerate(leaves)]
        along = sum(float((g.double() * d.double()).sum()) for g, d in zip(got, dirs))

        def f(t):
            xx, ww, bb, rr = (v.detach().double() + t * d.double() for v, d in zip(leaves, dirs))
            return float(((act64(xx @ ww.t() + bb, act) + rr) * a.double()).sum())
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(along - diff) <= 2e-5 * max(1.0, abs(diff)), (act, along, diff)


@pytest.mark.parametrize('dt', TYPES)
def test_product_infinities_and_nan_stay_in_their_rows(dt):
    from hot_amd import ops
    M, N, K = 40, 50, 72
    for act in ACTS:
        x, w, b, _ = linear_case(M, N, K, dt, True, False, seed=180)
        clean = ops.linear_act(x, w, b, act=act)
        x[7, 3] = float('nan')
        w[11, 70] = float('nan')
        y = ops.linear_act(x, w, b, act=act)
        assert y[7].isnan().all() and y[:, 11].isnan().all()
        keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
        keep[7] = False
        keep[:, 11] = False
        assert torch.equal(y[keep], clean[keep])
    x, w, b, _ = linear_case(M, N, K, dt, True, False, seed=181)
    b[3], b[4] = float('inf'), float('-inf')
    y = ops.linear_act(x, w, b, act='relu')
    assert (y[:, 3] == float('inf')).all() and (y[:, 4] == 0).all() and y[:, 5:].isfinite().all()


def test_product_rows_in_place_at_any_stride():
    from hot_amd import ops
    for dt in TYPES:
        big = rnd(190, 24, 400, dt=dt)
        w = rnd(191, 33, 72, dt=dt, scale=0.1)
        wide = rnd(192, 33, 200, dt=dt, scale=0.1)
        r = rnd(193, 24, 90, dt=dt)
        for view in (big[:, 8:80], big[:, 3:75], big[::2, 16:88], big[:, :144:2], big[:, 16:88].unflatten(0, (4, 6))):
            n = view.numel() // 72
            res = r[:n, 5:38]
            for weight in (w, wide[:, 8:80], wide[:, 1:73], wide[:, 100:172], w.t().contiguous().t()):
                y = ops.linear_act(view, weight, residual=res.reshape(*view.shape[:-1], 33) if view.dim() == 3 else res, act='relu')
                z = ops.linear_act(view.contiguous(), weight.contiguous(), residual=res.contiguous().view(*view.shape[:-1], 33), act='relu')
                assert torch.equal(y, z)
    x = rnd(194, 4, 1, 72).expand(4, 5, 72)
    assert torch.equal(ops.linear_act(x, rnd(195, 8, 72)), ops.linear_act(x.contiguous(), rnd(195, 8, 72)))


def eight_bit_sums(xq, xs, wq, ws, out):
    """16-bit results of 8-bit operands: products are added by eights, each aligned to the largest of its eight and cut off below
    2^-13 of it, so an eight is off by at most 8 * 2^-13 of its largest product, and the eights' largest add up to no more
    than the sum of all magnitudes"""
    if out == torch.float32:
        return 0
    return 2.0 ** -10 * (xq.double().abs() * xs.double()[:, None]) @ (wq.double().abs() * ws.double()[:, None]).t()


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('M', [3, 40, 100, 700])
@pytest.mark.parametrize('K', [1, 5, 101, 133])
def test_product_reads_nothing_behind_a_row(M, K, dt):
    """rows that end inside a 16-byte piece, with NaN behind and before them: at stride and start that look aligned, and at odd ones"""
    from hot_amd import ops
    N = 70
    x, w, b, _ = linear_case(M, N, K, dt, True, False, seed=230)
    want = ops.linear_act(x, w, b, act='relu')
    z, dz = z_bounds(x, w, b)
    check_forward(want, z, dz, 'relu', None, dt)
    dy = rnd(231, M, N + 1, dt=dt)
    ref = torch.autograd.grad(ops.linear_act(x.requires_grad_(True), w.requires_grad_(True), b, act='relu'), (x, w), dy[:, :N].contiguous())
    for start, width in ((16, 16 + 160), (3, 16 + 161)):
        bx, bw = (torch.full((n, width), float('nan'), dtype=dt, device=DEV) for n in (M, N))
        xv, wv = bx[:, start:start + K], bw[:, start:start + K]
        xv.copy_(x.detach()), wv.copy_(w.detach())
        assert torch.equal(ops.linear_act(xv, wv, b, act='relu'), want)
        xv, wv = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
        got = torch.autograd.grad(ops.linear_act(xv, wv, b, act='relu'), (xv, wv), dy[:, :N])
        assert all(torch.equal(g, r) for g, r in zip(got, ref))
    if dt == torch.bfloat16 and K > 1:
        q, s = ops.quantize_rows(x.detach())
        wq, ws = ops.quantize_rows(w.detach())
        want = ops.linear_act_quantized(q, s, wq, ws, b)
        bq = torch.full((M, 208), float('nan'), device=DEV).to(E4M3)
        bq[:, 16:16 + K] = q
        assert torch.equal(ops.linear_act_quantized(bq[:, 16:16 + K], s, wq, ws, b), want)


@pytest.mark.parametrize('out', TYPES)
@pytest.mark.parametrize('M,N,K', [(1, 1, 1), (1, 33, 16), (5, 64, 48), (16, 100, 4096), (17, 65, 130), (33, 16, 272), (130, 257, 1000), (700, 520, 144),
                                   (3000, 1100, 80), (2, 2050, 512)])
def test_product_of_8bit_operands(M, N, K, out):
    from hot_amd import ops
    for i, act in enumerate(('none', 'gelu', 'silu')):
        xq, xs = ops.quantize_rows(rnd(200 + i, M, K))
        wq, ws = ops.quantize_rows(rnd(210 + i, N, K, scale=K ** -0.5))
        b = rnd(220, N, dt=out) if i != 1 else None
        r = rnd(221, M, N, dt=out) if i != 2 else None
        z, dz = z_bounds(xq, wq, b, (xs, ws))
        y = ops.linear_act_quantized(xq, xs, wq, ws, b, act=act, residual=r, out_dtype=out)
        check_forward(y, z, dz + 2 * E * z.abs() + eight_bit_sums(xq, xs, wq, ws, out), act, r, out)
        if M * N >= 1000:       # and as a whole: the rounding of the result is most of it (uniform in half a step: 0.58 u at most)
            y64 = act64(z, act) + (0 if r is None else r.double())
            assert float((y.double() - y64).norm() / y64.norm()) <= (0.65 * half_step(out) if out != torch.float32 else 1e-6)


# ------------------------------------------------------------------------------------------------
# together, on streams, in graphs
# ------------------------------------------------------------------------------------------------
def block(ops, x, p):
    y, h = ops.rms_norm(x, p['g'], p['r'])
    u = ops.linear_act(y, p['w1'], p['b1'], act='gelu')
    return ops.linear_act(u, p['w2'], p['b2'], residual=h)


def block_params(D, F, R, dt, seed=300):
    return dict(g=(1 + 0.2 * rnd(seed, D)).to(dt), r=rnd(seed + 1, R, D, dt=dt), w1=rnd(seed + 2, F, D, dt=dt, scale=D ** -0.5),
                b1=rnd(seed + 3, F, dt=dt, scale=0.1), w2=rnd(seed + 4, D, F, dt=dt, scale=F ** -0.5), b2=rnd(seed + 5, D, dt=dt, scale=0.1))


@pytest.mark.parametrize('R,D,F', [(1, 24, 72), (37, 64, 130), (300, 256, 512)])
def test_a_block_of_them_with_gradients(R, D, F):
    """fp32: against the same block in 64 bits under autograd, relative to each tensor's size"""
    from hot_amd import ops
    x, p = rnd(310, R, D), block_params(D, F, R, torch.float32)
    leaves = [x] + list(p.values())
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    for t in leaves:
        t.requires_grad_(True)
    y = block(ops, x, p)
    dy = rnd(311, R, D)
    got = torch.autograd.grad(y, leaves, dy)
    xd, g, r, w1, b1, w2, b2 = d
    h = xd + r
    n = h * ((h * h).mean(-1, keepdim=True) + 1e-6).rsqrt() * g
    want_y = torch.nn.functional.gelu(n @ w1.t() + b1) @ w2.t() + b2 + h
    want = torch.autograd.grad(want_y, d, dy.double())
    for name, a, b in zip(['y', 'x'] + list(p), (y.detach(),) + got, (want_y.detach(),) + want):
        # a chain of two sums of D and F terms either way: (D + F + R) E of the largest magnitude, with room for cancellation
        assert float((a.double() - b).abs().max()) <= 4 * (D + F + R + 64) * E * float(b.abs().max()), name


def test_an_8bit_block():
    """serving: norm to 8 bits, product, hidden rows to 8 bits, product added to the stream; the 8-bit values enter the reference
    as they are, so only 32-bit sums and the last rounding differ"""
    from hot_amd import ops
    R, D, F, dt = 19, 96, 208, torch.bfloat16
    x, p = rnd(320, R, D, dt=dt), block_params(D, F, R, dt, seed=321)
    w1, s1 = ops.quantize_rows(p['w1'])
    w2, s2 = ops.quantize_rows(p['w2'])
    q, s, h = ops.rms_norm_quantized(x, p['g'], p['r'])
    u = ops.linear_act_quantized(q, s, w1, s1, p['b1'], act='silu', out_dtype=dt)
    uq, us = ops.quantize_rows(u)
    y = ops.linear_act_quantized(uq, us, w2, s2, p['b2'], residual=h, out_dtype=dt)
    z, dz = z_bounds(q, w1, p['b1'], (s, s1))
    check_forward(u, z, dz + 2 * E * z.abs() + eight_bit_sums(q, s, w1, s1, dt), 'silu', None, dt)
    z, dz = z_bounds(uq, w2, p['b2'], (us, s2))
    check_forward(y, z, dz + 2 * E * z.abs() + eight_bit_sums(uq, us, w2, s2, dt), 'none', h, dt)


def test_on_another_stream():
    from hot_amd import ops
    x, p = rnd(330, 500, 264, dt=torch.bfloat16), block_params(264, 512, 500, torch.bfloat16, seed=331)
    want = block(ops, x, p)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [block(ops, x, p) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_forward_and_backward_in_graphs():
    """two graphs captured from the same calls, replayed in turn with other eager work between: each replay equals the eager run"""
    from hot_amd import ops
    R, D, F, dt = 260, 136, 520, torch.bfloat16
    x, p = rnd(340, R, D, dt=dt), block_params(D, F, R, dt, seed=341)
    dy = rnd(350, R, D, dt=dt)

    def step():
        leaves = [x.detach().requires_grad_(True)] + [t.detach().requires_grad_(True) for t in p.values()]
        y = block(ops, leaves[0], dict(zip(p, leaves[1:])))
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for turn in range(3):
        x.copy_(rnd(360 + turn, R, D, dt=dt))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
            step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_reruns_are_bitwise_equal():
    from hot_amd import ops
    x, p = rnd(370, 2000, 520, dt=torch.float16), block_params(520, 1032, 2000, torch.float16, seed=371)
    dy = rnd(380, 2000, 520, dt=torch.float16)
    runs = []
    for _ in range(2):
        leaves = [t.detach().clone().requires_grad_(True) for t in [x] + list(p.values())]
        y = block(ops, leaves[0], dict(zip(p, leaves[1:])))
        runs.append([y.detach()] + list(torch.autograd.grad(y, leaves, dy)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_refusals():
    from hot_amd import ops
    from hot_amd._lib import HotkError
    x, w, W = rnd(390, 4, 16), rnd(391, 16), rnd(392, 8, 16)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(W)
    kind = torch.ones(4, dtype=torch.uint8, device=DEV)
    bad = [lambda: ops.rms_norm(x, w[:8]), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(x, w, x[:2]),
           lambda: ops.rms_norm(x, w, x.half()), lambda: ops.rms_norm(x.double(), w.double()), lambda: ops.rms_norm(x, w, eps=-1.),
           lambda: ops.rms_norm(x, w, eps=float('nan')), lambda: ops.rms_norm(x, w, kind=kind[:3]), lambda: ops.rms_norm(x, w, kind=kind.int()),
           lambda: ops.rms_norm(x, w, kind=kind, keep=-1), lambda: ops.rms_norm(x[:, :0], w[:0]),
           lambda: ops.rms_norm(torch.zeros(1, 40000, device=DEV), torch.zeros(40000, device=DEV)),
           lambda: ops.quantize_rows(torch.zeros(1, 40000, device=DEV)), lambda: ops.quantize_rows(x.long()),
           lambda: ops.linear_act(x, W[:, :8]), lambda: ops.linear_act(x, W.half()), lambda: ops.linear_act(x, W, w[:7]), lambda: ops.linear_act(x, W, act='elu'),
           lambda: ops.linear_act(x, W, residual=x), lambda: ops.linear_act(x, W[:0]), lambda: ops.linear_act(x, W.cpu()), lambda: ops.linear_act(x, W[0]),
           lambda: ops.linear_act_quantized(x, s, wq, ws), lambda: ops.linear_act_quantized(q, s[:2], wq, ws),
           lambda: ops.linear_act_quantized(q, s, wq, ws.half()), lambda: ops.linear_act_quantized(q, s, W, ws),
           lambda: ops.linear_act_quantized(q, s, wq, ws, out_dtype=torch.float64),
           lambda: ops.linear_act_quantized(q, s, wq, ws, rnd(393, 8)),                                 # an fp32 bias, a bf16 result
           lambda: ops.rms_norm_quantized(x.clone().requires_grad_(True), w), lambda: ops.quantize_rows(x.clone().requires_grad_(True)),
           lambda: ops.linear_act_quantized(q, s, wq, ws, rnd(393, 8).requires_grad_(True), out_dtype=torch.float32)]
    for i, f in enumerate(bad):
        with pytest.raises(HotkError):
            f()
            raise AssertionError(f'call {i} was taken')
    with torch.no_grad():
        ops.quantize_rows(x.clone().requires_grad_(True))


@pytest.mark.parametrize('R,D', [(1, 5), (5, 24), (1024, 40), (1025, 40), (6, 2049)])
def test_norm_gradients_of_some_inputs(R, D):
    """x, the weight or the residual alone: each gradient is the one that all together get"""
    from hot_amd import ops
    leaves = [rnd(401, R, D), rnd(402, D), rnd(403, R, D)]
    dy, dh = rnd(404, R, D), rnd(405, R, D)
    def grads(which):
        x, w, r = [l.clone().requires_grad_(i in which) for i, l in enumerate(leaves)]
        return dict(zip(which, torch.autograd.grad(ops.rms_norm(x, w, r), [(x, w, r)[i] for i in which], (dy, dh))))
    both = grads((0, 1, 2))
    for which in ((0,), (1,), (2,), (0, 1), (1, 2)):
        for i, g in grads(which).items():
            assert torch.equal(g, both[i])


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('R,D', [(2, 12001), (90, 32767), (130, 20000)])
def test_wide_rows_with_all_gradients(R, D, dt):
    """the widest rows (dh read late), weight gradients of few rows as one launch and as partial sums"""
    from hot_amd import ops
    x, w, r, _ = norm_case(R, D, dt, True, False, seed=410)
    for t in (x, w, r):
        t.requires_grad_(True)
    dy, dh = rnd(414, R, D, dt=dt), rnd(415, R, D, dt=dt)
    dx, dw, dr = torch.autograd.grad(ops.rms_norm(x, w, r), (x, w, r), (dy, dh))
    h64, inv, _ = norm64(x.detach(), w.detach(), r.detach(), 1e-6, None, dt)
    g, unit = dy.double() * w.detach().double(), h64 * inv
    want = inv * (g - unit * (g * unit).mean(-1, keepdim=True)) + dh.double()
    size = inv * (g.abs() + unit.abs() * (g * unit).abs().mean(-1, keepdim=True)) + dh.double().abs()
    hold('dx', dx, want, half_step(dt) * want.abs() + 3 * CHAIN * E * size + floor_of(dt))
    assert torch.equal(dx, dr)
    want = (dy.double() * unit).sum(0)
    hold('dw', dw, want, half_step(dt) * want.abs() + (CHAIN + R) * E * (dy.double() * unit).abs().sum(0) + floor_of(dt))


def test_views_that_negate():
    """a lazily negated view's memory holds other values: inputs are refused, a gradient is resolved"""
    from hot_amd import ops
    from hot_amd._lib import HotkError
    z = torch.complex(rnd(420, 6, 16), rnd(421, 6, 16))
    neg = z.conj().imag
    assert neg.is_neg()
    w = rnd(422, 16)
    for call in (lambda: ops.rms_norm(neg, w), lambda: ops.rms_norm(z.imag, w, neg), lambda: ops.rms_norm(z.imag, neg[0]), lambda: ops.quantize_rows(neg),
                 lambda: ops.linear_act(neg, neg.resolve_neg()), lambda: ops.linear_act(neg.resolve_neg(), neg)):
        with pytest.raises(HotkError, match='resolve_neg'):
            call()
    x = rnd(423, 6, 16).requires_grad_(True)
    for f in (lambda: ops.rms_norm(x, w), lambda: ops.linear_act(x, neg.resolve_neg(), act='gelu')):
        y = f()
        dy = neg if y.shape == neg.shape else neg[:, :6]
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(f(), x, dy.resolve_neg())[0])


@pytest.mark.parametrize('M,K,N', [(1, 742, 36), (70, 37, 24), (65, 64, 40)])
def test_kept_tensors_that_left_the_device(M, K, N):
    """what the forward pass keeps comes back from the host with strides of its own"""
    from hot_amd import ops
    leaves = [rnd(430, M, K + 9)[:, 3:K + 3], rnd(431, K, N).t(), rnd(432, N), rnd(433, M, N)]
    dy = rnd(434, M, N)
    def grads():
        x, w, b, r = [l.detach().requires_grad_(True) for l in leaves]
        y = ops.linear_act(x, w, b, act='silu', residual=r)
        z = ops.rms_norm(x, w[0])
        return torch.autograd.grad((y, z), (x, w, b, r), (dy, dy[:, :1].expand(M, K)))
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    want = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('M', [3, 200])
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
def test_scales_far_apart(M, dt):
    """one operand near the top of the range, the other small: the result is what the product holds, either way round"""
    from hot_amd import ops
    K, N = 256, 48
    x, w = rnd(440, M, K), rnd(441, N, K)
    for up, down in ((2.0 ** 120, 2.0 ** -110), (2.0 ** -110, 2.0 ** 120)):
        (xq, sx), (wq, sw) = ops.quantize_rows(x * up), ops.quantize_rows(w * down)
        got = ops.linear_act_quantized(xq, sx, wq, sw, out_dtype=dt)
        scale = sx.double()[:, None] * sw.double()
        want, size = (xq.double() @ wq.double().t()) * scale, (xq.double().abs() @ wq.double().abs().t()) * scale
        # 16-bit results: the eights' own 2^-10 of the sums (fp32: K additions in 32 bits), two products, one rounding
        hold('y', got, want, half_step(dt) * want.abs() + ((K + 4) * E if dt == torch.float32 else 2.0 ** -10) * size)
    sx[0], sw[1] = float('nan'), float('nan')
    got = ops.linear_act_quantized(xq, sx, wq, sw, out_dtype=dt)
    assert got[0].isnan().all() and got[:, 1].isnan().all() and got[1:, 2:].isfinite().all()


@pytest.mark.parametrize('M', [1, 16, 20, 64])
@pytest.mark.parametrize('K', [1, 15, 17, 131, 1029])
def test_few_rows_off_a_words_start(M, K):
    """rows that start at each byte of a word (8 bits) or at its middle (16 bits), last ones at their tensor's end, NaN around them"""
    from hot_amd import ops
    N = 21
    for start in range(4):
        for pad in (0, 1, 2, 5):                                     # the rows' stride goes through all bytes too
            def rows8(seed, n):
                flat = torch.full((start + n * (K + pad),), float('nan'), device=DEV).to(E4M3)
                view = flat[start:].view(n, K + pad)[:, :K]
                view.copy_(rnd(seed, n, K).to(E4M3))
                return view
            xq, wq, sx, sw = rows8(450, M), rows8(451, N), rnd(452, M).abs() + 0.1, rnd(453, N).abs() + 0.1
            got = ops.linear_act_quantized(xq, sx, wq, sw, out_dtype=torch.float32)
            scale = sx.double()[:, None] * sw.double()
            want, size = (xq.double() @ wq.double().t()) * scale, (xq.double().abs() @ wq.double().abs().t()) * scale
            hold('8 bits', got, want, half_step(torch.float32) * want.abs() + (K + 4) * E * size)
            for dt in (torch.bfloat16, torch.float16):
                def rows16(seed, n):
                    flat = torch.full((start + n * (K + pad),), float('nan'), device=DEV, dtype=dt)
                    view = flat[start:].view(n, K + pad)[:, :K]
                    view.copy_(rnd(seed, n, K).to(dt))
                    return view
                x, w = rows16(454, M), rows16(455, N)
                want = x.double() @ w.double().t()
                hold('16 bits', ops.linear_act(x, w), want, half_step(dt) * want.abs() + (K + 2) * E * (x.double().abs() @ w.double().abs().t()) + floor_of(dt))
