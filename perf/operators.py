"""The feed-forward operators of hot_amd.ops as measured cases: the root-mean-square norm of a residual stream (rms_norm,
and rms_norm_quantized with its result in 8 bits), rows to 8 bits with scales (quantize_rows), and the matrix product with
bias, activation and residual in its epilogue (linear_act, and linear_act_quantized over 8-bit operands).

With `own` false, `run` computes them from elementary torch operations in 32 bits; with `own` true it makes the calls that a
user makes.  `exact` is the definition in 64 bits.  Rows are tokens, nodes or entries of a batch; a mask is the `kind` array
of a padded batch (0 = padding)."""
import math

import torch

own = False

E4M3_MAX = 448.0               # largest finite e4m3 value: what a row's largest element is scaled to
SCALE_MIN = 2.0 ** -126        # smallest scale: a row of zeros has this one
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
EPS = 1e-6
ACTS = ('none', 'relu', 'leakyrelu', 'gelu', 'tanh', 'silu')
LARGEST = 16384 * 1024 * 4096  # M N K of the largest product below


def listed():
    return [
        # one new token's norm in a decoding step, with the block's output added to the stream: launch latency
        dict(name='norm token', op='norm', rows=1, width=4096, type='bf16', residual=True, mask=False, grad=False),
        # the pre-norm of an encoder layer over a padded batch of 128 molecules at hidden width 256, a training step
        dict(name='norm train entries', op='norm', rows=7936, width=256, type='fp32', residual=False, mask=True, grad=True),
        # a training step's norm of a wide residual stream: both outputs have a gradient
        dict(name='norm train wide', op='norm', rows=16384, width=4096, type='bf16', residual=True, mask=False, grad=True),
        # the norm in front of an 8-bit product while a batch of sequences of odd lengths is read in; no row is aligned
        dict(name='norm 8bit odd', op='norm8', rows=4099, width=1001, type='fp16', residual=True, mask=True, grad=False),
        # the same for a full batch at an ordinary width
        dict(name='norm 8bit', op='norm8', rows=8192, width=2048, type='bf16', residual=True, mask=False, grad=False),
        # the hidden activations of a feed-forward block between its two 8-bit products
        dict(name='quantize hidden', op='quantize', rows=8192, width=4096, type='bf16'),
        # the weights of a layer brought to 8 bits once, when a trained model is taken into service
        dict(name='quantize weight', op='quantize', rows=1023, width=512, type='fp32'),
        # one token through the first product of a feed-forward block: the weight is read once
        dict(name='linear token', op='linear', rows=1, width=1024, out=4096, type='bf16', act='gelu', bias=True,
             residual=False, grad=False),
        # the feed-forward block's first product over a padded batch of 128 molecules, a training step in 32 bits
        dict(name='linear train entries', op='linear', rows=7936, width=256, out=256, type='fp32', act='gelu', bias=True,
             residual=False, grad=True),
        # a training step of a wide feed-forward block's first product
        dict(name='linear train wide', op='linear', rows=16384, width=1024, out=4096, type='bf16', act='gelu', bias=True,
             residual=False, grad=True),
        # 16 sequences decoding together through the block's second product, added to the stream
        dict(name='linear 8bit tokens', op='linear8', rows=16, width=4096, out=1024, type='bf16', act='none', bias=True,
             residual=True),
        # a batch of prompts read in through an 8-bit product
        dict(name='linear 8bit', op='linear8', rows=8192, width=4096, out=2048, type='bf16', act='silu', bias=True,
             residual=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """a width of the range: a multiple of 64, of 8, or whatever comes"""
    v, step = _log(rng, lo, hi), rng.choice((64, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    op = rng.choice(('norm', 'norm8', 'quantize', 'linear', 'linear', 'linear8'))
    case = dict(op=op, type=rng.choice(tuple(TYPES)))
    if op in ('norm', 'norm8', 'quantize'):
        case.update(rows=_log(rng, 1, 16384), width=_width(rng, 8, 4096))
        if op != 'quantize':
            case.update(residual=rng.random() < 0.5, mask=rng.random() < 0.5, grad=op == 'norm' and rng.random() < 0.6)
        return case
    K, N = _width(rng, 16, 4096), _width(rng, 16, 4096)
    if op == 'linear8':
        K = -(-K // 16) * 16
    most = LARGEST // (K * N) if case['type'] != 'fp32' or op == 'linear8' else LARGEST // (8 * K * N)
    case.update(rows=_log(rng, 1, max(1, min(16384, most))), width=K, out=N, act=rng.choice(ACTS), bias=rng.random() < 0.7,
                residual=rng.random() < 0.4)
    if op == 'linear':
        case.update(grad=rng.random() < 0.6)
    return case


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = TYPES[case['type']]

    def normal(*size, scale=1.0):
        return (torch.randn(*size, generator=g, device='cuda') * scale).to(dt)

    R, D = case['rows'], case['width']
    s = dict(case=case)
    if case['op'] in ('norm', 'norm8', 'quantize'):
        # a residual stream: rows of different sizes, a few channels far larger than the others
        rows = torch.exp(torch.randn(R, 1, generator=g, device='cuda'))
        outlier = 1 + 20 * (torch.rand(D, generator=g, device='cuda') < 0.002)
        s['x'] = (torch.randn(R, D, generator=g, device='cuda') * rows * outlier).to(dt)
        if case['op'] == 'quantize':
            return s
        s['w'] = (1 + 0.2 * torch.randn(D, generator=g, device='cuda')).to(dt)
        s['r'] = normal(R, D) if case['residual'] else None
        s['kind'] = None
        if case['mask']:
            s['kind'] = torch.randint(1, 3, (R,), generator=g, device='cuda', dtype=torch.uint8)
            s['kind'][torch.rand(R, generator=g, device='cuda') < 0.3] = 0
        if case['grad']:
            s['dy'] = normal(R, D)
            s['dh'] = normal(R, D) if case['residual'] else None
            for k in ('x', 'w', 'r'):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    N = case['out']
    s['b'] = normal(N, scale=0.5) if case['bias'] else None
    s['r'] = normal(R, N) if case['residual'] else None
    if case['op'] == 'linear8':
        def eight(rows, cols, scale):
            v = torch.randn(rows, cols, generator=g, device='cuda') * scale
            step = (v.abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN)
            return (v / step[:, None]).to(torch.float8_e4m3fn), step
        s['xq'], s['xs'] = eight(R, D, 1.0)
        s['wq'], s['ws'] = eight(N, D, D ** -0.5)
        return s
    s['x'], s['w'] = normal(R, D), normal(N, D, scale=D ** -0.5)
    if case['grad']:
        s['dy'] = normal(R, N)
        for k in ('x', 'w', 'b', 'r'):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def run(s):
    op = s['case']['op']
    if own:
        from hot_amd import ops
        if op == 'norm':
            return _own_norm(ops, s)
        if op == 'norm8':
            return tuple(ops.rms_norm_quantized(s['x'], s['w'], s['r'], eps=EPS, kind=s['kind']))
        if op == 'quantize':
            return tuple(ops.quantize_rows(s['x']))
        if op == 'linear':
            return _own_linear(ops, s)
        return ops.linear_act_quantized(s['xq'], s['xs'], s['wq'], s['ws'], s['b'], act=s['case']['act'], residual=s['r'],
                                        out_dtype=TYPES[s['case']['type']])
    with torch.no_grad():
        return {'norm': _plain_norm, 'norm8': _plain_norm8, 'quantize': _plain_quantize, 'linear': _plain_linear,
                'linear8': _plain_linear8}[op](s)


def _own_norm(ops, s):
    out = ops.rms_norm(s['x'], s['w'], s['r'], eps=EPS, kind=s['kind'])
    if not s['case']['grad']:
        return out
    if s['r'] is None:
        return (out,) + torch.autograd.grad(out, (s['x'], s['w']), s['dy'])
    return tuple(out) + torch.autograd.grad(out, (s['x'], s['w'], s['r']), (s['dy'], s['dh']))


def _own_linear(ops, s):
    y = ops.linear_act(s['x'], s['w'], s['b'], act=s['case']['act'], residual=s['r'])
    if not s['case']['grad']:
        return y
    return (y,) + torch.autograd.grad(y, [s[k] for k in ('x', 'w', 'b', 'r') if s[k] is not None], s['dy'])


# ------------------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, rounded once at the end
# ------------------------------------------------------------------------------------------------
def _stream(s):
    """the stream as it is stored (the sum rounded to its type), its 32-bit values, and the rows that are kept"""
    x, r, kind = s['x'], s['r'], s['kind']
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    kept = None if kind is None else (kind != 0)[:, None]
    if kept is not None:
        h = torch.where(kept, h, torch.zeros_like(h))
    return h, h.float(), kept


def _plain_norm(s):
    w = s['w'].float()
    h, hf, kept = _stream(s)
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    unit = hf * rstd
    y = (unit * w).to(h.dtype)
    out = (y,) if s['r'] is None else (y, h)
    if s['case']['grad']:
        dy = s['dy'].float()
        if kept is not None:
            dy = torch.where(kept, dy, torch.zeros_like(dy))
        g = dy * w
        dx = rstd * (g - unit * (g * unit).mean(1, keepdim=True))
        if s['r'] is not None:
            dx = dx + s['dh'].float()
        if kept is not None:
            dx = torch.where(kept, dx, torch.zeros_like(dx))
        dx = dx.to(h.dtype)
        out += (dx, (dy * unit).sum(0).to(h.dtype)) + (() if s['r'] is None else (dx,))
    return out if len(out) > 1 else out[0]


def _to_8bit(v):
    scale = (v.abs().amax(1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (v / scale[:, None]).to(torch.float8_e4m3fn), scale


def _plain_norm8(s):
    h, hf, _ = _stream(s)
    y = hf * torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS) * s['w'].float()
    return _to_8bit(y) + (() if s['r'] is None else (h,))


def _plain_quantize(s):
    return _to_8bit(s['x'].float())


def _act(z, act):
    if act == 'relu':
        return z.clamp_min(0)
    if act == 'leakyrelu':
        return torch.where(z > 0, z, 0.01 * z)
    if act == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == 'tanh':
        return torch.tanh(z)
    if act == 'silu':
        return z * torch.sigmoid(z)
    return z


def _act_grad(z, act):
    if act == 'relu':
        return (z > 0).to(z.dtype)
    if act == 'leakyrelu':
        return torch.where(z > 0, 1.0, 0.01).to(z.dtype)
    if act == 'gelu':
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == 'tanh':
        t = torch.tanh(z)
        return 1 - t * t
    if act == 'silu':
        t = torch.sigmoid(z)
        return t * (1 + z * (1 - t))
    return torch.ones_like(z)


def _plain_linear(s):
    x, w, b, r, act = s['x'], s['w'], s['b'], s['r'], s['case']['act']
    xf, wf = x.float(), w.float()
    z = xf @ wf.t()
    if b is not None:
        z = z + b.float()
    y = _act(z, act)
    y = (y if r is None else y + r.float()).to(x.dtype)
    if not s['case']['grad']:
        return y
    dz = s['dy'].float() * _act_grad(z, act)
    out = (y, (dz @ wf).to(x.dtype), (dz.t() @ xf).to(x.dtype))
    return out + (() if b is None else (dz.sum(0).to(x.dtype),)) + (() if r is None else (s['dy'],))


def _plain_linear8(s):
    z = (s['xq'].float() @ s['wq'].float().t()) * s['xs'][:, None] * s['ws']
    if s['b'] is not None:
        z = z + s['b'].float()
    y = _act(z, s['case']['act'])
    return (y if s['r'] is None else y + s['r'].float()).to(TYPES[s['case']['type']])


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and k != 'kind'}
        return _exact_rows(case, s, d) if 'out' not in case else _exact_linear(case, d)


def _exact_rows(case, s, d):
    def eight(v):      # the values that the 8-bit ones stand for in units of the scale, before their rounding
        scale = torch.clamp(torch.linalg.vector_norm(v, ord=float('inf'), dim=-1) / E4M3_MAX, min=SCALE_MIN)
        return [torch.div(v, scale.unsqueeze(-1)), scale]

    if case['op'] == 'quantize':
        return eight(d['x'])
    keep = torch.ones(case['rows'], 1, dtype=torch.float64, device='cuda')
    if s['kind'] is not None:
        keep = s['kind'].ne(0).double().unsqueeze(-1)
    # the stream is what is stored: the sum in its type
    h = (d['x'] + d['r']).to(TYPES[case['type']]).double() * keep if 'r' in d else d['x'] * keep
    inv = (h.pow(2).sum(-1, keepdim=True) / case['width'] + EPS).pow(-0.5)
    y = torch.einsum('rd,r,d->rd', h, inv.squeeze(-1), d['w'])
    stored = [h] if 'r' in d else []
    if case['op'] == 'norm8':
        return eight(y) + stored
    out = [y] + stored
    if case['grad']:
        gy = d['dy'] * keep
        dw = torch.einsum('rd,rd,r->d', gy, h, inv.squeeze(-1))
        gw = gy * d['w']
        dx = gw * inv - h * inv.pow(3) * (gw * h).sum(-1, keepdim=True) / case['width']
        if 'r' in d:
            dx = dx + d['dh'] * keep
        out += [dx, dw] + ([dx] if 'r' in d else [])
    return out if len(out) > 1 else out[0]


def _exact_linear(case, d):
    if case['op'] == 'linear8':
        z = torch.mm(d['xq'] * d['xs'].unsqueeze(1), (d['wq'] * d['ws'].unsqueeze(1)).T)
    else:
        z = torch.mm(d['x'], d['w'].T)
    if 'b' in d:
        z += d['b']
    act = case['act']
    half = 0.5 * torch.erfc(-z / math.sqrt(2)) if act == 'gelu' else None      # the normal distribution function
    logistic = 1 / (1 + torch.exp(-z)) if act == 'silu' else None
    y = {'none': lambda: z, 'relu': lambda: torch.maximum(z, torch.zeros_like(z)),
         'leakyrelu': lambda: torch.maximum(z, 0.01 * z), 'gelu': lambda: z * half, 'tanh': lambda: z.tanh(),
         'silu': lambda: z * logistic}[act]()
    if 'r' in d:
        y = y + d['r']
    if not case.get('grad'):
        return y
    slope = {'none': lambda: torch.ones_like(z), 'relu': lambda: z.gt(0).double(),
             'leakyrelu': lambda: 0.01 + 0.99 * z.gt(0).double(),
             'gelu': lambda: half + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi),
             'tanh': lambda: z.cosh().pow(-2), 'silu': lambda: logistic + z * logistic * (1 - logistic)}[act]()
    dz = d['dy'] * slope
    out = [y, torch.mm(dz, d['w']), torch.mm(dz.T, d['x'])]
    return out + ([dz.sum(dim=0)] if 'b' in d else []) + ([d['dy']] if 'r' in d else [])


def work(case):
    e = 4 if case['type'] == 'fp32' else 2
    R, D = case['rows'], case['width']
    if case['op'] == 'quantize':
        return {'bytes': R * D * (e + 1) + 4 * R, 'flops': 3 * R * D}
    if case['op'] in ('norm', 'norm8'):
        n = 1 + 2 * case['residual']                         # x; the residual and the stored sum
        total = n * e * R * D + e * D + R * case['mask']
        total += R * D + 4 * R if case['op'] == 'norm8' else e * R * D
        if case['grad']:                                     # dy, dx, the sum's own gradient, and the weight's
            total += (2 + case['residual']) * e * R * D + e * D
        return {'bytes': total, 'flops': R * D * (4 + 8 * case['grad'] + 2 * (case['op'] == 'norm8'))}
    N = case['out']
    inputs = 1 if case['op'] == 'linear8' else e
    total = inputs * (R * D + N * D) + e * R * N * (1 + case['residual']) + e * N * case['bias']
    if case['op'] == 'linear8':
        total += 4 * (R + N)
    flops = 2 * R * N * D
    if case.get('grad'):
        total += e * (R * N + R * D + N * D + N * case['bias'])
        flops *= 3
    return {'bytes': total, 'flops': flops}
