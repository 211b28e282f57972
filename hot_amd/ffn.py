"""The feed-forward operators: root-mean-square norm of a residual stream (with its result in 8 bits where a product of 8-bit
operands follows), rows to 8 bits with scales, and the matrix product with bias, activation and residual in its epilogue.
All are reached through `hot_amd.ops`; kernels in csrc/rmsnorm.hip and csrc/linact.hip.

Tensors are fp32, bf16 or fp16 on one HIP device, [..., width], read in place when their rows lie at one stride; results are
new, contiguous tensors.  Sums, statistics and epilogues are in 32 bits and every result is rounded once.  Launches go to the
current stream of the tensors' device; workspaces come from torch's allocator per call, so calls can be captured into a
graph and captured graphs share nothing.  Gradients are of first order."""
import ctypes
from ctypes import byref, c_float, c_size_t

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import ACTS, HotkError, KEEP_VALID, LinearArgs, TYPE_BF16, TYPE_E4M3, TYPE_F16, TYPE_F32, call, check, lib, p, \
    require_device

_TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}
E4M3 = torch.float8_e4m3fn


def _type(t, what, eight=False):
    if eight and t.dtype == E4M3:
        return TYPE_E4M3
    if t.dtype not in _TYPES:
        raise HotkError(f'{what}: fp32, bf16 or fp16 expected, got {t.dtype}')
    return _TYPES[t.dtype]


def _same(ref, t, what, shape, dtype=None):
    """an operand that goes with `ref`: on its device, of its type (or `dtype`) and of this shape"""
    if not isinstance(t, torch.Tensor):
        raise HotkError(f'{what}: a tensor is expected, got {type(t).__name__}')
    if t.device != ref.device:
        raise HotkError(f'{what} is on {t.device}, the input on {ref.device}')
    if t.dtype != (dtype or ref.dtype):
        raise HotkError(f'{what}: {dtype or ref.dtype} expected, got {t.dtype}')
    if tuple(t.shape) != tuple(shape):
        raise HotkError(f'{what}: shape {tuple(shape)} expected, got {tuple(t.shape)}')


def _input(x, what, eight=False):
    if not isinstance(x, torch.Tensor):
        raise HotkError(f'{what}: a tensor is expected, got {type(x).__name__}')
    require_device(x, what)
    _type(x, what, eight)
    if x.dim() < 1 or x.size(-1) == 0:
        raise HotkError(f'{what}: [..., width] with width >= 1 expected, got shape {tuple(x.shape)}')


def _rows(t):
    """[..., C] as rows in place: (tensor, elements from row to row, rows); a copy where the rows lie at no single stride"""
    C = t.size(-1)
    n = t.numel() // C
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if n == 0:
        return t, C, 0
    if t.stride(-1) == 1 or C == 1:
        ld = None
        span = 1                     # rows that the dimensions to the right of k hold
        for k in range(t.dim() - 2, -1, -1):
            if t.size(k) != 1:
                if ld is None:
                    ld = t.stride(k) if span == 1 else None
                if ld is None or t.stride(k) != ld * span:
                    break
            span *= t.size(k)
        else:
            ld = C if ld is None else ld
            if ld >= C:
                return t, ld, n
    return t.contiguous(), C, n


def _kind(kind, x, n):
    if kind is None:
        return None
    if not isinstance(kind, torch.Tensor) or kind.dtype != torch.uint8 or kind.numel() != n or kind.device != x.device:
        raise HotkError(f'kind: uint8, one per row ({n}), on {x.device} expected')
    return kind.contiguous()


def _norm_args(x, weight, residual, kind, keep, eps):
    _input(x, 'x')
    D = x.size(-1)
    _same(x, weight, 'weight', (D,))
    if residual is not None:
        _same(x, residual, 'residual', x.shape)
    if lib().hotk_rmsnorm_supported(D, _TYPES[x.dtype]) != 1:
        raise HotkError(f'rows of up to 32768 elements are normalised, got {D}')
    if not 0 <= int(keep) <= 0xffffffff:
        raise HotkError(f'keep: a bit set over kinds expected, got {keep}')
    if not float(eps) >= 0.:
        raise HotkError(f'eps: a number >= 0 expected, got {eps}')
    return _kind(kind, x, x.numel() // D)


class _RMSNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, residual, kind, keep, eps, grad):
        ctx.set_materialize_grads(False)
        with torch.cuda.device(x.device):
            xs, ld, n = _rows(x)
            D, ty = x.size(-1), _TYPES[x.dtype]
            w = weight.contiguous()
            rs, ld_r = (None, 0) if residual is None else _rows(residual)[:2]
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
            rstd = torch.empty(n, dtype=torch.float32, device=x.device) if grad else None
            if n:
                call('hotk_rmsnorm_fwd', (2 + 2 * (h is not None)) * n * D * x.element_size(), p(xs), ld, p(rs), ld_r, p(w),
                     p(kind), keep, c_float(eps), p(y), p(h), p(rstd), n, D, ty)
        if rstd is not None:
            ctx.save_for_backward(x if h is None else h, rstd, w, kind)
            ctx.cfg = (n, D, ty, keep, x.shape)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, rstd, w, kind = ctx.saved_tensors
        n, D, ty, keep, shape = ctx.cfg
        if dy is None and dh is None:
            return (None,) * 7
        with torch.cuda.device(h.device):
            if dy is None:
                dy = torch.zeros(shape, dtype=h.dtype, device=h.device)
            dx = torch.empty(shape, dtype=h.dtype, device=h.device)
            dw = torch.empty(D, dtype=h.dtype, device=h.device)
            hs, ld_h, _ = _rows(h)
            gs, ld_g, _ = _rows(dy)
            ss, ld_s = (None, 0) if dh is None else _rows(dh)[:2]
            m = ctypes.c_int64()
            check(lib().hotk_rmsnorm_partials(n, D, ty, byref(m)), 'hotk_rmsnorm_partials')
            part = torch.empty(m.value, D, dtype=torch.float32, device=h.device)
            call('hotk_rmsnorm_bwd', (3 + (dh is not None)) * n * D * h.element_size(), p(gs), ld_g, p(ss), ld_s, p(hs), ld_h,
                 p(rstd), p(w), p(kind), keep, p(dx), p(part), n, D, ty)
            if ctx.needs_input_grad[1]:
                call('hotk_sum_partials', 4 * m.value * D, p(part), m.value, D, p(dw), ty)
        return dx, dw if ctx.needs_input_grad[1] else None, dx if ctx.needs_input_grad[2] else None, None, None, None, None


def rms_norm(x, weight, residual=None, eps=1e-6, kind=None, keep=KEEP_VALID):
    """y = h * (mean(h^2) + eps)^-1/2 * weight over the last dimension, h = x; with a residual h = x + residual, rounded to the
    type as the stream is stored, and the result is (y, h).

    x, residual [..., D], weight [D], one type (fp32, bf16, fp16), D <= 32768.  kind (uint8, one per row: a plan's `kind` or
    `nkind`) and keep: rows that keep leaves out are not read, and are zero in y, h and the gradients.  Differentiable in x,
    weight and residual."""
    kind = _norm_args(x, weight, residual, kind, keep, eps)
    return _RMSNorm.apply(x, weight, residual, kind, int(keep), float(eps), _wants_grad(x, weight, residual))


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_grad(what, *tensors):
    if _wants_grad(*tensors):
        raise HotkError(f'{what} has no gradient: call it under torch.no_grad() or on detached tensors')


def rms_norm_quantized(x, weight, residual=None, eps=1e-6, kind=None, keep=KEEP_VALID):
    """rms_norm with y in 8 bits for a product of 8-bit operands (linear_act_quantized): (q, scale), with a residual (q, scale,
    h).  scale[row] = max(max|y| / 448, 2^-126) in fp32, q = e4m3(y / scale), torch.float8_e4m3fn, from y in 32 bits.  A row
    that holds an infinity or NaN comes out with a scale that is one.  No gradient."""
    kind = _norm_args(x, weight, residual, kind, keep, eps)
    _refuse_grad('rms_norm_quantized', x, weight, residual)
    with torch.cuda.device(x.device):
        xs, ld, n = _rows(x)
        D = x.size(-1)
        w = weight.contiguous()
        rs, ld_r = (None, 0) if residual is None else _rows(residual)[:2]
        q = torch.empty(x.shape, dtype=E4M3, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if n:
            call('hotk_rmsnorm_quant', n * D * (1 + (1 + 2 * (h is not None)) * x.element_size()), p(xs), ld, p(rs), ld_r, p(w),
                 p(kind), int(keep), c_float(eps), p(q), p(scale), p(h), n, D, _TYPES[x.dtype])
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows(x):
    """(q, scale): rows of x [..., D] (fp32, bf16, fp16; D <= 32768) to torch.float8_e4m3fn with one fp32 scale each, scale =
    max(max|x| / 448, 2^-126), q = e4m3(x / scale): the operands of linear_act_quantized, weights ([N, K], a scale per output
    column) as well as activations.  A row that holds an infinity or NaN comes out with a scale that is one.  No gradient."""
    _input(x, 'x')
    _refuse_grad('quantize_rows', x)
    D = x.size(-1)
    if lib().hotk_rmsnorm_supported(D, _TYPES[x.dtype]) != 1:
        raise HotkError(f'rows of up to 32768 elements are quantized, got {D}')
    with torch.cuda.device(x.device):
        xs, ld, n = _rows(x)
        q = torch.empty(x.shape, dtype=E4M3, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        if n:
            call('hotk_quantize_rows', n * D * (1 + x.element_size()), p(xs), ld, p(q), p(scale), n, D, _TYPES[x.dtype])
    return q, scale


# ------------------------------------------------------------------------------------------------
# matrix product with bias, activation and residual
# ------------------------------------------------------------------------------------------------
def _turn(t, ld, R, C, ty, save=None, act=0, out=None, ld_out=0, out_t=None, ld_t=0, partial=None):
    n = (out is not None) + (out_t is not None)
    call('hotk_linear_turn', R * C * t.element_size() * (1 + n), p(t), ld, p(save), act, p(out), ld_out, p(out_t), ld_t, p(partial),
         R, C, ty)


def _up(n, size):
    """n elements of `size` bytes in whole 16-byte pieces"""
    m = 16 // size
    return -(-n // m) * m


def _aligned(t, ld, R, C, ty):
    """the rows as the product reads them (whole, aligned 16-byte pieces): in place, or a copy padded with zeros"""
    size = t.element_size()
    if R == 0 or ((C * size) % 16 == 0 and (ld * size) % 16 == 0 and t.data_ptr() % 16 == 0):
        return t, ld
    ld_o = _up(C, size)
    o = torch.empty(R, ld_o, dtype=t.dtype, device=t.device)
    _turn(t, ld, R, C, ty, out=o, ld_out=ld_o)
    return o, ld_o


def _product(x, ld_x, w, ld_w, M, N, K, ty, out_dtype, bias=None, res=None, ld_res=0, act=0, save=None, x_scale=None,
             w_scale=None):
    """[M, N] = epilogue(x w^T) through hotk_linear_act; K counts whole 16-byte pieces"""
    y = torch.empty(M, N, dtype=out_dtype, device=x.device)
    if M == 0:
        return y
    need = c_size_t(0)
    check(lib().hotk_linear_workspace_bytes(M, N, K, ty, byref(need)), 'hotk_linear_workspace_bytes')
    ws = torch.empty(need.value, dtype=torch.uint8, device=x.device) if need.value else None
    ptr = lambda t: 0 if t is None else t.data_ptr()
    a = LinearArgs(M=M, N=N, K=K, x=ptr(x), ld_x=ld_x, w=ptr(w), ld_w=ld_w, bias=ptr(bias), res=ptr(res), ld_res=ld_res,
                   y=ptr(y), ld_y=N, save=ptr(save), x_scale=ptr(x_scale), w_scale=ptr(w_scale), type=ty,
                   out_type=_TYPES[out_dtype], act=act, reserved=0)
    moved = (M + N) * K * x.element_size() + M * N * y.element_size() * (1 + (res is not None))
    call('hotk_linear_act', moved, byref(a), p(ws), need.value)
    return y


class _LinearAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, keep_slope):
        ctx.set_materialize_grads(False)
        with torch.cuda.device(x.device):
            xs, ld_x, M = _rows(x)
            ws, ld_w, N = _rows(weight)
            K, ty = x.size(-1), _TYPES[x.dtype]
            rs, ld_r = (None, 0) if residual is None else _rows(residual)[:2]
            xa, ld_xa = _aligned(xs, ld_x, M, K, ty)
            wa, ld_wa = _aligned(ws, ld_w, N, K, ty)
            save = None
            if act and keep_slope:
                save = torch.empty(M, N, dtype=torch.float32 if ty == TYPE_F32 else torch.int16, device=x.device)
            y = _product(xa, ld_xa, wa, ld_wa, M, N, _up(K, x.element_size()), ty, x.dtype, None if bias is None else bias.contiguous(),
                         rs, ld_r, act, save)
        ctx.save_for_backward(x, weight, save)
        ctx.cfg = (M, N, K, ty, act)
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, save = ctx.saved_tensors
        M, N, K, ty, act = ctx.cfg
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        if dy is None:
            return (None,) * 6
        dx = dw = db = None
        if M == 0:
            dx = torch.zeros_like(x) if want_x else None
            dw = torch.zeros_like(weight) if want_w else None
            db = torch.zeros(N, dtype=x.dtype, device=x.device) if want_b else None
            return dx, dw, db, dy if want_r else None, None, None
        if want_x or want_w or want_b:
            with torch.cuda.device(x.device):
                size = x.element_size()
                empty = lambda *s, dtype=x.dtype: torch.empty(*s, dtype=dtype, device=x.device)
                gs, ld_g, _ = _rows(dy)
                Np, Mp = _up(N, size), _up(M, size)
                # dz (dy itself where there is no activation and its rows can be read in place), its transpose for dw, and
                # its column sums, from one pass
                plain = not act and (N * size) % 16 == 0 and (ld_g * size) % 16 == 0 and gs.data_ptr() % 16 == 0
                dz = None if plain or not want_x else empty(M, Np)
                dzt = empty(N, Mp) if want_w else None
                part = empty(-(-M // 64), N, dtype=torch.float32) if want_b else None
                if dz is not None or dzt is not None or part is not None:
                    _turn(gs, ld_g, M, N, ty, save, act, dz, Np, dzt, Mp, part)
                if want_b:
                    db = empty(N)
                    call('hotk_sum_partials', 4 * part.numel(), p(part), part.size(0), N, p(db), ty)
                if want_x:
                    ws, ld_w, _ = _rows(weight)
                    wt = empty(K, Np)
                    _turn(ws, ld_w, N, K, ty, out_t=wt, ld_t=Np)
                    dx = _product(gs if plain else dz, ld_g if plain else Np, wt, Np, M, K, Np, ty, x.dtype).view(x.shape)
                if want_w:
                    xs, ld_x, _ = _rows(x)
                    xt = empty(K, Mp)
                    _turn(xs, ld_x, M, K, ty, out_t=xt, ld_t=Mp)
                    dw = _product(dzt, Mp, xt, Mp, N, K, Mp, ty, x.dtype)
        return dx, dw, db, dy if want_r else None, None, None


def _act_code(act):
    if act not in ACTS:
        raise HotkError(f'act: one of {sorted(ACTS)} expected, got {act!r}')
    return ACTS[act]


def linear_act(x, weight, bias=None, act='none', residual=None):
    """y = act(x @ weight.T + bias) + residual in one product: x [..., K], weight [N, K] (torch.nn.Linear's layout), bias [N],
    residual and y [..., N], one type (fp32, bf16, fp16).  act: 'none', 'relu', 'leakyrelu' (slope 0.01), 'gelu' (by erf),
    'tanh', 'silu'.  Differentiable in x, weight, bias and residual.

    Rows that start at 16-byte boundaries and hold whole 16-byte pieces (K a multiple of 8, of 4 in fp32) are read in place;
    others are copied once with zeros behind them.  Rows of up to 8 MiB, else HotkError."""
    _input(x, 'x')
    code = _act_code(act)
    _linear_args(x, weight, bias, residual, x.dtype)
    return _LinearAct.apply(x, weight, bias, residual, code, _wants_grad(x, weight, bias))


def _linear_args(x, weight, bias, residual, out_dtype):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.size(0) == 0:
        raise HotkError('weight: [N, K] with N >= 1 expected')
    N, K = weight.shape
    if x.size(-1) != K:
        raise HotkError(f'x has rows of {x.size(-1)}, weight of {K}')
    _same(x, weight, 'weight', (N, K))
    if bias is not None:
        _same(x, bias, 'bias', (N,), out_dtype)
    if residual is not None:
        _same(x, residual, 'residual', (*x.shape[:-1], N), out_dtype)


def linear_act_quantized(xq, x_scale, wq, w_scale, bias=None, act='none', residual=None, out_dtype=torch.bfloat16):
    """y = act((xq @ wq.T) * x_scale[:, None] * w_scale + bias) + residual over 8-bit operands as quantize_rows and
    rms_norm_quantized make them: xq [..., K], wq [N, K] torch.float8_e4m3fn, x_scale [...], w_scale [N] fp32; bias, residual
    and y in out_dtype (bf16, fp16, fp32).  For an fp32 result products are added up in 32 bits; for 16-bit ones the 8-bit
    matrix instruction adds them by eights to 2^-13 of the largest of the eight, and the eights in 32 bits.  K a multiple of 16
    is read in place.  No gradient."""
    _input(xq, 'xq', eight=True)
    if xq.dtype != E4M3:
        raise HotkError(f'xq: {E4M3} expected, got {xq.dtype}')
    if out_dtype not in _TYPES:
        raise HotkError(f'out_dtype: fp32, bf16 or fp16 expected, got {out_dtype}')
    code = _act_code(act)
    _linear_args(xq, wq, bias, residual, out_dtype)
    _same(xq, x_scale, 'x_scale', xq.shape[:-1], torch.float32)
    _same(xq, w_scale, 'w_scale', wq.shape[:1], torch.float32)
    _refuse_grad('linear_act_quantized', bias, residual, x_scale, w_scale)
    with torch.cuda.device(xq.device):
        xs, ld_x, M = _rows(xq)
        ws, ld_w, N = _rows(wq)
        K = xq.size(-1)
        rs, ld_r = (None, 0) if residual is None else _rows(residual)[:2]
        xa, ld_xa = _aligned(xs, ld_x, M, K, TYPE_E4M3)
        wa, ld_wa = _aligned(ws, ld_w, N, K, TYPE_E4M3)
        y = _product(xa, ld_xa, wa, ld_wa, M, N, _up(K, 1), TYPE_E4M3, out_dtype, None if bias is None else bias.contiguous(), rs,
                     ld_r, code, None, x_scale.contiguous(), w_scale.contiguous())
    return y.view(*xq.shape[:-1], N)
