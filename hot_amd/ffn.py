"""The feed-forward operators: root-mean-square norm of a residual stream (with its result in 8 bits where a product of 8-bit
operands follows), rows to 8 bits with scales, and the matrix product with bias, activation and residual in its epilogue.
All are reached through `hot_amd.ops`; host side in csrc/ffn_torch.cpp, kernels in csrc/rmsnorm.hip and csrc/linact.hip.

Tensors are fp32, bf16 or fp16 on one HIP device, [..., width], read in place when their rows lie at one stride; results are
new, contiguous tensors.  Sums, statistics and epilogues are in 32 bits and every result is rounded once.  Launches go to the
current stream of the tensors' device; workspaces come from torch's allocator per call, so calls can be captured into a
graph and captured graphs share nothing.  Gradients are of first order and in reverse mode; create_graph=True is refused in the backward pass, and tensors that carry a
forward-mode derivative (torch.autograd.forward_ad) everywhere, as are tensors that stand for others (torch.func, vmap, classes
with __torch_dispatch__)."""
import torch

from . import _lib
from ._lib import HotkError, KEEP_VALID

_binding = None


def _ext():
    """the compiled host side, tied to the loaded library on first use"""
    global _binding
    if _binding is None:
        _binding = _lib.torch_binding()
    return _binding


def _wrong(name, e):
    return HotkError(f'{name}: an argument is not of the documented kind ({str(e).splitlines()[0]})')


def rms_norm(x, weight, residual=None, eps=1e-6, kind=None, keep=KEEP_VALID):
    """y = h * (mean(h^2) + eps)^-1/2 * weight over the last dimension, h = x; with a residual h = x + residual, rounded to the
    type as the stream is stored, and the result is (y, h).

    x, residual [..., D], weight [D], one type (fp32, bf16, fp16), D <= 32768.  kind (uint8, one per row: a plan's `kind` or
    `nkind`) and keep: rows that keep leaves out are not read, and are zero in y, h and the gradients.  The squares are added up in
    fp32: a row whose sum of squares passes its range (3e38, elements of some 1e18) comes out as zeros.  Differentiable in x,
    weight and residual."""
    try:
        return (_binding or _ext()).rms_norm(x, weight, residual, eps, kind, keep)
    except TypeError as e:
        raise _wrong('rms_norm', e) from None


def rms_norm_quantized(x, weight, residual=None, eps=1e-6, kind=None, keep=KEEP_VALID):
    """rms_norm with y in 8 bits for a product of 8-bit operands (linear_act_quantized): (q, scale), with a residual (q, scale,
    h).  scale[row] = max(max|y| / 448, 2^-126) in fp32, q = e4m3(y / scale), torch.float8_e4m3fn, from y in 32 bits.  A row
    that holds an infinity or NaN comes out with a scale that is one.  No gradient."""
    try:
        return (_binding or _ext()).rms_norm_quantized(x, weight, residual, eps, kind, keep)
    except TypeError as e:
        raise _wrong('rms_norm_quantized', e) from None


def quantize_rows(x):
    """(q, scale): rows of x [..., D] (fp32, bf16, fp16; D <= 32768) to torch.float8_e4m3fn with one fp32 scale each, scale =
    max(max|x| / 448, 2^-126), q = e4m3(x / scale): the operands of linear_act_quantized, weights ([N, K], a scale per output
    column) as well as activations.  A row that holds an infinity or NaN comes out with a scale that is one.  No gradient."""
    try:
        return (_binding or _ext()).quantize_rows(x)
    except TypeError as e:
        raise _wrong('quantize_rows', e) from None


def linear_act(x, weight, bias=None, act='none', residual=None, dz_parts=None):
    """y = act(x @ weight.T + bias) + residual in one product: x [..., K], weight [N, K] (torch.nn.Linear's layout), bias [N],
    residual and y [..., N], one type (fp32, bf16, fp16).  act: 'none', 'relu', 'leakyrelu' (slope 0.01), 'gelu' (by erf),
    'tanh', 'silu'.  Differentiable in x, weight, bias and residual.

    dz_parts, for the gradients of bf16 and fp16 behind an activation: the two products take dz = dy act'(z) rounded to the type
    (1: dx and dw are off by 1.4 times their own rounding) or as two numbers of the type (2: by their rounding alone, for twice the
    matrix work).  None: two parts up to M N K = 2^25, one above, so a gradient's precision goes by the batch's size; name one
    where it should not.

    Rows that start at 16-byte boundaries and hold whole 16-byte pieces (K a multiple of 8, of 4 in fp32) are read in place;
    others are copied once with zeros behind them; up to 64 rows of x, where the kernel for few rows is the faster one, are
    read at any alignment, and the weight with them.  Rows of x and weight hold up to 8 MiB, those of y too where x or weight has a
    gradient, else HotkError; shorter rows that lie further apart are copied."""
    try:
        return (_binding or _ext()).linear_act(x, weight, bias, act, residual, dz_parts)
    except TypeError as e:
        raise _wrong('linear_act', e) from None


def linear_act_quantized(xq, x_scale, wq, w_scale, bias=None, act='none', residual=None, out_dtype=torch.bfloat16):
    """y = act((xq @ wq.T) * x_scale[:, None] * w_scale + bias) + residual over 8-bit operands as quantize_rows and
    rms_norm_quantized make them: xq [..., K], wq [N, K] torch.float8_e4m3fn, x_scale [...], w_scale [N] fp32; bias, residual
    and y in out_dtype (bf16, fp16, fp32).  For an fp32 result products are added up in 32 bits; for 16-bit ones the 8-bit
    matrix instruction adds them by eights to 2^-13 of the largest of the eight, and the eights in 32 bits.  K a multiple of 16
    is read in place.  No gradient."""
    try:
        return (_binding or _ext()).linear_act_quantized(xq, x_scale, wq, w_scale, bias, act, residual, out_dtype)
    except TypeError as e:
        raise _wrong('linear_act_quantized', e) from None
