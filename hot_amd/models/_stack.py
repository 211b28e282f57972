"""Shared assembly helpers for the model stacks (Encoder / EncLayer / MLP in the sparse, dense and k-uniform layouts).

What is fixed by checkpoint compatibility with the reference (hot_pytorch/models/encoder.py:20-96, mlp.py:15-40,
extension.py:20-124) is the set of attribute names and the position of parameterised modules inside each nn.Sequential --
nothing else.  This module holds the pieces the three stacks share, written once:

  * a `Layout` record naming the building blocks of a data layout (which Linear, which pointwise wrapper, which attention);
  * `orders_and_widths`, the (order, width) schedule of a stack from its constructor arguments;
  * `pre_norm_block`, the LayerNorm -> Linear -> GELU -> Linear -> Dropout feed-forward block whose parameterised members
    sit at Sequential positions 0, 1 and 3 (keys `ffn.0.*`, `ffn.1.*`, `ffn.3.*`);
  * `norm_of`, the norm that a stack's norm='layernorm' | 'rmsnorm' names, and `feed_forward`, the block over plain rows with
    RMSNorm: norm, product with GELU, product with the residual, each one kernel (a block whose members have been replaced or
    have hooks runs member by member);
  * `shared_feature_map`, the one FAVOR+ map an encoder hands to all its kernel-attention layers, and `maybe_redraw`.
"""
from collections import namedtuple

import torch
import torch.nn as nn

from .. import ops
from .._lib import HotkError
from .common.kernel import KernelFeatureMap
from .common.rmsnorm import RMSNorm

Layout = namedtuple('Layout', 'name linear apply nonlinear add kernel_attn readout_attn batch_type')


def sparse_layout():
    from .sparse.linear import Linear
    from .sparse.f import Apply, Nonlinear, Add
    from .sparse.kernelattn import KernelSelfAttn
    from .sparse.attn import SelfAttn
    from ..batch.sparse import Batch
    return Layout('sparse', Linear, Apply, Nonlinear, Add, KernelSelfAttn, SelfAttn, Batch)


def dense_layout():
    from .dense.linear import Linear
    from .dense.f import Apply, Nonlinear, Add
    from .dense.kernelattn import KernelSelfAttn
    from .dense.attn import SelfAttn
    from ..batch.dense import Batch
    return Layout('dense', Linear, Apply, Nonlinear, Add, KernelSelfAttn, SelfAttn, Batch)


def layout_of(sparse: bool) -> Layout:
    return sparse_layout() if sparse else dense_layout()


def orders_and_widths(ord_in, ord_hidden, ord_out, dim_in, dim_hidden, dim_out):
    """[(order_k, width_k)] for k = 0 .. n_layers: the tensors between the layers of a stack.  dim_hidden may be one int
    (all hidden widths equal) or a list with one width per hidden tensor."""
    hidden = list(ord_hidden)
    widths = list(dim_hidden) if isinstance(dim_hidden, (list, tuple)) else [dim_hidden] * len(hidden)
    if len(widths) != len(hidden):
        raise ValueError(f'{len(hidden)} hidden orders but {len(widths)} hidden widths')
    return list(zip([ord_in] + hidden + [ord_out], [dim_in] + widths + [dim_out]))


def pre_norm_block(norm, first, act, second, drop):
    """feed-forward block; parameterised members at positions 0, 1, 3"""
    return nn.Sequential(norm, first, act, second, drop)


def norm_of(name, dim):
    if name not in ('layernorm', 'rmsnorm'):
        raise AssertionError(f'unknown norm {name!r}')
    return nn.LayerNorm(dim) if name == 'layernorm' else RMSNorm(dim)


_MODULE_HOOKS = ('_forward_pre_hooks', '_forward_hooks', '_backward_pre_hooks', '_backward_hooks')


def _plain_call(m, cls):
    """calling m runs cls.forward and nothing else"""
    return type(m) is cls and 'forward' not in m.__dict__ and not any(getattr(m, name) for name in _MODULE_HOOKS)


def _as_assembled(ffn):
    """the block is what pre_norm_block made of RMSNorm, nn.Linear, GELU by erf, nn.Linear and nn.Dropout, without hooks"""
    everywhere = torch.nn.modules.module
    return (_plain_call(ffn, nn.Sequential) and len(ffn) == 5
            and all(_plain_call(m, cls) for m, cls in zip(ffn, (RMSNorm, nn.Linear, nn.GELU, nn.Linear, nn.Dropout))) and ffn[2].approximate == 'none'
            and not any(getattr(everywhere, '_global' + name, None) for name in _MODULE_HOOKS))


def feed_forward(ffn, x, residual=None, eight=None):
    """h + ffn(h) for a pre_norm_block over rows, h = x (+ residual); with the members that an encoder of norm='rmsnorm' gives it
    three kernels, otherwise (a member replaced, or hooks on the block or a member) the block as it is called.  eight: the
    block's two weights and their scales in 8 bits (quantize_block): the products then take 8-bit rows (no gradient)"""
    if not _as_assembled(ffn):
        if eight is not None:
            raise HotkError('8-bit feed-forward products take the block as it was assembled: its members have been replaced, or hooks set')
        h = x if residual is None else x + residual
        return h + ffn(h)
    norm, first, _, second, drop = ffn
    if eight is not None:
        w1, s1, w2, s2 = eight
        q, s, *h = ops.rms_norm_quantized(x, norm.weight, residual, eps=norm.eps)
        u = ops.linear_act_quantized(q, s, w1, s1, first.bias, act='gelu', out_dtype=x.dtype)
        return ops.linear_act_quantized(*ops.quantize_rows(u), w2, s2, second.bias, residual=h[0] if h else x, out_dtype=x.dtype)
    y, h = (norm(x), x) if residual is None else norm(x, residual)
    u = ops.linear_act(y, first.weight, first.bias, act='gelu')
    if drop.training and drop.p > 0:
        return h + drop(ops.linear_act(u, second.weight, second.bias))
    return ops.linear_act(u, second.weight, second.bias, residual=h)


def quantize_block(ffn):
    """a block's weights for feed_forward(eight=...): 8 bits with one scale per output column"""
    if not _as_assembled(ffn):
        raise HotkError('8-bit feed-forward products take the block as it was assembled: its members have been replaced, or hooks set')
    with torch.no_grad():
        return (*ops.quantize_rows(ffn[1].weight), *ops.quantize_rows(ffn[3].weight))


def shared_feature_map(att_cfg, dim_qk, n_heads):
    """(feature map or None, skip_redraw flag): kernel attention variants share ONE projection per encoder, redrawn on
    every training forward unless the flag is set by the user (encoder.py:71-75)"""
    if att_cfg not in ('kernel', 'generalized_kernel'):
        return None, True
    width = dim_qk // n_heads if dim_qk >= n_heads else 1
    return KernelFeatureMap(width, generalized_attention=(att_cfg == 'generalized_kernel')), False


def maybe_redraw(module):
    if module.feature_map is not None and not module.skip_redraw_projections:
        module.feature_map.redraw_projections()
