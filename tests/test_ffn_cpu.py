"""CPU (no GPU): what the feed-forward operators refuse, on the Python side and at the C entries; size queries."""
import ctypes

import pytest
import torch

from hot_amd import _lib, ops
from hot_amd._lib import HotkError

L = _lib.lib()
NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(4096)         # an address that is never followed: every call below ends before a launch
EINVAL, EWORKSPACE, EUNSUPPORTED, ETOOLARGE = -1, -2, -4, -5


def test_no_cpu_path():
    x, w = torch.randn(3, 8), torch.randn(8)
    for f in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_quantized(x, w), lambda: ops.quantize_rows(x),
              lambda: ops.linear_act(x, torch.randn(4, 8)),
              lambda: ops.linear_act_quantized(x.to(torch.float8_e4m3fn), x[:, 0], torch.randn(4, 8).to(torch.float8_e4m3fn), x[0])):
        with pytest.raises(HotkError):
            f()


@pytest.mark.parametrize('bad', [None, 3, 'x'])
def test_not_a_tensor(bad):
    for f in (ops.quantize_rows, lambda v: ops.rms_norm(v, torch.ones(2)), lambda v: ops.linear_act(v, torch.ones(2, 2))):
        with pytest.raises(HotkError):
            f(bad)


def test_norm_entries_refuse():
    fwd = lambda x=SOME, ld=8, res=NULL, h=NULL, y=SOME, R=2, D=8, ty=0: L.hotk_rmsnorm_fwd(
        x, ld, res, 8, SOME, NULL, 6, 1e-6, y, h, NULL, R, D, ty, NULL)
    assert fwd(R=0) == 0
    assert fwd(x=NULL) == EINVAL and fwd(y=NULL) == EINVAL and fwd(ld=7) == EINVAL and fwd(R=-1) == EINVAL
    assert fwd(res=SOME, h=NULL) == EINVAL
    assert fwd(x=ctypes.c_void_p(4098)) == EINVAL                      # an fp32 row between two elements
    assert fwd(D=0) == EUNSUPPORTED and fwd(D=32769, ld=40000) == EUNSUPPORTED and fwd(ty=3) == EUNSUPPORTED and fwd(ty=9) == EUNSUPPORTED
    assert L.hotk_rmsnorm_supported(32768, 1) == 1 and L.hotk_rmsnorm_supported(32769, 1) == 0
    assert L.hotk_quantize_rows(SOME, 8, NULL, SOME, 2, 8, 0, NULL) == EINVAL
    assert L.hotk_quantize_rows(NULL, 8, NULL, NULL, 0, 8, 0, NULL) == 0
    assert L.hotk_rmsnorm_quant(SOME, 8, NULL, 0, SOME, NULL, 6, 1e-6, SOME, NULL, NULL, 2, 8, 0, NULL) == EINVAL
    bwd = lambda rstd=SOME, part=NULL, dw=SOME, R=2: L.hotk_rmsnorm_bwd(SOME, 8, NULL, 0, SOME, 8, rstd, SOME, NULL, 6, SOME, part, dw, R, 8, 0, NULL)
    assert bwd(rstd=NULL) == EINVAL and bwd(part=SOME) == EINVAL                      # few rows: no partial sums
    assert bwd(R=5000) == EINVAL and bwd(R=5000, part=SOME) == EINVAL                 # many: those, and no dw
    assert L.hotk_sum_partials(NULL, 3, 4, SOME, 0, NULL) == EINVAL and L.hotk_sum_partials(NULL, 0, 0, NULL, 0, NULL) == 0
    n = ctypes.c_int64()
    for R, D, ty in ((0, 8, 0), (1, 8, 1), (1024, 8, 1), (1025, 8, 1), (100000, 8, 2), (100000, 32768, 0)):
        assert L.hotk_rmsnorm_partials(R, D, ty, ctypes.byref(n)) == 0 and min(1, R // 1025) <= n.value <= R // 1025 * R


def _args(**kw):
    a = dict(M=4, N=8, K=32, x=4096, ld_x=32, w=4096, ld_w=32, bias=0, res=0, ld_res=0, y=4096, ld_y=8, save=0, x_scale=0,
             w_scale=0, type=1, out_type=1, act=0, flags=0, x_lo=0)
    a.update(kw)
    return _lib.LinearArgs(**a)


@pytest.mark.parametrize('why,change,code', [
    ('no x', dict(x=0), EINVAL), ('no w', dict(w=0), EINVAL), ('no y', dict(y=0), EINVAL), ('rows overlap', dict(ld_x=24), EINVAL),
    ('w rows overlap', dict(ld_w=24), EINVAL), ('y rows overlap', dict(ld_y=7), EINVAL), ('res rows overlap', dict(res=4096, ld_res=7), EINVAL),
    ('no width', dict(K=0, ld_x=0), EINVAL), ('no columns', dict(N=0), EINVAL), ('negative rows', dict(M=-1), EINVAL),
    ('act', dict(act=6), EINVAL), ('act', dict(act=-1), EINVAL), ('type', dict(type=7), EUNSUPPORTED), ('out type', dict(out_type=3), EUNSUPPORTED),
    ('mixed types', dict(out_type=0), EUNSUPPORTED), ('8 bits without scales', dict(type=3), EINVAL),
    ('scales without 8 bits', dict(x_scale=4096, w_scale=4096), EINVAL), ('one scale', dict(type=3, x_scale=4096), EINVAL),
    ('slope of 8 bits', dict(type=3, x_scale=4096, w_scale=4096, save=4096), EINVAL),
    ('half a piece', dict(M=400, K=28, ld_x=28, ld_w=28), EUNSUPPORTED), ('ends inside a piece', dict(M=400, K=28), EUNSUPPORTED), ('x down alone', dict(flags=1, ld_x=8), EUNSUPPORTED),
    ('unknown flag', dict(flags=8), EINVAL), ('second part between pieces', dict(flags=2, ld_w=8, x_lo=4098), EUNSUPPORTED),
    ('second part of 8 bits', dict(type=3, x_scale=4096, w_scale=4096, x_lo=4096), EUNSUPPORTED), ('8 bits down', dict(type=3, x_scale=4096, w_scale=4096, flags=2, ld_w=32), EUNSUPPORTED),
    ('w columns in no whole pieces', dict(flags=2, N=5, ld_w=5, ld_y=5), EUNSUPPORTED), ('row stride', dict(M=400, ld_x=36), EUNSUPPORTED), ('w row stride', dict(M=400, ld_w=36), EUNSUPPORTED),
    ('x between pieces', dict(M=400, x=4098), EUNSUPPORTED), ('w between pieces', dict(M=400, w=4104), EUNSUPPORTED),
    ('x between elements', dict(x=4097), EINVAL), ('w between elements', dict(w=4097), EINVAL),
    ('y between elements', dict(y=4097), EINVAL), ('bias between elements', dict(bias=4097), EINVAL),
    ('row too long', dict(ld_x=1 << 23), ETOOLARGE)])
def test_product_entry_refuses(why, change, code):
    assert L.hotk_linear_act(ctypes.byref(_args(**change)), NULL, 0, NULL) == code, why


def test_product_entry_empty_and_workspace():
    assert L.hotk_linear_act(ctypes.byref(_args(M=0, x=0, w=0, y=0)), NULL, 0, NULL) == 0
    assert L.hotk_linear_act(None, NULL, 0, NULL) == EINVAL
    need = ctypes.c_size_t()
    assert L.hotk_linear_workspace_bytes(ctypes.byref(_args(K=0, ld_x=0)), ctypes.byref(need)) == EINVAL
    long = dict(M=128, N=128, K=65536, ld_x=65536, ld_w=65536, ld_y=128)                         # few tiles, a long contraction
    assert L.hotk_linear_workspace_bytes(ctypes.byref(_args(**long)), ctypes.byref(need)) == 0 and need.value > 0
    assert L.hotk_linear_act(ctypes.byref(_args(**long)), NULL, 0, NULL) == EWORKSPACE
    assert L.hotk_linear_act(ctypes.byref(_args(**long)), NULL, need.value, NULL) == EWORKSPACE
    assert L.hotk_linear_act(ctypes.byref(_args(**long)), SOME, need.value - 1, NULL) == EWORKSPACE
    assert L.hotk_linear_workspace_bytes(ctypes.byref(_args()), ctypes.byref(need)) == 0 and need.value == 0


def test_backward_entries_refuse():
    dz = lambda i=SOME, ld=8, save=NULL, act=0, out=SOME, lo=NULL, ld_o=8, part=NULL, total=NULL, R=4, C=8, ty=1: L.hotk_linear_dz(
        i, ld, save, act, out, lo, ld_o, part, total, R, C, ty, NULL)
    assert dz(R=0) == 0
    assert dz(i=NULL) == EINVAL and dz(ld=7) == EINVAL and dz(ld_o=7) == EINVAL and dz(out=NULL) == EINVAL and dz(C=0, ld=0, ld_o=0) == EINVAL
    assert dz(act=3) == EINVAL and dz(act=6, save=SOME) == EINVAL and dz(i=ctypes.c_void_p(4097)) == EINVAL
    assert dz(total=SOME, R=2000) == EINVAL and dz(total=SOME, part=SOME) == EINVAL          # a total of one block only
    assert dz(out=NULL, lo=SOME, part=SOME) == EINVAL                                        # the rest of nothing
    assert dz(ty=5) == EUNSUPPORTED and dz(ty=3) == EUNSUPPORTED
    n = ctypes.c_int64()
    for R in (0, 1, 16, 17, 8191, 8193, 10 ** 7):
        assert L.hotk_linear_dz_partials(R, ctypes.byref(n)) == 0 and min(R, 1) <= n.value <= min(R, 512), (R, n.value)
    pad = lambda i=SOME, ld=8, out=SOME, ld_o=16, R=4, nb=8: L.hotk_pad_rows(i, ld, out, ld_o, R, nb, NULL)
    assert pad(R=0) == 0 and pad(i=NULL) == EINVAL and pad(ld=7) == EINVAL and pad(ld_o=8) == EINVAL and pad(ld_o=24) == EINVAL
    assert pad(out=ctypes.c_void_p(4104)) == EINVAL and pad(nb=0) == EINVAL
