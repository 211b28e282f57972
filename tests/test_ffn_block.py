"""CPU (no GPU): when the k-uniform encoder's feed-forward block may run as fused kernels, and that another one runs as it is called."""
import pytest
import torch
import torch.nn as nn

from hot_amd._lib import HotkError
from hot_amd.models import _stack
from hot_amd.models.common.rmsnorm import RMSNorm


def block(p=0.):
    return _stack.pre_norm_block(RMSNorm(8), nn.Linear(8, 12), nn.GELU(), nn.Linear(12, 8), nn.Dropout(p, inplace=True))


class Low(nn.Linear):
    def forward(self, x):
        return super().forward(x) + x.sum(-1, keepdim=True)


def seen(*_):
    return None


CHANGES = {
    'norm': lambda f: f.__setitem__(0, nn.LayerNorm(8)), 'first': lambda f: f.__setitem__(1, Low(8, 12)), 'act': lambda f: f.__setitem__(2, nn.ReLU()),
    'act form': lambda f: f.__setitem__(2, nn.GELU('tanh')), 'second': lambda f: f.__setitem__(3, nn.Sequential(nn.Linear(12, 8))),
    'dropout': lambda f: f.__setitem__(4, nn.AlphaDropout(0.5)), 'one more': lambda f: f.append(nn.Tanh()), 'one less': lambda f: f.__delitem__(4),
    'own forward': lambda f: setattr(f[2], 'forward', torch.relu), 'parametrized': lambda f: nn.utils.parametrizations.weight_norm(f[1]),
    'hook on the block': lambda f: f.register_forward_hook(seen), 'hook on a product': lambda f: f[1].register_forward_hook(seen),
    'hook before the activation': lambda f: f[2].register_forward_pre_hook(seen), 'hook on the norm': lambda f: f[0].register_forward_hook(seen),
    'backward hook': lambda f: f[3].register_full_backward_hook(seen), 'backward hook before': lambda f: f[3].register_full_backward_pre_hook(seen),
}


@pytest.mark.parametrize('change', CHANGES)
def test_a_changed_block_is_not_fused(change):
    f = block()
    assert _stack._as_assembled(f)
    back = CHANGES[change](f)
    assert not _stack._as_assembled(f)
    with pytest.raises(HotkError, match='as it was assembled'):
        _stack.quantize_block(f)
    with pytest.raises(HotkError, match='as it was assembled'):
        _stack.feed_forward(f, torch.randn(3, 8), None, eight=(None,) * 4)
    if hasattr(back, 'remove'):
        back.remove()
        assert _stack._as_assembled(f)


def test_hooks_on_all_modules():
    f = block()
    handle = nn.modules.module.register_module_forward_hook(seen)
    try:
        assert not _stack._as_assembled(f)
    finally:
        handle.remove()
    assert _stack._as_assembled(f)


@pytest.mark.parametrize('residual', [False, True])
def test_a_changed_block_runs_as_it_is_called(residual):
    """a LayerNorm in place of the norm: the whole block is torch modules, so it runs here"""
    f = block()
    f[0], f[2] = nn.LayerNorm(8), nn.ReLU()
    calls = []
    f[1].register_forward_hook(lambda m, i, o: calls.append(tuple(o.shape)))
    x, r = torch.randn(3, 8), torch.randn(3, 8) if residual else None
    h = x + r if residual else x
    assert torch.equal(_stack.feed_forward(f, x, r), h + f(h)) and calls == [(3, 12)] * 2
