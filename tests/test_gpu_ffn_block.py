"""GPU (-m gpu): the k-uniform encoder's feed-forward block with hooks and replaced members, against the same block in 64 bits."""
import pytest
import torch
import torch.nn as nn

from test_gpu_ffn_models import DEV, E, rms64, uniform

pytestmark = pytest.mark.gpu


def inner_of(layer, x, idx):
    return layer.attn(layer.ln(x), idx)


@pytest.mark.parametrize('residual', [False, True])
def test_hooks_run_and_change_nothing_but_the_order_of_sums(residual):
    enc, x, _ = uniform(seed=21)
    layer = enc.layers[0]
    layer.residual = residual
    h = enc.input(x).detach()
    fused = layer(h).detach()
    seen = []
    handles = [m.register_forward_hook(lambda m, i, o: seen.append((type(m).__name__, tuple(o.shape)))) for m in (layer.ffn, *layer.ffn)]
    called = layer(h).detach()
    assert seen == [('RMSNorm', (70, 48)), ('Linear', (70, 80)), ('GELU', (70, 80)), ('Linear', (70, 48)), ('Dropout', (70, 48)), ('Sequential', (70, 48))]
    # two sums of 48 and 80 terms in 32 bits on either side
    assert float((called.double() - fused.double()).abs().max()) <= 8 * (48 + 80 + 64) * E * float(fused.double().abs().max())
    handles[2].remove()
    doubled = layer.ffn[1].register_forward_hook(lambda m, i, o: 2 * o)
    assert not torch.allclose(layer(h).detach(), fused, rtol=1e-2, atol=1e-2)           # a hook's result counts
    doubled.remove()
    for k in (0, 1, 3, 4, 5):
        handles[k].remove()
    assert torch.equal(layer(h).detach(), fused)


def test_replaced_members_are_what_runs():
    enc, x, _ = uniform(seed=22)
    layer = enc.layers[0]
    h = enc.input(x).detach()
    layer.ffn[2] = nn.ReLU()
    p = {k: v.detach().double() for k, v in layer.ffn.named_parameters()}
    a = inner_of(layer, h, None).detach().double()
    want = torch.relu(rms64(a, p['0.weight']) @ p['1.weight'].t() + p['1.bias']) @ p['3.weight'].t() + p['3.bias'] + a
    got = layer(h).detach()
    assert float((got.double() - want).abs().max()) <= 4 * (48 + 80 + 64) * E * float(want.abs().max())


def test_8_bits_refuse_a_changed_block():
    from hot_amd._lib import HotkError
    enc, x, idx = uniform(seed=23)
    enc.eval()
    with torch.no_grad():
        eight = enc.quantize_feed_forward()(x, idx)
        layer = enc.layers[1]
        for change in (lambda: layer.ffn[1].register_forward_hook(lambda *_: None), lambda: layer.ffn.register_forward_pre_hook(lambda *_: None)):
            handle = change()
            with pytest.raises(HotkError, match='as it was assembled'):
                enc(x, idx)
            handle.remove()
            assert torch.equal(enc(x, idx), eight)
        for k, other in ((2, nn.ReLU()), (1, nn.Identity()), (1, nn.Linear(48, 80).to(DEV))):
            own, layer.ffn[k] = layer.ffn[k], other
            with pytest.raises(HotkError):
                enc(x, idx)
            layer.ffn[k] = own
            assert torch.equal(enc(x, idx), eight)
        whole, layer.ffn = layer.ffn, nn.Sequential(nn.Identity())
        with pytest.raises(HotkError):
            enc(x, idx)
        layer.ffn = whole
        assert torch.equal(enc(x, idx), eight)
