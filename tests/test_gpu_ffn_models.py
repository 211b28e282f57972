"""GPU (-m gpu): the encoders with norm='rmsnorm' -- the feed-forward operators inside the framework's own models -- against the
same modules' parameters in 64 bits, and the 8-bit feed-forward of the k-uniform encoder."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
E = 2.0 ** -24


def rms64(x, w, eps=1e-6):
    return x * ((x * x).mean(-1, keepdim=True) + eps).rsqrt() * w


def uniform(seed=0, dropout=0., dim=48, ff=80, n=70, b=33):
    from hot_amd.models.extension import Encoder
    torch.manual_seed(seed)
    enc = Encoder(1, 3, [1], 24, 8, dim, 16, 16, ff, 4, 8, 8, 4, dropout=dropout, norm='rmsnorm').to(DEV)
    enc.skip_redraw_projections = True
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(n, 24, generator=g).to(DEV)
    idx = torch.stack([torch.randperm(n, generator=g)[:3] for _ in range(b)]).to(DEV)
    return enc, x, idx


def test_uniform_encoder_layer_against_64_bits():
    enc, x, idx = uniform()
    h = enc.input(x)
    for layer in enc.layers:
        at = idx if layer.ord_out != 1 else None
        for residual in (False, True) if at is None else (False,):        # (the skip keeps its rows only where the order stays)
            layer.residual = residual
            inner = layer.attn(layer.ln(h), at).detach()
            got = layer(h, at).detach()
            a = inner.double() + (h.detach().double() if residual else 0)
            p = {k: v.detach().double() for k, v in layer.ffn.named_parameters()}
            n = rms64(a, p['0.weight'])
            want = torch.nn.functional.gelu(n @ p['1.weight'].t() + p['1.bias']) @ p['3.weight'].t() + p['3.bias'] + a
            # two sums of 48 and 80 terms in 32 bits, each below 4 in magnitude against a result of the same size
            assert float((got.double() - want).abs().max()) <= 4 * (48 + 80 + 64) * E * float(want.abs().max())
        layer.residual = False
        h = layer(h, at)


def test_uniform_encoder_gradients_against_64_bits():
    """the feed-forward block's own gradients: the same block in 64 bits under autograd, from the same attention output"""
    from hot_amd.models import _stack
    enc, x, _ = uniform(seed=3)
    layer = enc.layers[0]
    a, r = torch.randn(70, 48, device=DEV, requires_grad=True), torch.randn(70, 48, device=DEV, requires_grad=True)
    dy = torch.randn(70, 48, device=DEV)
    params = list(layer.ffn.parameters())
    got = torch.autograd.grad(_stack.feed_forward(layer.ffn, a, r), [a, r] + params, dy)
    d = [t.detach().double().requires_grad_(True) for t in [a, r] + params]
    h = d[0] + d[1]
    y = torch.nn.functional.gelu(rms64(h, d[2]) @ d[3].t() + d[4]) @ d[5].t() + d[6] + h
    want = torch.autograd.grad(y, d, dy.double())
    for i, (g, w) in enumerate(zip(got, want)):
        assert float((g.double() - w).abs().max()) <= 4 * (48 + 80 + 70 + 64) * E * float(w.abs().max()), i


def test_uniform_encoder_trains_with_dropout():
    enc, x, idx = uniform(seed=5, dropout=0.5)
    enc.train()
    torch.manual_seed(9)
    y = enc(x, idx)
    y.square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in enc.parameters() if p.requires_grad)
    torch.manual_seed(9)
    assert torch.equal(enc(x, idx), y)             # the same draw, the same result
    enc.eval()
    with torch.no_grad():
        assert torch.equal(enc(x, idx), enc(x, idx))


def test_uniform_encoder_serves_in_8_bits():
    from hot_amd import ops
    from hot_amd._lib import HotkError
    enc, x, idx = uniform(seed=7)
    enc.eval()
    keys = list(enc.state_dict())
    with torch.no_grad():
        full = enc(x, idx)
        assert enc.quantize_feed_forward() is enc and list(enc.state_dict()) == keys
        eight = enc(x, idx)
        # the last layer by hand
        h = enc.layers[0](enc.input(x))
        last = enc.layers[1]
        a = last.attn(last.ln(h), idx)
        q, s = ops.rms_norm_quantized(a, last.ffn[0].weight)
        w1, s1 = ops.quantize_rows(last.ffn[1].weight)
        w2, s2 = ops.quantize_rows(last.ffn[3].weight)
        u = ops.linear_act_quantized(q, s, w1, s1, last.ffn[1].bias, act='gelu', out_dtype=torch.float32)
        y = ops.linear_act_quantized(*ops.quantize_rows(u), w2, s2, last.ffn[3].bias, residual=a, out_dtype=torch.float32)
        assert torch.equal(eight, enc.output(y))
        assert not torch.equal(eight, full)
        # each 8-bit value is off by at most 2^-4 of itself, its sums by the root of that over 48 and 80 terms: a few percent
        assert float((eight - full).norm() / full.norm()) < 2.0 ** -4
    with torch.enable_grad():
        assert torch.equal(enc(x, idx).detach(), full)             # with gradients: the full weights
    with torch.no_grad():
        enc.layers[1].ffn[1].weight.mul_(1.5)
        with pytest.raises(HotkError):
            enc(x, idx)
        enc.quantize_feed_forward()
        enc(x, idx)
    from hot_amd.models.extension import EncLayer
    with pytest.raises(HotkError):
        EncLayer(1, 1, 16, 8, 8, 16, 2, att_cfg='generalized_kernel', feature_map=enc.feature_map).quantize_feed_forward()


def test_quantized_encoder_copies_and_replaced_weights():
    """a copy or a pickle serves the full weights, also after its own have changed; weights replaced as a whole are noticed"""
    import copy
    import io
    from hot_amd._lib import HotkError
    enc, x, idx = uniform(seed=9)
    enc.eval()
    with torch.no_grad():
        full = enc(x, idx)
        eight = enc.quantize_feed_forward()(x, idx)
        assert not torch.equal(eight, full)
        f = io.BytesIO()
        torch.save(enc, f)
        f.seek(0)
        for other in (copy.deepcopy(enc), torch.load(f, weights_only=False)):
            assert torch.equal(other(x, idx), full)
            w = other.layers[1].ffn[1].weight
            changed = []
            for _ in range(4):                                       # whatever number its version has
                w.mul_(1.25)
                changed.append(other(x, idx))
            assert not any(torch.equal(c, full) for c in changed)
            assert not torch.equal(other.quantize_feed_forward()(x, idx), changed[-1])
        assert torch.equal(enc(x, idx), eight)
        lin = enc.layers[0].ffn[3]
        for change in (lambda: setattr(lin, 'weight', torch.nn.Parameter(lin.weight * 2)), lambda: setattr(lin.weight, 'data', lin.weight * 2)):
            change()
            with pytest.raises(HotkError):
                enc(x, idx)
            enc.quantize_feed_forward()(x, idx)


def sparse_batch(seed, sizes=(9, 5, 12)):
    from hot_amd.batch import sparse as bs
    from hot_amd.utils.graphs import ba_edges
    import numpy as np
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    ei = [torch.from_numpy(ba_edges(n, 2, rng)) for n in sizes]
    return bs.make_batch([torch.randn(n, 8, generator=g).to(DEV) for n in sizes], [e.to(DEV) for e in ei],
                         [torch.randn(e.size(1), 8, generator=g).to(DEV) for e in ei])


def test_sparse_norm_of_a_padded_batch():
    from hot_amd.batch import sparse as bs
    from hot_amd.models.common import RMSNorm
    from hot_amd.models.sparse import Apply
    G = sparse_batch(11)
    norm = Apply(RMSNorm(40)).to(DEV)
    with torch.no_grad():
        norm.f.weight.copy_(1 + 0.2 * torch.randn(40, device=DEV))
    v = torch.randn(*G.values.shape[:2], 40, device=DEV)
    want = rms64(v.double(), norm.f.weight.double()) * G.mask[..., None]
    v[~G.mask] = float('nan')                                        # padding rows are not read
    v.requires_grad_(True)
    out = norm(bs.batch_like(G, v, skip_masking=True)).values
    assert (out[~G.mask] == 0).all()
    assert float((out.double() - want).abs().max()) <= 200 * E * float(want.abs().max())
    dv, = torch.autograd.grad(out, v, torch.randn_like(out))
    assert (dv[~G.mask] == 0).all() and dv.isfinite().all()


@pytest.mark.parametrize('sparse', [True, False])
def test_encoder_with_rmsnorm_runs_and_has_gradients(sparse):
    from hot_amd.models import Encoder
    from hot_amd.models.common import RMSNorm
    torch.manual_seed(0)
    enc = Encoder(2, 0, [2], 16 if sparse else 6, 4, 32, 32, 32, 64, 4, 16, 16, 4, 'default', 'generalized_kernel', sparse=sparse,
                  norm='rmsnorm').to(DEV)
    assert not any(isinstance(m, torch.nn.LayerNorm) for m in enc.modules()) and any(isinstance(m, RMSNorm) for m in enc.modules())
    if sparse:
        G = sparse_batch(12)
    else:
        from hot_amd.batch.dense import Batch
        A = torch.randn(2, 7, 7, 6, device=DEV)
        G = Batch(A, [7, 5])
    y = enc(G)
    y = y.values if hasattr(y, 'values') and not torch.is_tensor(y) else y
    (y if torch.is_tensor(y) else y.A).square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in enc.parameters() if p.requires_grad)


def test_results_can_be_changed_in_place():
    from hot_amd import ops
    x, w = torch.randn(3, 5, 16, device=DEV, requires_grad=True), torch.randn(8, 16, device=DEV, requires_grad=True)
    y = ops.linear_act(x, w, act='relu')
    y.mul_(2)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    z = ops.linear_act(x, w, act='relu')
    ex, ew = torch.autograd.grad(z, (x, w), torch.full_like(z, 2.))
    assert torch.equal(dx, ex) and torch.equal(dw, ew)
    n, h = ops.rms_norm(x, w[0], x)
    n.add_(1)
    with pytest.raises(RuntimeError):
        h.add_(1)                                     # the stream is what the backward pass reads
        torch.autograd.grad(n, x, torch.ones_like(n))


def test_first_order_only():
    from hot_amd import ops
    x, w = torch.randn(4, 16, device=DEV, requires_grad=True), torch.randn(16, device=DEV, requires_grad=True)
    for y in (ops.rms_norm(x, w), ops.linear_act(x, torch.randn(8, 16, device=DEV), act='silu')):
        with pytest.raises(RuntimeError, match='first order'):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_launches_are_timed_like_the_framework_s_others():
    from hot_amd import _lib, ops
    x, w = torch.randn(1100, 16, device=DEV, requires_grad=True), torch.randn(24, 16, device=DEV, requires_grad=True)
    _lib.timing_begin(None)
    ops.linear_act(ops.rms_norm(x, w[0]), w, act='gelu').sum().backward()
    seen = _lib.timing_end()
    assert {'hotk_rmsnorm_fwd', 'hotk_rmsnorm_bwd', 'hotk_sum_partials', 'hotk_linear_act', 'hotk_linear_dz'} <= set(seen)
    assert seen['hotk_linear_act'][1] == 3 and all(ms >= 0 and calls > 0 and nbytes > 0 for ms, calls, nbytes in seen.values())
    ops.rms_norm(x, w[0])
    assert _lib.timing_end() == {}
