"""GPU (-m gpu): the sparse and dense encoders with norm='rmsnorm': their norms' gradients against 64 bits, and every gradient of a whole
encoder against the same encoder with norms computed by torch in 64 bits."""
import copy

import pytest
import torch
import torch.nn as nn

from test_gpu_ffn_models import DEV, E, rms64, sparse_batch

pytestmark = pytest.mark.gpu
CHAIN = 160     # additions and products behind one gradient of a row of 40 (test_gpu_ffn.py)


def batch_of(sparse, width, seed):
    g = torch.Generator().manual_seed(seed)
    if sparse:
        G = sparse_batch(seed)
        return G, torch.randn(*G.values.shape[:-1], width, generator=g).to(DEV)
    from hot_amd.batch.dense import Batch
    A = torch.randn(2, 7, 7, width, generator=g).to(DEV)
    return Batch(A, [7, 5]), A


def like(G, v):
    if hasattr(G, 'values'):
        from hot_amd.batch import sparse as bs
        return bs.batch_like(G, v)
    from hot_amd.batch.dense import Batch
    return Batch(v, G.n_nodes)


def values(H):
    return H if torch.is_tensor(H) else getattr(H, 'values', getattr(H, 'A', None))


@pytest.mark.parametrize('sparse', [True, False])
def test_gradients_of_a_padded_norm(sparse):
    from hot_amd.models import dense, sparse as sparse_models
    from hot_amd.models.common import RMSNorm
    Apply = (sparse_models if sparse else dense).Apply
    G, v = batch_of(sparse, 40, 31)
    norm = Apply(RMSNorm(40)).to(DEV)
    with torch.no_grad():
        norm.f.weight.copy_(1 + 0.2 * torch.randn(40, generator=torch.Generator().manual_seed(32)))
    v.requires_grad_(True)
    out = values(norm(like(G, v)))
    dy = torch.randn(out.shape, generator=torch.Generator().manual_seed(33)).to(DEV)
    dv, dw = torch.autograd.grad(out, (v, norm.f.weight), dy)
    on = G.mask[..., None].double()
    vd, wd = (v.detach().double() * on).requires_grad_(True), norm.f.weight.detach().double().requires_grad_(True)
    want_v, want_w = torch.autograd.grad(rms64(vd, wd) * on, (vd, wd), dy.double())
    # a row's gradient is rstd (g - u mean(g u)): CHAIN operations of size rstd max|g| (1 + max|u|^2); the weight's a sum over the rows
    rstd = ((vd * vd).mean(-1, keepdim=True) + 1e-6).rsqrt()
    u, g = (vd * rstd).detach(), (dy.double() * wd).detach()
    size = (rstd * g.abs().amax(-1, keepdim=True) * (1 + u.abs().amax(-1, keepdim=True) ** 2) * on).detach()
    assert ((dv.double() - want_v * on).abs() <= 3 * CHAIN * E * size).all()
    terms = (dy.double() * u * on).abs().flatten(0, -2)
    assert ((dw.double() - want_w).abs() <= (CHAIN + terms.size(0)) * E * terms.sum(0)).all()


class Norm64(nn.Module):
    """the norm in 64 bits by torch, under the same parameter's name"""

    def __init__(self, weight, eps):
        super().__init__()
        self.weight, self.eps = weight, eps

    def forward(self, x):
        return rms64(x.double(), self.weight.double(), self.eps).to(x.dtype)


def with_norm64(module):
    from hot_amd.models.common import RMSNorm
    for name, child in module.named_children():
        if type(child) is RMSNorm:
            setattr(module, name, Norm64(child.weight, child.eps))
        else:
            with_norm64(child)
    return module


@pytest.mark.parametrize('sparse', [True, False])
@pytest.mark.parametrize('ord_out', [0, 2])
def test_encoder_gradients_against_norms_in_64_bits(sparse, ord_out):
    """each norm differs by some 64 E of its values; the softmax maps and products behind it may enlarge that tenfold and more: 1e-4
    of each parameter's gradient (of a hundredth of the mean gradient, where one is smaller) leaves twenty-five times that"""
    from hot_amd.models import Encoder
    torch.manual_seed(34)
    enc = Encoder(2, ord_out, [2], 8 if sparse else 6, 4, 32, 32, 32, 64, 4, 16, 16, 4, 'default', 'kernel', sparse=sparse, norm='rmsnorm').to(DEV)
    enc.skip_redraw_projections = True
    other = with_norm64(copy.deepcopy(enc))
    assert [n for n, _ in enc.named_parameters()] == [n for n, _ in other.named_parameters()]
    G, v = batch_of(sparse, 8 if sparse else 6, 35)
    results = []
    for e in (enc, other):
        y = values(e(like(G, v.clone())))
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(36)).to(DEV)
        results.append((y.detach(), torch.autograd.grad(y, [p for p in e.parameters() if p.requires_grad], dy, allow_unused=True)))
    (y, got), (want_y, want) = results
    assert float((y - want_y).norm()) <= 1e-4 * float(want_y.norm())
    names = [n for n, p in enc.named_parameters() if p.requires_grad]
    used = [(n, a.double(), b.double()) for n, a, b in zip(names, got, want) if b is not None]
    assert len(used) == sum(a is not None for a in got) and len(used) > 10
    mean = (sum(float((b * b).sum()) for _, _, b in used) / sum(b.numel() for _, _, b in used)) ** 0.5
    for n, a, b in used:
        assert float((a - b).norm()) <= 1e-4 * max(float(b.norm()), 1e-2 * mean * b.numel() ** 0.5), n
