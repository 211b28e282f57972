"""Root-mean-square norm as a module: the norm='rmsnorm' choice of the encoders, in place of nn.LayerNorm."""
import torch
import torch.nn as nn

from ... import ops


class RMSNorm(nn.Module):
    """y = x * (mean(x^2) + eps)^-1/2 * weight over the last dimension (ops.rms_norm).  forward(x, residual=None, kind=None): with
    a residual the result is (y, x + residual); kind: rows of a padded batch, padding rows come out as zeros"""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None, kind=None):
        return ops.rms_norm(x, self.weight, residual, eps=self.eps, kind=kind)

    def extra_repr(self):
        return f'{self.dim}, eps={self.eps}'
