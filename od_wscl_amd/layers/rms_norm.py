"""Root-mean-square norm over the last axis, with the residual's addition and its gradients, and its 8-bit output
(csrc/rms_norm.hip; the autograd node: csrc/bind.cpp).  Beside FrozenBatchNorm2d (statistics of maps) and the embeddings' L2 norm
(sim_head/sim_net.py): the norm of activation rows, for heads of one's own between layers.linear.Linear layers.  No reference counterpart."""
import torch
from torch import nn

from .. import _lib as L


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last axis; with a residual (y, h): h = x + residual, y the norm of h.

    x (..., D) fp32 or bf16, any row pitch; weight (D,) fp32 or bf16 or None; residual of x's shape, in x's type or fp32 (h has its
    type; it is rounded once, and y is the norm of the rounded h).  Statistics and products are fp32, y is rounded once to x's type.
    Gradients for x, weight and residual: the weight's summed over the rows in fp32, in one order; no second and no forward-mode
    derivatives (refused).  h^2 has to fit fp32.  A backward pass can be captured into a HIP graph; where a graph made on the default
    stream before still holds a node that it would reach, that is refused."""
    return L.bind().rms_norm(x, weight, residual, eps)


def rms_norm_fp8(x, weight=None, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: (q, scale), or (q, scale, h) with a residual.  q float8_e4m3fn of x's shape, scale fp32 (...,):
    y ~ q.float() * scale[..., None], scale = max |y| / 448 of the row (2^-126 for a row of zeros).  q is the quotient correctly
    rounded (ties to even); it is rounded to fp32 first in rows over 32768 elements, in rows whose largest |h weight| is not between
    1e-30 and 1e30, and where 2^-126 is the scale.  A row that holds a NaN is all NaN.  No gradients."""
    return L.bind().rms_norm_fp8(x, weight, residual, eps)


class RMSNorm(nn.Module):
    """rms_norm with a gain of its own (ones): forward(x) -> y, forward(x, residual) -> (y, x + residual)."""

    def __init__(self, dim, eps=1e-6, elementwise_affine=True):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim)) if elementwise_affine else None
        self.dim = dim

    def forward(self, x, residual=None):
        if x.shape[-1] != self.dim:
            raise ValueError("RMSNorm: x has %d columns, the norm %d" % (x.shape[-1], self.dim))
        return rms_norm(x, self.weight, residual, self.eps)

    def extra_repr(self):
        return "%d, eps=%g" % (self.dim, self.eps)
