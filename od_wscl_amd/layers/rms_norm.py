"""Root-mean-square norm over the last axis, with the residual's addition and its gradients, and its 8-bit output
(csrc/rms_norm.hip).  Beside FrozenBatchNorm2d (statistics of maps) and the embeddings' L2 norm (sim_head/sim_net.py): the norm of
activation rows, for heads of one's own between layers.linear.Linear layers.  No reference counterpart."""
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import _lib as L

_BF16 = {torch.float32: 0, torch.bfloat16: 1}


def _rows(t, D):
    """(rows, D) view with dense columns; a copy only where there is none."""
    if t.dim() != 2:
        t = t.reshape(-1, D)
    return t if t.stride(1) == 1 or D == 1 else t.contiguous()


def _check(what, x, weight, residual, eps):
    L.need_gpu(x, weight, residual)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("%s: x has shape %s" % (what, tuple(x.shape)))
    device = x.get_device()
    for name, t in (("x", x), ("weight", weight), ("residual", residual)):
        if t is None:
            continue
        if t.dtype not in _BF16:
            raise TypeError("%s: %s is %s (torch.float32 | torch.bfloat16)" % (what, name, t.dtype))
        if t.get_device() != device:
            raise ValueError("%s: %s is on %s, x on %s" % (what, name, t.device, x.device))
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != x.shape[-1]):
        raise ValueError("%s: weight has shape %s, x %s" % (what, tuple(weight.shape), tuple(x.shape)))
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("%s: residual has shape %s, x %s" % (what, tuple(residual.shape), tuple(x.shape)))
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise TypeError("%s: residual is %s beside x in %s (x's type or torch.float32)" % (what, residual.dtype, x.dtype))
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError("%s: eps = %r" % (what, eps))


def _types(x, residual, weight):
    h = x if residual is None else residual
    return _BF16[x.dtype] + 2 * _BF16[h.dtype] + (4 * _BF16[weight.dtype] if weight is not None else 0)


def _run(what, x, weight, residual, eps, out, rstd=None, scale=None):
    """The forward launch into `out` (y, or with `scale` the 8-bit codes); returns h (None without a residual)."""
    D = x.shape[-1]
    x2 = _rows(x, D)
    r2 = _rows(residual, D) if residual is not None else None
    w = weight.contiguous() if weight is not None else None
    h = residual.new_empty(x.shape) if residual is not None else None
    args = (x2.data_ptr(), x2.stride(0), 0 if r2 is None else r2.data_ptr(), 0 if r2 is None else r2.stride(0), 0 if w is None else w.data_ptr(),
            x2.shape[0], D, eps, out.data_ptr())
    hp, types = 0 if h is None else h.data_ptr(), _types(x, residual, weight)
    if scale is None:
        code = L.lib().odw_rms_norm(*args, hp, 0 if rstd is None else rstd.data_ptr(), types, L.stream())
    else:
        code = L.lib().odw_rms_norm_fp8(*args, scale.data_ptr(), hp, types, L.stream())
    L.check(code, what)
    return h


def _forward(x, weight, residual, eps, want_rstd):
    with L.on_device_of(x):
        y = x.new_empty(x.shape)
        rstd = x.new_empty(x.numel() // x.shape[-1], dtype=torch.float32) if want_rstd else None
        return y, _run("rms_norm", x, weight, residual, eps, y, rstd=rstd), rstd


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _forward(x, weight, residual, eps, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.dtypes = (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        # (once_differentiable's bookkeeping is a third of the host's time here; without create_graph it has nothing to do)
        return _backward_once(ctx, dy, dh) if torch.is_grad_enabled() else _backward(ctx, dy, dh)


def _backward(ctx, dy, dh):
    h, weight, rstd = ctx.saved_tensors
    x_type, h_type = ctx.dtypes
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    if dy is None:                                # only h was used
        return (dh.to(x_type) if need_x and dh is not None else None, torch.zeros_like(weight) if need_w else None, dh if need_r else None, None)
    shape = h.shape
    D = shape[-1]
    h2, g2 = _rows(h, D), _rows(dy, D)
    d2 = _rows(dh, D) if dh is not None else None
    w = weight.contiguous() if weight is not None else None
    R = h2.shape[0]
    lib = L.lib()
    with L.on_device_of(h):
        mixed = h_type is not None and h_type != x_type
        dx = h.new_empty(shape, dtype=x_type) if need_x or (need_r and not mixed) else None
        dres = h.new_empty(shape) if need_r and mixed else None
        dw = w.new_empty(D) if need_w else None
        nbytes = lib.odw_rms_norm_bwd_workspace(R, D) if need_w else 0
        ws = h.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        types = _BF16[x_type] + 2 * _BF16[x_type if h_type is None else h_type] + (4 * _BF16[w.dtype] if w is not None else 0)
        at = [0 if t is None else t.data_ptr() for t in (g2, d2, h2, w, rstd, dx, dres, dw, ws)]
        L.check(lib.odw_rms_norm_bwd(at[0], g2.stride(0), at[1], 0 if d2 is None else d2.stride(0), at[2], h2.stride(0), at[3], at[4], R, D,
                                     at[5], at[6], at[7], types, at[8], nbytes, L.stream()), "rms_norm_bwd")
    return dx if need_x else None, dw, (dres if mixed else dx) if need_r else None, None


_backward_once = once_differentiable(_backward)


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """y = x / sqrt(mean(x^2) + eps) * weight over the last axis; with a residual (y, h): h = x + residual, y the norm of h.

    x (..., D) fp32 or bf16, any row pitch; weight (D,) fp32 or bf16 or None; residual of x's shape, in x's type or fp32 (h has its
    type; it is rounded once, and y is the norm of the rounded h).  Statistics and products are fp32, y is rounded once to x's type.
    Gradients for x, weight and residual: the weight's summed over the rows in fp32, in one order.  h^2 has to fit fp32."""
    _check("rms_norm", x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return _RMSNorm.apply(x, weight, residual, eps)
    y, h, _ = _forward(x, weight, residual, eps, False)
    return y if h is None else (y, h)


@torch.no_grad()
def rms_norm_fp8(x, weight=None, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: (q, scale), or (q, scale, h) with a residual.  q float8_e4m3fn of x's shape, scale fp32 (...,):
    y ~ q.float() * scale[..., None], scale = max |y| / 448 of the row (2^-126 for a row of zeros).  q is the quotient correctly
    rounded (ties to even); in rows over 32768 elements it is rounded to fp32 first.  A row that holds a NaN is all NaN.  No gradients."""
    _check("rms_norm_fp8", x, weight, residual, eps)
    with L.on_device_of(x):
        q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
        scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
        h = _run("rms_norm_fp8", x, weight, residual, eps, q, scale=scale)
    return (q, scale) if h is None else (q, scale, h)


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
