"""Residual add with layer norm or RMS norm, channels last, on the gfx950 kernels of mm_layer_norm.hip: the norm at the entry of a
layer, as the reference's blocks call it (mamba_ssm.ops.triton.layer_norm: layer_norm_fn, rms_norm_fn, RMSNorm; mixer_seq_simple.py:24,
190-212).

    h = x + residual                          float32
    y = (h - mean) / sqrt(var + eps) * weight + bias           RMS norm: h / sqrt(mean(h^2) + eps) * weight + bias

``prenorm=True`` also returns h, the residual that the next layer adds to, in the residual's dtype. The norm is that of h itself, not
of its rounded copy. Statistics and sums are float32, results are rounded once.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from ._autograd import differentiated
from ._native import ext
from .group_norm import _flat


def _forward(x, weight, bias, residual, eps, prenorm, wide, is_rms_norm):
    xf, rf = _flat(x), None if residual is None else _flat(residual)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    out, res = ext().layer_norm_fwd(xf, rf, weight, bias, eps, is_rms_norm, prenorm, wide)
    if x.dim() != 2:
        out = out.view(x.shape)
    return xf, rf, weight, bias, res, out if not prenorm else (out, res if x.dim() == 2 else res.view(x.shape))


class LayerNormFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, prenorm, wide, is_rms_norm):
        xf, rf, weight, bias, res, out = _forward(x, weight, bias, residual, eps, prenorm, wide, is_rms_norm)
        ctx.args = (eps, is_rms_norm)
        ctx.has_residual = residual is not None
        ctx.wide = (residual.dtype if residual is not None else torch.float32 if wide else x.dtype) == torch.float32
        ctx.set_materialize_grads(False)
        # A float32 residual_out is h itself; it lives on as the next layer's input, so that x and residual need not.
        ctx.kept = rf is not None and res is not None and res.dtype == torch.float32
        ctx.dtype = x.dtype
        ctx.save_for_backward(*((None, res) if ctx.kept else (xf, rf)), weight, bias)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dres=None):
        x, residual, weight, bias = ctx.saved_tensors
        if dout is None and dres is None:
            return (None,) * 8
        shape = (dres if dout is None else dout).shape
        if dout is None:
            dout = torch.zeros(shape, device=dres.device, dtype=ctx.dtype)
        eps, is_rms_norm = ctx.args
        want = ctx.needs_input_grad
        # With one dtype the two gradients are one tensor.
        one = not ctx.wide or ctx.dtype == torch.float32
        want_dx = want[0] or (one and want[3])
        dx, dr, dw, db = ext().layer_norm_bwd(x, residual, weight, bias, eps, is_rms_norm, _flat(dout), None if dres is None else _flat(dres),
                                              ctx.wide, want_dx, ctx.has_residual and want[3] and not one, want[1], want[2])
        dx = None if dx is None else dx.view(shape)
        dr = (dx if one else None if dr is None else dr.view(shape)) if ctx.has_residual else None
        return dx, dw, db, dr, None, None, None, None


def layer_norm_fn(x, weight, bias=None, residual=None, eps=1e-6, prenorm=False, residual_in_fp32=False, is_rms_norm=False):
    """x: (..., channels); weight, bias: (channels,) or None; residual: like x, of x's dtype or float32, or None. Returns y in x's
    dtype, with prenorm (y, residual_out): residual_out has residual's dtype, without a residual x's, or float32 with
    residual_in_fp32. Differentiable in x, weight, bias and residual."""
    if x.dim() < 1 or (residual is not None and residual.shape != x.shape):
        raise ValueError("x must be (..., channels), and residual must have its shape")
    args = (x, weight, bias, residual, float(eps), bool(prenorm), bool(residual_in_fp32), bool(is_rms_norm))
    if differentiated(x, weight, bias, residual):
        return LayerNormFn.apply(*args)
    return _forward(*args)[5]


def rms_norm_fn(x, weight, bias=None, residual=None, eps=1e-6, prenorm=False, residual_in_fp32=False):
    """layer_norm_fn without the mean."""
    return layer_norm_fn(x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm=True)


class RMSNorm(nn.Module):
    def __init__(self, hidden_size, eps=1e-5, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        self.register_parameter("bias", None)

    def forward(self, x, residual=None, prenorm=False, residual_in_fp32=False):
        return rms_norm_fn(x, self.weight, self.bias, residual, self.eps, prenorm, residual_in_fp32)
