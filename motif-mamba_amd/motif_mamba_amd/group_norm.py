"""Group norm of each token's channel groups with a gate or an activation, channels last, on the gfx950
kernels of mm_group_norm.hip: the norm behind a linear-attention or state-space layer.

The statistics run over one token's group of channels / n_groups channels; a causal model cannot take them
over tokens. ``is_rms_norm`` leaves the mean out. ``z`` gates with silu(z), behind the norm
(``norm_before_gate=True``, retention) or in front of it (False, the state-space duals). Without z,
``activation`` "silu" (or "swish") applies to the result. Statistics and sums are float32.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._autograd import differentiated
from ._native import ext

_NONE, _AFTER, _BEFORE, _ACT = 0, 1, 2, 3


def _flat(t):
    """(rows, channels), a view where there is one."""
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    t = t.reshape(-1, t.shape[-1]) if t.shape[-1] else t.reshape(t[..., 0:0].numel(), 0)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _forward(x, n_groups, weight, bias, z, eps, is_rms_norm, gate):
    xf, zf = _flat(x), None if z is None else _flat(z)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    out = ext().group_norm_fwd(xf, n_groups, weight, bias, zf, eps, is_rms_norm, gate)
    return xf, weight, bias, zf, out.view(x.shape)


class GroupNormFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, n_groups, weight, bias, z, eps, is_rms_norm, gate):
        xf, weight, bias, zf, out = _forward(x, n_groups, weight, bias, z, eps, is_rms_norm, gate)
        ctx.args = (n_groups, eps, is_rms_norm, gate)
        ctx.save_for_backward(xf, weight, bias, zf)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, bias, z = ctx.saved_tensors
        n_groups, eps, is_rms_norm, gate = ctx.args
        want = ctx.needs_input_grad
        dx, dw, db, dz = ext().group_norm_bwd(x, n_groups, weight, bias, z, eps, is_rms_norm, gate, _flat(dout),
                                              want[2] or want[3])
        shape = dout.shape
        return dx.view(shape), None, dw, db, None if dz is None else dz.view(shape), None, None, None


def group_norm_fn(x, n_groups, weight=None, bias=None, z=None, eps=1e-5, activation=None, is_rms_norm=False,
                  norm_before_gate=True):
    """x: (..., channels), channels a multiple of n_groups; weight, bias: (channels,) or None; z: like x or
    None. Returns y in x's shape and dtype, contiguous. Differentiable in x, weight, bias and z."""
    if activation not in (None, "silu", "swish"):
        raise NotImplementedError("activation must be None, silu, or swish")
    if z is not None and activation is not None:
        raise ValueError("activation applies without z; a z gates with silu(z)")
    if x.dim() < 1 or (z is not None and z.shape != x.shape):
        raise ValueError("x must be (..., channels), and z must have its shape")
    gate = (_AFTER if norm_before_gate else _BEFORE) if z is not None else _ACT if activation else _NONE
    args = (x, int(n_groups), weight, bias, z, float(eps), bool(is_rms_norm), gate)
    if differentiated(x, weight, bias, z):
        return GroupNormFn.apply(*args)
    return _forward(*args)[4]
