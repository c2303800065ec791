"""A layer with the gated delta rule out of this package's operators: residual add and RMS norm, input projection, causal conv1d, norm
of q and k, delta rule, gated group norm, output projection.

``forward`` takes prompts and training batches (and fills a cache), ``step`` one token with that cache; both take and hand on the
residual stream, as the reference's blocks do (mixer_seq_simple.py:190-212).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from ._autograd import differentiated
from .causal_conv1d import causal_conv1d_fn, causal_conv1d_update
from .delta_rule import delta_rule_fn, delta_rule_update
from .group_norm import group_norm_fn
from .layer_norm import RMSNorm


class GatedDeltaBlock(nn.Module):
    """d_model -> d_model with nheads heads of headdim channels and a (d_state, headdim) state each; q and k, normed to length 1, are
    shared by the nheads / n_groups heads of a group. beta is the sigmoid of the token's own projection, the decay of head h
    exp(-exp(A_log_h) dt), dt the softplus of another."""

    def __init__(self, d_model, nheads, headdim=64, d_state=64, n_groups=1, d_conv=4, eps=1e-5, residual_in_fp32=True, device=None, dtype=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.nheads, self.headdim, self.d_state, self.n_groups, self.d_conv, self.eps = nheads, headdim, d_state, n_groups, d_conv, eps
        self.residual_in_fp32 = residual_in_fp32
        self.d_inner, self.d_qk = nheads * headdim, n_groups * d_state
        self.d_qkv = self.d_inner + 2 * self.d_qk
        self.norm = RMSNorm(d_model, eps=eps, device=device)
        self.in_proj = nn.Linear(d_model, self.d_inner + self.d_qkv + 2 * nheads, bias=False, **kw)
        self.conv_weight = nn.Parameter(torch.randn(self.d_qkv, d_conv, **kw) * d_conv ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(self.d_qkv, **kw))
        # A in 1 .. 16, softplus(dt_bias) between 1e-3 and 1e-1: memories from one token to a thousand.
        self.A_log = nn.Parameter(torch.log(torch.rand(nheads, device=device) * 15 + 1))
        dt = torch.exp(torch.rand(nheads, device=device) * 4.6 - 6.9)
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        # x / |x| is RMS norm times d_state ** -0.5.
        self.register_buffer("qk_weight", torch.full((self.d_qk,), d_state ** -0.5, device=device), persistent=False)
        self.norm_weight = nn.Parameter(torch.ones(self.d_inner, device=device))
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=False, **kw)

    def allocate_inference_cache(self, batch_size):
        """(conv_state, state) of an empty text."""
        w = self.conv_weight
        return (torch.zeros(batch_size, self.d_qkv, self.d_conv, device=w.device, dtype=w.dtype),
                torch.zeros(batch_size, self.nheads, self.d_state, self.headdim, device=w.device, dtype=torch.float32))

    def _enter(self, hidden, residual):
        x, residual = self.norm(hidden, residual, prenorm=True, residual_in_fp32=self.residual_in_fp32)
        return self.in_proj(x).split([self.d_inner, self.d_qkv, self.nheads, self.nheads], -1), residual

    def _operands(self, qkv, b, a):
        v, q, k = qkv.split([self.d_inner, self.d_qk, self.d_qk], -1)
        q, k = (group_norm_fn(x, self.n_groups, self.qk_weight, eps=1e-6 / self.d_state, is_rms_norm=True) for x in (q, k))
        g = -torch.exp(self.A_log) * F.softplus(a.float() + self.dt_bias)
        return (q.unflatten(-1, (self.n_groups, self.d_state)), k.unflatten(-1, (self.n_groups, self.d_state)),
                v.unflatten(-1, (self.nheads, self.headdim)), torch.sigmoid(b.float()), g)

    def _finish(self, y, z):
        y = group_norm_fn(y.flatten(-2), self.nheads, self.norm_weight, z=z, eps=self.eps, is_rms_norm=True)
        return self.out_proj(y)

    def forward(self, hidden, residual=None, cache=None):
        """hidden: (batch, seqlen, d_model); residual: like it (float32 with residual_in_fp32) or None. Returns (out, residual), out
        not yet added to it. With a cache (from allocate_inference_cache) the text is taken as its first tokens and the cache holds
        what follows from them afterwards."""
        (z, qkv, b, a), residual = self._enter(hidden, residual)
        x = qkv.transpose(1, 2).contiguous()
        conv = causal_conv1d_fn(x, self.conv_weight, self.conv_bias, activation="silu").transpose(1, 2).contiguous()
        args = self._operands(conv, b, a)
        if cache is None:
            return self._finish(delta_rule_fn(*args), z), residual
        conv_state, state = cache
        # The cache holds values: it is no part of the graph.
        conv_state.copy_(F.pad(x.detach(), (self.d_conv, 0))[..., x.shape[-1]:])
        y, last = delta_rule_fn(*args, return_last_state=True)
        state.copy_(last.detach())
        return self._finish(y, z), residual

    def step(self, hidden, residual, cache):
        """hidden, residual: (batch, d_model), one token; the cache is updated in place. Not differentiable: under torch.no_grad()."""
        # Before anything is written.
        if differentiated(hidden, residual, *self.parameters()):
            raise RuntimeError("step has no derivatives: call it under torch.no_grad()")
        conv_state, state = cache
        (z, qkv, b, a), residual = self._enter(hidden, residual)
        conv = causal_conv1d_update(qkv.contiguous(), conv_state, self.conv_weight, self.conv_bias, activation="silu")
        return self._finish(delta_rule_update(state, *self._operands(conv, b, a)), z.contiguous()), residual
