"""A layer whose state decays by one scalar per head and step, out of this package's operators: input projection,
causal conv1d, linear attention, gated group norm, output projection.

``forward`` takes prompts and training batches (and fills a cache), ``step`` one token with that cache, as the Motif
block's forward and step do (mamba_simplemotif.py:241-402).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from ._autograd import differentiated
from .causal_conv1d import causal_conv1d_fn, causal_conv1d_update
from .group_norm import group_norm_fn
from .linear_attention import linear_attention_fn, linear_attention_update


class LinearAttentionBlock(nn.Module):
    """d_model -> d_model with nheads heads of headdim channels and a (d_state, headdim) state each; q and k shared by the
    nheads / n_groups heads of a group. The decay of head h at a token is exp(-exp(A_log_h) dt), dt = softplus of the
    token's own projection; its value enters as v dt."""

    def __init__(self, d_model, nheads, headdim=64, d_state=64, n_groups=1, d_conv=4, eps=1e-5, device=None, dtype=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.nheads, self.headdim, self.d_state, self.n_groups, self.d_conv, self.eps = nheads, headdim, d_state, n_groups, d_conv, eps
        self.d_inner, self.d_qk = nheads * headdim, n_groups * d_state
        self.d_xbc = self.d_inner + 2 * self.d_qk
        self.in_proj = nn.Linear(d_model, self.d_inner + self.d_xbc + nheads, bias=False, **kw)
        self.conv_weight = nn.Parameter(torch.randn(self.d_xbc, d_conv, **kw) * d_conv ** -0.5)
        self.conv_bias = nn.Parameter(torch.zeros(self.d_xbc, **kw))
        # A in 1 .. 16, softplus(dt_bias) between 1e-3 and 1e-1: memories from one token to a thousand.
        self.A_log = nn.Parameter(torch.log(torch.rand(nheads, device=device) * 15 + 1))
        dt = torch.exp(torch.rand(nheads, device=device) * 4.6 - 6.9)
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.norm_weight = nn.Parameter(torch.ones(self.d_inner, device=device))
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=False, **kw)

    def allocate_inference_cache(self, batch_size):
        """(conv_state, state) of an empty text."""
        w = self.conv_weight
        return (torch.zeros(batch_size, self.d_xbc, self.d_conv, device=w.device, dtype=w.dtype),
                torch.zeros(batch_size, self.nheads, self.d_state, self.headdim, device=w.device))

    def _split(self, zxdt):
        return zxdt.split([self.d_inner, self.d_xbc, self.nheads], -1)

    def _operands(self, xbc, dt):
        v, q, k = xbc.split([self.d_inner, self.d_qk, self.d_qk], -1)
        dt = F.softplus(dt.float() + self.dt_bias)
        v = (v.unflatten(-1, (self.nheads, self.headdim)) * dt.unsqueeze(-1)).to(v.dtype)   # dt stays float32: rounded once
        return q.unflatten(-1, (self.n_groups, self.d_state)), k.unflatten(-1, (self.n_groups, self.d_state)), v, -torch.exp(self.A_log) * dt

    def _finish(self, y, z):
        y = group_norm_fn(y.flatten(-2), self.n_groups, self.norm_weight, z=z, eps=self.eps, is_rms_norm=True, norm_before_gate=False)
        return self.out_proj(y)

    def forward(self, hidden, cache=None):
        """hidden: (batch, seqlen, d_model). With a cache (from allocate_inference_cache) the text is taken as its first
        tokens and the cache holds what follows from them afterwards."""
        z, xbc, dt = self._split(self.in_proj(hidden))
        x = xbc.transpose(1, 2).contiguous()
        conv = causal_conv1d_fn(x, self.conv_weight, self.conv_bias, activation="silu").transpose(1, 2).contiguous()
        q, k, v, g = self._operands(conv, dt)
        if cache is None:
            return self._finish(linear_attention_fn(q, k, v, g, scale=1.0), z)
        conv_state, state = cache
        # The cache holds values: it is no part of the graph.
        conv_state.copy_(F.pad(x.detach(), (self.d_conv, 0))[..., x.shape[-1]:])
        y, last = linear_attention_fn(q, k, v, g, scale=1.0, return_last_state=True)
        state.copy_(last.detach())
        return self._finish(y, z)

    def step(self, hidden, cache):
        """hidden: (batch, d_model), one token; the cache is updated in place. Not differentiable: under torch.no_grad()."""
        # Before anything is written.
        if differentiated(hidden, *self.parameters()):
            raise RuntimeError("step has no derivatives: call it under torch.no_grad()")
        conv_state, state = cache
        z, xbc, dt = self._split(self.in_proj(hidden))
        conv = causal_conv1d_update(xbc.contiguous(), conv_state, self.conv_weight, self.conv_bias, activation="silu")
        q, k, v, g = self._operands(conv, dt)
        return self._finish(linear_attention_update(state, q, k, v, g, scale=1.0), z.contiguous())
