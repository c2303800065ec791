"""Linear attention with one decay for each head, on the gfx950 kernels of mm_linattn.hip.

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        S: (dk, dv) for each batch row and head, float32
    o_t = scale * S_t^T q_t

* ``linear_attention_fn`` -- whole sequences (prompts, training), chunked, differentiable in q, k, v,
  log_decay and initial_state, with the gradient of the returned last state;
* ``linear_attention_update`` -- one token on a kept state, which is updated in place.

q and k are shared by the heads of a group, as B and C are in ``selective_scan_fn``: a layer whose state
decays by ``exp(dt_t A_h)`` (the state-space dual of the scan) passes ``q=C, k=B, v=x * dt``,
``log_decay=dt * A`` and ``scale=1``; retention passes a constant ``log_decay`` of shape (nheads,).
float32, float16 and bfloat16; log_decay may have a dtype of its own (float32 is advised: a decay's
error is raised to the power of its memory). Sums, scores and states are float32 from end to end; 16-bit
outputs are rounded once. log_decay is meant to be at most 0; -inf forgets the state, so a packed batch
marks each document's first token with it (below -128 counts as that, above 128 as an infinite growth).
Infinite inputs give the outputs and states of the recurrence, slowly.

dk and dv up to 128 (else NotImplementedError).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._autograd import differentiated
from ._native import ext


# The kernels address 64 tokens of a tensor with 32 bits.
_SEQ_STRIDE = 1 << 22


def _rows(t):
    """t with contiguous rows, and tokens less than 2^22 elements apart; copied where it is not so."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return t.contiguous()
    return t.contiguous() if t.dim() == 4 and t.shape[1] > 1 and t.stride(1) >= _SEQ_STRIDE else t


def _spread(log_decay, lead, v):
    """log_decay as (*lead, nheads), and whether it is one value per head."""
    heads = v.shape[-2]
    per_head = log_decay.dim() == 1
    if per_head and log_decay.shape[0] != heads:
        raise ValueError(f"log_decay must have shape (nheads,) = ({heads},) or {(*lead, heads)}")
    return log_decay.expand(*lead, heads) if per_head else log_decay, per_head


def _scale(scale, q):
    return q.shape[-1] ** -0.5 if scale is None else float(scale)


def _forward(q, k, v, log_decay, scale, initial_state, return_last_state, keep_states=False):
    q, k, v = _rows(q), _rows(k), _rows(v)
    g, per_head = _spread(log_decay, v.shape[:2], v)
    res = ext().linattn_fwd(q, k, v, g, scale, initial_state, return_last_state, keep_states)
    states = res.pop() if keep_states else None
    return q, k, v, per_head, states, tuple(res) if return_last_state else res[0]


class LinearAttentionFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, return_last_state):
        # Long rows of few heads run in segments; the states those start from serve the backward too.
        q, k, v, ctx.per_head, states, out = _forward(q, k, v, log_decay, scale, initial_state, return_last_state, True)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, states)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast=None):
        q, k, v, log_decay, initial_state, states = ctx.saved_tensors
        if dout is None:
            if dlast is None:
                return None, None, None, None, None, None, None
            dout = torch.zeros_like(v, memory_format=torch.contiguous_format)
        g, _ = _spread(log_decay, v.shape[:2], v)
        want = ctx.needs_input_grad
        dq, dk, dv, dg, ds = ext().linattn_bwd(q, k, v, g, ctx.scale, initial_state, _rows(dout), dlast, states, ctx.per_head, want[3],
                                               want[5] and initial_state is not None)
        return dq, dk, dv, dg, None, ds, None


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, return_last_state=False):
    """q, k: (batch, seqlen, n_groups, dk); v: (batch, seqlen, nheads, dv), nheads a multiple of n_groups;
    log_decay: (batch, seqlen, nheads) or (nheads,); initial_state: (batch, nheads, dk, dv) float32 or None
    (zeros); scale: None for dk ** -0.5. Returns out (batch, seqlen, nheads, dv) in v's dtype [, last_state
    (batch, nheads, dk, dv) float32, the state linear_attention_update continues from]."""
    if v.dim() != 4:
        raise ValueError("v must have shape (batch, seqlen, nheads, dv)")
    args = (q, k, v, log_decay, _scale(scale, q), initial_state, return_last_state)
    if differentiated(q, k, v, log_decay, initial_state):
        return LinearAttentionFn.apply(*args)
    return _forward(*args)[5]


def linear_attention_update(state, q, k, v, log_decay, scale=None):
    """One token. state: (batch, nheads, dk, dv) float32, updated in place (its last dimension contiguous);
    q, k: (batch, n_groups, dk); v: (batch, nheads, dv); log_decay: (batch, nheads) or (nheads,). Returns
    out (batch, nheads, dv) in v's dtype. Calls on one state must be ordered. No derivatives: inputs that require a gradient are
    refused in grad mode, and the state's version counts the update, so that a backward which needs what stood there raises."""
    if v.dim() != 3:
        raise ValueError("v must have shape (batch, nheads, dv)")
    g, _ = _spread(log_decay, v.shape[:1], v)
    return ext().linattn_update(state, _rows(q), _rows(k), _rows(v), g, _scale(scale, q))
