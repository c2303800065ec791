"""The gated delta rule, on the gfx950 kernels of mm_delta.hip: a state that is corrected under a key as well as decayed.

    S'_t = exp(log_decay_t) S_{t-1}                        S: (dk, dv) for each batch row and head, float32
    S_t  = S'_t + beta_t k_t (v_t - S'_t^T k_t)^T
    o_t  = scale * S_t^T q_t

* ``delta_rule_fn`` -- whole sequences (prompts, training), chunked, differentiable in q, k, v, beta, log_decay and initial_state,
  with the gradient of the returned last state;
* ``delta_rule_update`` -- one token on a kept state, which is updated in place.

Without the correction (S'_t^T k_t left out) and with beta folded into v this is ``linear_attention_fn``. q and k are shared by the
heads of a group, as there. Keys are meant to have norm 1 (``group_norm_fn`` with ``is_rms_norm``, a weight of dk ** -0.5 and one
group per head gives it) and beta to lie between 0 and 2. Without log_decay nothing decays.
float32, float16 and bfloat16; beta and log_decay may have dtypes of their own (float32 is advised: a decay's error is raised to the
power of its memory). Sums, scores and states are float32 from end to end; 16-bit outputs are rounded once. log_decay is meant to be
at most 0; -inf forgets the state, so a packed batch marks each document's first token with it (below -128 counts as that, above 128
as an infinite growth). Infinities and NaN in the inputs give the outputs and states of the recurrence, slowly; in the gradients of
its (batch row, head) what one reaches is NaN or infinite, and other elements may be NaN.

dk and dv up to 128 (else NotImplementedError).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._autograd import differentiated
from ._native import ext
from .linear_attention import _rows, _scale, _spread


def _decays(log_decay, lead, v):
    return (None, False) if log_decay is None else _spread(log_decay, lead, v)


def _forward(q, k, v, beta, log_decay, scale, initial_state, return_last_state, keep_states=False):
    q, k, v = _rows(q), _rows(k), _rows(v)
    g, per_head = _decays(log_decay, v.shape[:2], v)
    res = ext().delta_fwd(q, k, v, beta, g, scale, initial_state, return_last_state, keep_states)
    states = res.pop() if keep_states else None
    return q, k, v, per_head, states, tuple(res) if return_last_state else res[0]


class DeltaRuleFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, beta, log_decay, scale, initial_state, return_last_state):
        # Long rows of few heads run in segments; the states those start from, and what each makes of a state, serve the backward too.
        q, k, v, ctx.per_head, states, out = _forward(q, k, v, beta, log_decay, scale, initial_state, return_last_state, True)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, beta, log_decay, initial_state, states)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast=None):
        q, k, v, beta, log_decay, initial_state, states = ctx.saved_tensors
        if dout is None:
            if dlast is None:
                return (None,) * 8
            dout = torch.zeros_like(v, memory_format=torch.contiguous_format)
        g, _ = _decays(log_decay, v.shape[:2], v)
        want = ctx.needs_input_grad
        dq, dk, dv, db, dg, ds = ext().delta_bwd(q, k, v, beta, g, ctx.scale, initial_state, _rows(dout), dlast, states, ctx.per_head, want[4],
                                                 want[6] and initial_state is not None)
        return dq, dk, dv, db, dg, None, ds, None


def delta_rule_fn(q, k, v, beta, log_decay=None, scale=None, initial_state=None, return_last_state=False):
    """q, k: (batch, seqlen, n_groups, dk); v: (batch, seqlen, nheads, dv), nheads a multiple of n_groups; beta: (batch, seqlen,
    nheads); log_decay: (batch, seqlen, nheads), (nheads,) or None; initial_state: (batch, nheads, dk, dv) float32 or None (zeros);
    scale: None for dk ** -0.5. Returns out (batch, seqlen, nheads, dv) in v's dtype [, last_state (batch, nheads, dk, dv) float32,
    the state delta_rule_update continues from]."""
    if v.dim() != 4:
        raise ValueError("v must have shape (batch, seqlen, nheads, dv)")
    args = (q, k, v, beta, log_decay, _scale(scale, q), initial_state, return_last_state)
    if differentiated(q, k, v, beta, log_decay, initial_state):
        return DeltaRuleFn.apply(*args)
    return _forward(*args)[5]


def delta_rule_update(state, q, k, v, beta, log_decay=None, scale=None):
    """One token. state: (batch, nheads, dk, dv) float32, updated in place (its last dimension contiguous); q, k: (batch, n_groups,
    dk); v: (batch, nheads, dv); beta: (batch, nheads); log_decay: (batch, nheads), (nheads,) or None. Returns out (batch, nheads, dv)
    in v's dtype. Calls on one state must be ordered. No derivatives: inputs that require a gradient are refused in grad mode, and
    the state's version counts the update, so that a backward which needs what stood there raises."""
    if v.dim() != 3:
        raise ValueError("v must have shape (batch, nheads, dv)")
    g, _ = _decays(log_decay, v.shape[:1], v)
    return ext().delta_update(state, _rows(q), _rows(k), _rows(v), beta, g, _scale(scale, q))
