"""Linear attention with one decay for each head, token by token in float64 on the CPU, and bounds for what the
kernels may differ from it by."""
import torch


def recurrence(q, k, v, log_decay, scale, initial_state=None):
    """S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t; returns (out, last state). q, k (b, L, G, dk)."""
    b, L, H, dv = v.shape
    R = H // q.shape[2]
    q, k = q.repeat_interleave(R, 2), k.repeat_interleave(R, 2)
    g = log_decay.expand(b, L, H)
    s = initial_state if initial_state is not None else q.new_zeros(b, H, q.shape[3], dv)
    outs = []
    for t in range(L):
        s = g[:, t].exp()[..., None, None] * s + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        outs.append((q[:, t].unsqueeze(-1) * s).sum(-2))
    out = torch.stack(outs, 1) if outs else v.new_zeros(b, 0, H, dv)
    return out * scale, s


NAMES = ("q", "k", "v", "log_decay", "initial_state")


def with_grads(t, scale, dout=None, dlast=None):
    """t: dict of q, k, v, log_decay and maybe initial_state. Outputs and gradients in float64 by autograd through
    the recurrence."""
    leaves = {n: t[n].detach().cpu().double().requires_grad_(True) for n in NAMES if t.get(n) is not None}
    out, last = recurrence(leaves["q"], leaves["k"], leaves["v"], leaves["log_decay"], scale, leaves.get("initial_state"))
    res = {"out": out.detach(), "last_state": last.detach()}
    if dout is not None:
        loss = (out * dout.cpu().double()).sum()
        if dlast is not None:
            loss = loss + (last * dlast.cpu().double()).sum()
        grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
        for n, g in zip(leaves, grads):
            res["d" + n] = torch.zeros_like(leaves[n]) if g is None else g
    return res


def magnitudes(t, scale, dout=None, dlast=None):
    """The sums of the absolute values of all terms of every output: a product of the absolute inputs is the same
    sum without its signs. Rounding errors are fractions of these."""
    a = {n: (x if n == "log_decay" else x.abs()) for n, x in t.items() if x is not None}
    return with_grads(a, abs(scale), None if dout is None else dout.abs(), None if dlast is None else dlast.abs())


# Half a unit in the last place of the result's type.
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# What the terms themselves carry. 16-bit inputs: state, scores and gradients in two bfloat16 planes are within
# 2^-17 of their value, at most four such factors and the float32 sums stand behind one term (2^-15). float32
# inputs: 2^-24 per operation, sums over 32 x 4 tokens or columns and a few dozen chunk steps deep: 2^-24 * 64.
TERM = {torch.float32: 2.0 ** -18, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -15}


def check(got, exact, size, dtype, what, whole_row=False):
    """|got - exact| within half a unit of got's type plus a fraction of the terms' magnitudes (whole_row: of the
    largest along the sequence: a decay's gradient is corrected by sums over its neighbours')."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    g, e = got.detach().cpu().double(), exact.double()
    if whole_row and size.dim() == 3 and size.numel():
        size = size.amax(1, keepdim=True).expand_as(size)
    tol = ROUND[got.dtype] * e.abs() + TERM[dtype] * size + (6e-8 if got.dtype == torch.float16 else 1e-37)
    err = (g - e).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst error {err[bad].max().item():.3g} " \
                                f"with a bound of {tol[bad].min().item():.3g}"
