"""The gated delta rule token by token in float64 on the CPU, and bounds for what the kernels may differ from it by."""
import torch

NAMES = ("q", "k", "v", "beta", "log_decay", "initial_state")


def recurrence(q, k, v, beta, log_decay, scale, initial_state=None):
    """S' = exp(g_t) S, S = S' + beta_t k_t (v_t - S'^T k_t)^T, o_t = scale S^T q_t; returns (out, last state). q, k (b, L, G, dk)."""
    b, L, H, dv = v.shape
    R = H // q.shape[2]
    q, k = q.repeat_interleave(R, 2), k.repeat_interleave(R, 2)
    g = None if log_decay is None else log_decay.expand(b, L, H)
    s = initial_state if initial_state is not None else q.new_zeros(b, H, q.shape[3], dv)
    outs = []
    for t in range(L):
        if g is not None:
            s = g[:, t].exp()[..., None, None] * s
        z = v[:, t] - (k[:, t].unsqueeze(-1) * s).sum(-2)
        s = s + k[:, t].unsqueeze(-1) * (beta[:, t].unsqueeze(-1) * z).unsqueeze(-2)
        outs.append((q[:, t].unsqueeze(-1) * s).sum(-2))
    out = torch.stack(outs, 1) if outs else v.new_zeros(b, 0, H, dv)
    return out * scale, s


def with_grads(t, scale, dout=None, dlast=None):
    """t: dict of NAMES (log_decay and initial_state may be missing). Outputs and gradients in float64 by autograd through the
    recurrence."""
    leaves = {n: t[n].detach().cpu().double().requires_grad_(True) for n in NAMES if t.get(n) is not None}
    out, last = recurrence(*(leaves.get(n) for n in NAMES[:5]), scale, leaves.get("initial_state"))
    res = {"out": out.detach(), "last_state": last.detach()}
    if dout is not None:
        loss = (out * dout.cpu().double()).sum()
        if dlast is not None:
            loss = loss + (last * dlast.cpu().double()).sum()
        grads = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
        for n, g in zip(leaves, grads):
            res["d" + n] = torch.zeros_like(leaves[n]) if g is None else g
    return res


# Half a unit in the last place of the result's type.
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Tokens of a chunk.
CHUNK = {torch.float32: 32, torch.float16: 32, torch.bfloat16: 64}


def _rows(name, x):
    """x with all elements of one (batch row, head or group) in its last dimension."""
    if name in ("last_state", "dinitial_state"):
        return x.flatten(2)
    if x.dim() == 1:
        return x[None, :, None]
    return x.transpose(1, 2).flatten(2)


def check(got, exact, dtype, dk, L, what, one_key=False):
    """Keys of norm 1 and beta in 0 .. 2 make every transition I - beta k k^T a contraction, and decays at most 1 do not undo that.
    So every entry of P is at most 1, an error in the state grows no more than the state, and the errors of the chunks add up. A
    chunk's value is a sum of dk products with the state and of C with its tokens' corrections, which are such sums themselves;
    each of these, some dk + 2 C in a row, rounds its partial sum once, 2^-24 of at most the (batch row, head)'s largest value m.
    (The planes' 2^-25 of each factor are part of that.) With n chunks: (dk + 2 C) (n + 1) 2^-24 m, and four times that for
    gradients, whose four terms may cancel. That is the most; roundings are as often up as down, so that their root mean square is
    the square root of the number of them: 16 times that bounds the error's norm, with m the results' own root mean square.

    one_key: all tokens have one key, so that every product k . k' is one number with one rounding error e, and the roundings are not
    up as often as down: with beta 2 a chunk's transition along the key, (1 - 2 (1 + e))^C, is off by 2 C e where independent errors
    would give 2 C^(1/2) e. The same chunked sums in float32 on the CPU are off by 2.2e-5 there (130 tokens, dk 64). The norm is then
    held to the count itself, as the elements are."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    g, e = got.detach().cpu().double(), exact.detach().double()
    if not g.numel():
        return
    assert torch.isfinite(g).all(), what
    C = CHUNK[dtype]
    steps = (dk + 2 * C) * (-(-L // C) + 1)
    gr, er = _rows(what, g), _rows(what, e)
    m = er.abs().amax(-1, keepdim=True)
    tol = ROUND[got.dtype] * er.abs() + 4 * steps * 2.0 ** -24 * m + (6e-8 if got.dtype == torch.float16 else 1e-37)
    err = (gr - er).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst error {err[bad].max().item():.3g} " \
                                f"with a bound of {tol[bad].min().item():.3g}"
    if got.dtype == torch.float32:
        rms = er.square().mean().sqrt() + 1e-37
        assert (gr - er).square().mean().sqrt() <= (4 * steps if one_key else 16 * steps ** 0.5) * 2.0 ** -24 * rms, (what, ((gr - er).square().mean().sqrt() / rms).item())
