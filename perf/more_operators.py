"""The operators of a layer whose state is corrected as well as decayed, as measurable cases: the gated delta rule (prompts,
training steps, single tokens) and the residual add with the norm at the layer's entry, forward and backward.

``own`` False runs the plain form, elementary torch operations in float32; True makes the calls a user makes. Both take what
``prepare`` returns.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _mm():
    path = os.path.join(os.getcwd(), "motif-mamba_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import motif_mamba_amd
    return motif_mamba_amd


def listed():
    return [
        # One token of one sequence through a 5,120-channel layer of 40 heads, two heads to a key: a chat at batch 1; latency.
        dict(name="token_b1", kind="token", batch=1, heads=40, groups=20, dk=128, dv=128, decay="token", beta=1, dtype="bf16"),
        # The same step for a full serving batch: the states' memory traffic.
        dict(name="token_b256", kind="token", batch=256, heads=40, groups=20, dk=128, dv=128, decay="token", beta=1,
             dtype="bf16"),
        # Two prompts of an odd length through a 1,536-channel layer, q, k and v slices of one projection.
        dict(name="prompt_odd", kind="prompt", batch=2, L=1777, heads=24, groups=24, dk=64, dv=64, decay="token", beta=1,
             layout="fused", states=False, dtype="bf16"),
        # The prompt pass of a 5,120-channel layer, two heads to a key.
        dict(name="prompt_wide", kind="prompt", batch=4, L=4096, heads=40, groups=20, dk=128, dv=128, decay="token", beta=1,
             layout="fused", states=False, dtype="bf16"),
        # A long document in float32, continued from the state of what came before, reflections allowed (beta up to 2).
        dict(name="prompt_long_fp32", kind="prompt", batch=1, L=32768, heads=24, groups=8, dk=64, dv=64, decay="token", beta=2,
             layout="dense", states=True, dtype="fp32"),
        # A training step of a 1,536-channel layer, keys of each head's own.
        dict(name="train_heads", kind="train", batch=8, L=2048, heads=24, groups=24, dk=64, dv=64, decay="token", beta=1,
             layout="fused", states=False, dtype="bf16"),
        # A training step with wide states, keys shared by four heads (their gradients sum over those).
        dict(name="train_shared", kind="train", batch=4, L=4096, heads=16, groups=4, dk=128, dv=128, decay="token", beta=1,
             layout="dense", states=False, dtype="bf16"),
        # A training step on a piece of a longer text: state taken in and handed on, with both gradients; no decay.
        dict(name="train_states_fp16", kind="train", batch=4, L=1000, heads=32, groups=8, dk=64, dv=64, decay="none", beta=1,
             layout="dense", states=True, dtype="fp16"),
        # The add and norm of 64 sequences' single tokens at a 2,560-channel layer's entry, float32 residual stream; latency.
        dict(name="norm_token", kind="norm", rows=64, channels=2560, rms=True, bias=False, residual="fp32", prenorm=True,
             dtype="bf16"),
        # The same of a prompt.
        dict(name="norm_prompt", kind="norm", rows=16384, channels=2560, rms=True, bias=False, residual="fp32", prenorm=True,
             dtype="bf16"),
        # Forward and backward of a training step's.
        dict(name="norm_train", kind="norm_train", rows=16384, channels=2560, rms=True, bias=False, residual="fp32",
             prenorm=True, dtype="bf16"),
        # Forward and backward of a layer norm without a residual, odd size, float32.
        dict(name="norm_train_odd", kind="norm_train", rows=5331, channels=1001, rms=False, bias=True, residual="none",
             prenorm=False, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["token", "prompt", "prompt", "train", "train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("norm"):
        c = dict(kind=kind, rows=_log_int(rng, 1, 16384), channels=_log_int(rng, 64, 5120), rms=rng.random() < 0.5,
                 bias=rng.random() < 0.5, residual=rng.choice(["none", "fp32", "fp32", dtype]), prenorm=rng.random() < 0.6,
                 dtype=dtype)
        if rng.random() < 0.6:
            c["channels"] = max(64, c["channels"] // 64 * 64)
        while c["rows"] * c["channels"] > 16384 * 2560 // (2 if dtype == "fp32" else 1):
            c["rows"] = (c["rows"] + 1) // 2
        return c
    groups = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, batch=_log_int(rng, 1, 8), L=_log_int(rng, 2, 8192), heads=groups * rng.choice([1, 2, 3, 5]), groups=groups,
             dk=rng.choice([16, 32, 40, 64, 64, 96, 128]), dv=rng.choice([32, 48, 64, 64, 80, 128]),
             decay=rng.choice(["token", "token", "fixed", "none"]), beta=rng.choice([1, 1, 2]), dtype=dtype)
    if kind == "token":
        c["batch"] = _log_int(rng, 1, 256)
        del c["L"]
        return c
    c.update(layout=rng.choice(["fused", "dense"]), states=rng.random() < 0.4)
    if kind == "prompt" and rng.random() < 0.15:
        c["batch"], c["L"] = 1, _log_int(rng, 8192, 32768)
    most = {"prompt": 4 * 4096 * 40 * 128 * 128, "train": 4 * 4096 * 16 * 128 * 128 // 2}[kind]
    while c["batch"] * c["L"] * c["heads"] * c["dk"] * c["dv"] * (4 if dtype == "fp32" else 1) > most:
        if c["batch"] > 1:
            c["batch"] = (c["batch"] + 1) // 2
        else:
            c["L"] = c["L"] * 2 // 3
    return c


# ---- inputs --------------------------------------------------------------------------------------


class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def n(self, *shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=self.g) * scale

    def u(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=self.g) * (hi - lo) + lo


def _log_decay(c, r, *lead):
    h = c["heads"]
    if c["decay"] == "fixed":
        # Half-lives spread over the heads, from some 20 tokens to thousands.
        return torch.log1p(-torch.exp2(-5.0 - 8.0 * torch.arange(h, device="cuda", dtype=torch.float32) / max(1, h)))
    # -A softplus(dt + bias): A in 1 .. 16 by head, softplus(bias) between 1e-3 and 1e-1.
    dt = torch.exp(r.u(h, lo=math.log(1e-3), hi=math.log(1e-1)))
    bias = dt + torch.log(-torch.expm1(-dt))
    return -torch.log1p(torch.exp(r.n(*lead, h, scale=0.5) + bias)) * r.u(h, lo=1.0, hi=16.0)


def _delta_inputs(c, r):
    b, h, g, dk, dv = c["batch"], c["heads"], c["groups"], c["dk"], c["dv"]
    dt = DTYPES[c["dtype"]]
    lead = (b,) if c["kind"] == "token" else (b, c["L"])
    # Keys and queries come with norm 1, as a layer hands them on.
    q, k = (r.n(*lead, g, dk) for _ in range(2))
    q, k = (x / (x * x).sum(-1, keepdim=True).sqrt() for x in (q, k))
    if c.get("layout") == "fused":
        qkv = torch.cat([q.flatten(-2), k.flatten(-2), r.n(*lead, h * dv)], -1).to(dt)
        q, k, v = qkv.split([g * dk, g * dk, h * dv], -1)
        t = dict(q=q.unflatten(-1, (g, dk)), k=k.unflatten(-1, (g, dk)), v=v.unflatten(-1, (h, dv)))
    else:
        t = dict(q=q.to(dt), k=k.to(dt), v=r.n(*lead, h, dv).to(dt))
    t["beta"] = c["beta"] / (1.0 + torch.exp(-r.n(*lead, h)))
    if c["decay"] != "none":
        t["log_decay"] = _log_decay(c, r, *lead)
    if c["kind"] == "token":
        t["state"] = r.n(b, h, dk, dv)
    elif c["states"]:
        t["initial_state"] = r.n(b, h, dk, dv)
    if c["kind"] == "train":
        t["dout"] = r.n(*lead, h, dv).to(dt)
        if c["states"]:
            t["dlast"] = r.n(b, h, dk, dv)
    return t


def _norm_inputs(c, r):
    n, m = c["rows"], c["channels"]
    dt = DTYPES[c["dtype"]]
    t = dict(x=(r.n(n, m) + 0.1).to(dt), weight=1.0 + r.n(m, scale=0.1))
    if c["bias"]:
        t["bias"] = r.n(m, scale=0.1)
    if c["residual"] != "none":
        t["residual"] = r.n(n, m, scale=2.0).to(DTYPES[c["residual"]])
    if c["kind"] == "norm_train":
        t["dout"] = r.n(n, m).to(dt)
        if c["prenorm"]:
            t["dres"] = r.n(n, m).to(t.get("residual", t["x"]).dtype)
    return t


_GRADS = {"train": ("q", "k", "v", "beta", "log_decay", "initial_state"), "norm_train": ("x", "residual", "weight", "bias")}


def _wanted(case, t):
    return [k for k in _GRADS[case["kind"]] if k in t and not (k == "log_decay" and case["decay"] == "fixed")]


def prepare(case, seed):
    r = _Rand(seed)
    t = _norm_inputs(case, r) if case["kind"].startswith("norm") else _delta_inputs(case, r)
    if case["kind"] in _GRADS:
        for k in _wanted(case, t):
            t[k] = t[k].detach().requires_grad_(True)
    return {"case": case, "t": t}


# ---- the plain forms -----------------------------------------------------------------------------

CHUNK = 64


def _plain_delta(q, k, v, beta, log_decay=None, initial_state=None):
    """Chunked: the corrections of a chunk's tokens to each other by forward substitution, row by row for all chunks at once, then
    chunk after chunk with the state."""
    b, L, G, dk = q.shape
    H, dv = v.shape[2], v.shape[3]
    R, C = H // G, CHUNK
    n = max(1, -(-L // C))

    def cut(x):  # (b, n, heads, C, ...)
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, n * C - L))
        return x.unflatten(1, (n, C)).transpose(2, 3)

    qc, kc = (cut(x).repeat_interleave(R, 2) for x in (q, k))
    vc = cut(v)
    bc = cut(beta.float().expand(b, L, H).unsqueeze(-1))
    g = torch.zeros(b, L, H, device=q.device) if log_decay is None else log_decay.float().expand(b, L, H)
    c = cut(g.unsqueeze(-1)).squeeze(-1).cumsum(-1)
    keep = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    decay = (c.unsqueeze(-1) - c.unsqueeze(-2)).masked_fill(~keep, float("-inf")).exp()
    a = (kc @ kc.transpose(-1, -2)) * decay * bc
    eye = torch.eye(C, device=q.device)
    rows = [eye[:1].expand(b, n, H, 1, C)]
    for i in range(1, C):
        rows.append(eye[i:i + 1] - a[..., i:i + 1, :i] @ torch.cat(rows, -2))
    inv = torch.cat(rows, -2)
    u0 = inv @ (bc * vc)
    w = inv @ (bc * kc * c.exp().unsqueeze(-1))
    m = (qc @ kc.transpose(-1, -2)) * decay
    qin = qc * c.exp().unsqueeze(-1)
    kout = (kc * (c[..., -1:] - c).exp().unsqueeze(-1)).transpose(-1, -2)
    all_ = c[..., -1].exp()[..., None, None]
    s = torch.zeros(b, H, dk, dv, device=q.device) if initial_state is None else initial_state.float()
    outs = []
    for j in range(n):
        u = u0[:, j] - w[:, j] @ s
        outs.append(qin[:, j] @ s + m[:, j] @ u)
        s = all_[:, j] * s + kout[:, j] @ u
    out = torch.stack(outs, 1).transpose(2, 3).flatten(1, 2)[:, :L] * dk ** -0.5
    return out.to(v.dtype), s


def _plain_token(state, q, k, v, beta, log_decay=None):
    b, H, dk, dv = state.shape
    R = H // q.shape[1]
    qh, kh = q.float().repeat_interleave(R, 1), k.float().repeat_interleave(R, 1)
    if log_decay is not None:
        state.mul_(log_decay.float().exp().expand(b, H)[..., None, None])
    z = (v.float() - (kh.unsqueeze(-1) * state).sum(-2)) * beta.float().unsqueeze(-1)
    state.add_(kh.unsqueeze(-1) * z.unsqueeze(-2))
    return ((qh.unsqueeze(-1) * state).sum(-2) * dk ** -0.5).to(v.dtype)


def _plain_norm(c, x, weight, bias=None, residual=None):
    h = x.float()
    if residual is not None:
        h = h + residual.float()
    d = h if c["rms"] else h - h.mean(-1, keepdim=True)
    y = d / ((d * d).mean(-1, keepdim=True) + 1e-5).sqrt() * weight
    if bias is not None:
        y = y + bias
    return y.to(x.dtype), h.to(x.dtype if residual is None else residual.dtype)


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if kind == "token":
        args = {k: t[k] for k in ("state", "q", "k", "v", "beta", "log_decay") if k in t}
        out = _mm().delta_rule_update(**args) if own else _plain_token(**args)
        return {"out": out, "state": t["state"]}
    names = _wanted(case, t) if kind in _GRADS else []
    if kind.startswith("norm"):
        args = {k: t[k] for k in ("x", "weight", "bias", "residual") if k in t}
        if own:
            got = _mm().layer_norm_fn(**args, eps=1e-5, prenorm=case["prenorm"], is_rms_norm=case["rms"])
            outs = list(got) if case["prenorm"] else [got]
        else:
            outs = list(_plain_norm(case, **args))[:2 if case["prenorm"] else 1]
        douts = [t.get("dout"), t.get("dres")][:len(outs)]
        res = dict(zip(("out", "residual_out"), (o.detach() for o in outs)))
    else:
        args = {k: t[k] for k in ("q", "k", "v", "beta", "log_decay", "initial_state") if k in t}
        last = kind == "prompt" or case["states"]
        if own:
            got = _mm().delta_rule_fn(**args, return_last_state=last)
            outs = list(got) if last else [got]
        else:
            outs = list(_plain_delta(**args))[:2 if last else 1]
        douts = [t.get("dout"), t.get("dlast")][:len(outs)]
        res = dict(zip(("out", "last_state"), (o.detach() for o in outs)))
    if names:
        res.update({"d" + k: v for k, v in zip(names, torch.autograd.grad(outs, [t[k] for k in names], douts))})
    return res


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    kind, s = case["kind"], SIZES[case["dtype"]]
    if kind.startswith("norm"):
        n, m = case["rows"], case["channels"]
        res = 0 if case["residual"] == "none" else SIZES[case["residual"]]
        out = (res or s) if case["prenorm"] else 0
        par = 4 * m * (2 if case["bias"] else 1)
        fwd = n * m * (2 * s + res + out)
        if kind == "norm":
            return {"bytes": fwd + par, "flops": n * m * 8}
        # Forward, then the two gradients read, those of x and the residual written; x and residual stay the same inputs.
        return {"bytes": fwd + n * m * (2 * s + res + out) + 2 * par, "flops": n * m * 24}
    b, h, g, dk, dv = case["batch"], case["heads"], case["groups"], case["dk"], case["dv"]
    L = case.get("L", 1)
    gates = {"token": b * L * h, "fixed": h, "none": 0}[case["decay"]]
    if kind == "token":
        return {"bytes": b * (8 * h * dk * dv + s * (2 * g * dk + 2 * h * dv)) + 4 * (b * h + gates), "flops": b * h * dk * dv * 7}
    state = 4 * b * h * dk * dv
    qk, v = s * b * L * g * dk, s * b * L * h * dv
    # Token by token: the state's product with k, its update and its product with q.
    fwd = b * L * h * dk * dv * 7
    if kind == "prompt":
        return {"bytes": 2 * qk + 2 * v + 4 * (b * L * h + gates) + state * (2 if case["states"] else 1), "flops": fwd}
    return {"bytes": 4 * qk + 4 * v + 4 * (2 * b * L * h + gates * (2 if case["decay"] == "token" else 1)) + (4 * state if case["states"] else 0),
            "flops": 4 * fwd}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_steps(q, k, v, beta, g, s):
    """Token by token, as the operator is defined; q and k of each head's own."""
    outs = []
    for t in range(v.shape[1]):
        if g is not None:
            s = s * g[:, t].exp()[..., None, None]
        z = v[:, t].unsqueeze(-2) - torch.matmul(k[:, t].unsqueeze(-2), s)
        s = s + (beta[:, t].unsqueeze(-1) * k[:, t]).unsqueeze(-1) * z
        outs.append(torch.matmul(q[:, t].unsqueeze(-2), s).squeeze(-2))
    return torch.stack(outs, 1) * q.shape[-1] ** -0.5, s


def _exact_grads(q, k, v, beta, g, s0, do, ds):
    """One (batch, head): the whole text as one triangular system and its derivatives written out."""
    scale, L = q.shape[-1] ** -0.5, q.shape[0]
    c = g.cumsum(0)
    keep = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
    d = (c[:, None] - c[None, :]).masked_fill_(~keep, float("-inf")).exp_()
    into, left = c.exp()[:, None], (c[-1] - c).exp()[:, None]
    n = ((k @ k.T) * d).tril_(-1)
    lhs = n * beta[None, :]
    lhs.diagonal().add_(1.0)                                     # (1 + n beta) z = x
    z = torch.linalg.solve_triangular(lhs, v - into * (k @ s0), upper=False, unitriangular=True)
    u = beta[:, None] * z
    m = (q @ k.T) * d
    out = scale * (into * (q @ s0) + m @ u)
    last = c[-1].exp() * s0 + (k * left).T @ u
    du = scale * (m.T @ do) + left * (k @ ds)
    # z's gradient is beta du; x's solves the transposed system.
    dx = torch.linalg.solve_triangular(lhs.T, beta[:, None] * du, upper=True, unitriangular=True)
    dbeta = (z * (du - n.T @ dx)).sum(1)
    pq, pn = scale * (do @ u.T) * d, -((dx @ u.T) * d).tril(-1)
    dq = pq @ k + scale * into * (do @ s0.T)
    dk = pq.T @ q + pn @ k + pn.T @ k - into * (dx @ s0.T) + left * (u @ ds.T)
    w = pq * (q @ k.T) + pn * (k @ k.T)
    li, ll = into[:, 0], left[:, 0]
    out_terms = ll * ((k @ ds) * u).sum(1)
    dc = w.sum(1) - w.sum(0) + li * (scale * ((q @ s0) * do).sum(1) - ((k @ s0) * dx).sum(1)) - out_terms
    dc[-1] += (ds * last).sum()
    return {"out": out, "last_state": last, "dq": dq, "dk": dk, "dv": dx, "dbeta": dbeta,
            "dlog_decay": dc.flip(0).cumsum(0).flip(0),
            "dinitial_state": c[-1].exp() * ds + scale * (q * into).T @ do - (k * into).T @ dx}


def _exact_delta(case, t):
    f = {k: v.detach().double() for k, v in t.items()}
    b, h, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    R = h // case["groups"]
    if case["kind"] == "token":
        q, k = f["q"].repeat_interleave(R, 1), f["k"].repeat_interleave(R, 1)
        g = f["log_decay"].expand(b, h)[:, None] if "log_decay" in f else None
        o, s = _exact_steps(q[:, None], k[:, None], f["v"][:, None], f["beta"][:, None], g, f["state"])
        return {"out": o[:, 0], "state": s}
    L = case["L"]
    g = f["log_decay"].expand(b, L, h) if "log_decay" in f else None
    s0 = f.get("initial_state", torch.zeros(b, h, dk, dv, dtype=torch.float64, device="cuda"))
    if case["kind"] == "prompt":
        o, s = _exact_steps(f["q"].repeat_interleave(R, 2), f["k"].repeat_interleave(R, 2), f["v"], f["beta"], g, s0)
        return {"out": o, "last_state": s}
    if L > 4096:
        return None
    if g is None:
        g = torch.zeros(b, L, h, dtype=torch.float64, device="cuda")
    ds = f.get("dlast", torch.zeros_like(s0))
    got = [[_exact_grads(f["q"][i, :, j // R], f["k"][i, :, j // R], f["v"][i, :, j], f["beta"][i, :, j], g[i, :, j], s0[i, j],
                         f["dout"][i, :, j], ds[i, j]) for j in range(h)] for i in range(b)]

    def heads(name, dim):
        return torch.stack([torch.stack([x[name] for x in row], dim) for row in got], 0)

    res = {"out": heads("out", 1)}
    if case["states"]:
        res["last_state"] = heads("last_state", 0)
    res["dq"], res["dk"] = (heads(n, 1).unflatten(2, (case["groups"], R)).sum(3) for n in ("dq", "dk"))
    res["dv"], res["dbeta"] = heads("dv", 1), heads("dbeta", 1)
    if case["decay"] == "token":
        res["dlog_decay"] = heads("dlog_decay", 1)
    if case["states"]:
        res["dinitial_state"] = heads("dinitial_state", 0)
    return res


def _exact_norm(case, t):
    f = {k: v.detach().double() for k, v in t.items()}
    h = f["x"] + f.get("residual", 0.0)
    mean = 0.0 if case["rms"] else h.mean(-1, keepdim=True)
    rstd = ((h - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    y = (h - mean) * rstd
    res = {"out": y * f["weight"] + f.get("bias", 0.0)}
    if case["prenorm"]:
        res["residual_out"] = h
    if case["kind"] == "norm":
        return res
    dy = f["dout"] * f["weight"]
    dh = dy - y * (dy * y).mean(-1, keepdim=True)
    if not case["rms"]:
        dh = dh - dy.mean(-1, keepdim=True)
    dh = dh * rstd + f.get("dres", 0.0)
    res["dx"] = dh
    if "residual" in f:
        res["dresidual"] = dh
    res["dweight"] = (f["dout"] * y).sum(0)
    if "bias" in f:
        res["dbias"] = f["dout"].sum(0)
    return res


def exact(case, seed):
    t = prepare(case, seed)["t"]
    return _exact_norm(case, t) if case["kind"].startswith("norm") else _exact_delta(case, t)
