"""The linear-attention layer's operators as measurable cases: attention with one decay for each head
(prompts, training steps, single tokens) and the gated group norm behind it.

``own`` False runs the plain form, elementary torch operations in float32; True makes the calls a user
makes. Both take what ``prepare`` returns.
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
        # One token of one sequence through a 5,120-channel layer of 80 heads: a chat at batch 1; latency.
        dict(name="token_b1", kind="token", batch=1, heads=80, groups=1, dk=128, dv=64, decay="token", dtype="bf16"),
        # The same step for a full serving batch: the states' memory traffic.
        dict(name="token_b256", kind="token", batch=256, heads=80, groups=1, dk=128, dv=64, decay="token", dtype="bf16"),
        # Two prompts of an odd length through a 1,536-channel layer, q, k and v slices of one projection.
        dict(name="prompt_odd", kind="prompt", batch=2, L=1777, heads=24, groups=1, dk=64, dv=64, decay="token",
             layout="fused", states=False, dtype="bf16"),
        # The prompt pass of a 5,120-channel layer, one group of q and k for all heads.
        dict(name="prompt_wide", kind="prompt", batch=4, L=4096, heads=80, groups=1, dk=128, dv=64, decay="token",
             layout="fused", states=False, dtype="bf16"),
        # A very long document in float32, continued from the state of what came before.
        dict(name="prompt_long_fp32", kind="prompt", batch=1, L=65536, heads=40, groups=4, dk=64, dv=64,
             decay="token", layout="dense", states=True, dtype="fp32"),
        # A training step of a 1,536-channel layer whose heads share q and k (their gradients sum over 24 heads).
        dict(name="train_shared", kind="train", batch=8, L=2048, heads=24, groups=1, dk=128, dv=64, decay="token",
             layout="fused", states=False, dtype="bf16"),
        # A training step with q and k of each head's own and a fixed decay for each head (retention).
        dict(name="train_heads", kind="train", batch=4, L=4096, heads=16, groups=16, dk=128, dv=128, decay="fixed",
             layout="dense", states=False, dtype="bf16"),
        # A training step on a piece of a longer text: state taken in and handed on, with both gradients.
        dict(name="train_states_fp16", kind="train", batch=4, L=1000, heads=64, groups=8, dk=64, dv=64,
             decay="token", layout="dense", states=True, dtype="fp16"),
        # The norm of 64 sequences' single tokens, one group for each of 80 heads, gated; latency.
        dict(name="norm_token", kind="norm", rows=64, channels=5120, groups=80, rms=False, gate="after", dtype="bf16"),
        # The norm of a prompt, one group for all channels, the gate multiplied in before it.
        dict(name="norm_prompt", kind="norm", rows=16384, channels=5120, groups=1, rms=True, gate="before",
             dtype="bf16"),
        # Forward and backward of the norm of a training step, one group for each head.
        dict(name="norm_train", kind="norm_train", rows=16384, channels=1536, groups=24, rms=False, gate="after",
             dtype="bf16"),
        # Forward and backward with an activation and no gate, odd group size, float32.
        dict(name="norm_train_odd", kind="norm_train", rows=5331, channels=1000, groups=8, rms=False, gate="none",
             dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["token", "prompt", "prompt", "train", "train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("norm"):
        groups = rng.choice([1, 1, 2, 8, 24, 80])
        size = _log_int(rng, 16, 128) if groups > 8 else _log_int(rng, 64, 5120 // groups)
        c = dict(kind=kind, rows=_log_int(rng, 1, 16384), channels=groups * size, groups=groups,
                 rms=rng.random() < 0.5, gate=rng.choice(["after", "before", "none"]), dtype=dtype)
        return c
    groups = rng.choice([1, 1, 2, 4, 8])
    c = dict(kind=kind, batch=_log_int(rng, 1, 8), L=_log_int(rng, 2, 8192), heads=groups * rng.choice([1, 2, 3, 5, 8, 10]),
             groups=groups, dk=rng.choice([16, 32, 40, 64, 64, 96, 128]), dv=rng.choice([32, 48, 64, 64, 80, 128]),
             decay=rng.choice(["token", "token", "fixed"]), dtype=dtype)
    if kind == "token":
        c["batch"] = _log_int(rng, 1, 256)
        del c["L"]
        return c
    c.update(layout=rng.choice(["fused", "dense"]), states=rng.random() < 0.4)
    if kind == "prompt" and rng.random() < 0.15:
        c["batch"], c["L"] = 1, _log_int(rng, 8192, 65536)
    most = {"prompt": 4 * 4096 * 80 * 128 * 64, "train": 4 * 4096 * 16 * 128 * 128 // 2}[kind]
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


def _attention_inputs(c, r):
    b, h, g, dk, dv = c["batch"], c["heads"], c["groups"], c["dk"], c["dv"]
    dt = DTYPES[c["dtype"]]
    lead = (b,) if c["kind"] == "token" else (b, c["L"])
    if c.get("layout") == "fused":
        qkv = r.n(*lead, 2 * g * dk + h * dv).to(dt)
        q, k, v = qkv.split([g * dk, g * dk, h * dv], -1)
        t = dict(q=q.unflatten(-1, (g, dk)), k=k.unflatten(-1, (g, dk)), v=v.unflatten(-1, (h, dv)))
    else:
        t = dict(q=r.n(*lead, g, dk).to(dt), k=r.n(*lead, g, dk).to(dt), v=r.n(*lead, h, dv).to(dt))
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
    t = dict(x=(r.n(n, m, scale=2.0) + 0.5).to(dt), weight=1.0 + r.n(m, scale=0.1))
    if not c["rms"]:
        t["bias"] = r.n(m, scale=0.1)
    if c["gate"] != "none":
        t["z"] = r.n(n, m).to(dt)
    if c["kind"] == "norm_train":
        t["dout"] = r.n(n, m).to(dt)
    return t


_GRADS = {"train": ("q", "k", "v", "log_decay", "initial_state"), "norm_train": ("x", "weight", "bias", "z")}


def _wanted(case, t):
    return [k for k in _GRADS[case["kind"]] if k in t and not (k == "log_decay" and case["decay"] == "fixed")]


def prepare(case, seed):
    r = _Rand(seed)
    t = _norm_inputs(case, r) if case["kind"].startswith("norm") else _attention_inputs(case, r)
    if case["kind"] in _GRADS:
        for k in _wanted(case, t):
            t[k] = t[k].detach().requires_grad_(True)
    return {"case": case, "t": t}


# ---- the plain forms -----------------------------------------------------------------------------

CHUNK = 64


def _plain_attention(q, k, v, log_decay, initial_state=None):
    """Chunked: within a chunk the masked product of q and k, between chunks the states that each
    chunk adds, brought to every later chunk's start by their decays in one product."""
    b, L, G, dk = q.shape
    H, dv = v.shape[2], v.shape[3]
    R, C = H // G, CHUNK
    n = max(1, -(-L // C))
    pad = n * C - L
    g = log_decay.float().expand(b, L, H)

    def cut(x):  # (b, n, heads, C, ...)
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, pad))
        return x.unflatten(1, (n, C)).transpose(2, 3)

    qc, kc = cut(q).unsqueeze(3), cut(k).unsqueeze(3)
    vc = cut(v).unflatten(2, (G, R))
    c = cut(g.unsqueeze(-1)).squeeze(-1).unflatten(2, (G, R)).cumsum(-1)
    keep = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    decay = (c.unsqueeze(-1) - c.unsqueeze(-2)).masked_fill(~keep, float("-inf")).exp()
    out = ((qc @ kc.transpose(-1, -2)) * decay) @ vc
    added = kc.transpose(-1, -2) @ (vc * (c[..., -1:] - c).exp().unsqueeze(-1))
    total = c[..., -1].permute(0, 2, 3, 1).cumsum(-1)                      # (b, G, R, n)
    before = torch.nn.functional.pad(total, (1, 0))                        # decay up to each chunk's start
    earlier = torch.ones(n + 1, n, dtype=torch.bool, device=q.device).tril(-1)
    carry = (before.unsqueeze(-1) - total.unsqueeze(-2)).masked_fill(~earlier, float("-inf")).exp()
    starts = carry @ added.permute(0, 2, 3, 1, 4, 5).flatten(-2)           # (b, G, R, n + 1, dk * dv)
    if initial_state is not None:
        starts = starts + before.exp().unsqueeze(-1) * initial_state.float().reshape(b, G, R, 1, dk * dv)
    starts = starts.unflatten(-1, (dk, dv))
    out = out + (qc @ starts[:, :, :, :-1].permute(0, 3, 1, 2, 4, 5)) * c.exp().unsqueeze(-1)
    out = out.flatten(2, 3).transpose(2, 3).flatten(1, 2)[:, :L] * dk ** -0.5
    return out.to(v.dtype), starts[:, :, :, -1].reshape(b, H, dk, dv)


def _plain_token(state, q, k, v, log_decay):
    b, H, dk, dv = state.shape
    R = H // q.shape[1]
    qh, kh = q.float().repeat_interleave(R, 1), k.float().repeat_interleave(R, 1)
    state.mul_(log_decay.float().exp().expand(b, H)[..., None, None])
    state.add_(kh.unsqueeze(-1) * v.float().unsqueeze(-2))
    return ((qh.unsqueeze(-1) * state).sum(-2) * dk ** -0.5).to(v.dtype)


def _plain_norm(c, x, weight, bias=None, z=None):
    h = x.float()
    silu = lambda a: a / (1.0 + (-a).exp())  # noqa: E731
    if c["gate"] == "before":
        h = h * silu(z.float())
    h = h.unflatten(-1, (c["groups"], -1))
    if not c["rms"]:
        h = h - h.mean(-1, keepdim=True)
    h = (h / ((h * h).mean(-1, keepdim=True) + 1e-5).sqrt()).flatten(-2) * weight
    if bias is not None:
        h = h + bias
    if c["gate"] == "after":
        h = h * silu(z.float())
    elif c["gate"] == "none":
        h = silu(h)
    return h.to(x.dtype)


# ---- one pass ------------------------------------------------------------------------------------


def _own_norm(c, x, weight, bias=None, z=None):
    return _mm().group_norm_fn(x, c["groups"], weight, bias, z=z, eps=1e-5,
                               activation="silu" if c["gate"] == "none" else None, is_rms_norm=c["rms"],
                               norm_before_gate=c["gate"] != "before")


def run(state):
    case, t = state["case"], state["t"]
    kind = case["kind"]
    if kind == "token":
        args = (t["state"], t["q"], t["k"], t["v"], t["log_decay"])
        out = _mm().linear_attention_update(*args) if own else _plain_token(*args)
        return {"out": out, "state": t["state"]}
    names = _wanted(case, t) if kind in _GRADS else []
    if kind.startswith("norm"):
        args = {k: t[k] for k in ("x", "weight", "bias", "z") if k in t}
        out = _own_norm(case, **args) if own else _plain_norm(case, **args)
        outs, douts, res = [out], [t.get("dout")], {"out": out.detach()}
    else:
        args = {k: t[k] for k in ("q", "k", "v", "log_decay", "initial_state") if k in t}
        if not own:
            out, last = _plain_attention(**args)
        elif kind == "prompt" or case["states"]:
            out, last = _mm().linear_attention_fn(**args, return_last_state=True)
        else:
            out = _mm().linear_attention_fn(**args)
        outs, douts, res = [out], [t.get("dout")], {"out": out.detach()}
        if kind == "prompt" or case["states"]:
            res["last_state"] = last.detach()
            if kind == "train":
                outs, douts = [out, last], [t["dout"], t["dlast"]]
    if names:
        res.update({"d" + k: v for k, v in zip(names, torch.autograd.grad(outs, [t[k] for k in names], douts))})
    return res


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    kind, s = case["kind"], SIZES[case["dtype"]]
    if kind.startswith("norm"):
        n, m = case["rows"], case["channels"]
        z = 0 if case["gate"] == "none" else 1
        par = 4 * m * (1 if case["rms"] else 2)
        if kind == "norm":
            return {"bytes": s * n * m * (2 + z) + par, "flops": n * m * (8 + 6 * z)}
        return {"bytes": s * n * m * (4 + 2 * z) + 2 * par, "flops": n * m * (24 + 14 * z)}
    b, h, g, dk, dv = case["batch"], case["heads"], case["groups"], case["dk"], case["dv"]
    if kind == "token":
        n_g = h if case["decay"] == "fixed" else b * h
        return {"bytes": b * (8 * h * dk * dv + s * (2 * g * dk + 2 * h * dv)) + 4 * n_g, "flops": b * h * dk * dv * 5}
    L = case["L"]
    n_g = h if case["decay"] == "fixed" else b * L * h
    state = 4 * b * h * dk * dv
    qk, v = s * b * L * g * dk, s * b * L * h * dv
    # Token by token: the state's update and its product with q.
    fwd = b * L * h * dk * dv * 5
    if kind == "prompt":
        return {"bytes": 2 * qk + 2 * v + 4 * n_g + state * (2 if case["states"] else 1), "flops": fwd}
    return {"bytes": 4 * qk + 4 * v + 4 * n_g * (1 if case["decay"] == "fixed" else 2) + (4 * state if case["states"] else 0),
            "flops": 4 * fwd}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_steps(q, k, v, g, s):
    """Token by token, as the operator is defined; q and k of each head's own."""
    outs = []
    for t in range(v.shape[1]):
        s = s * g[:, t].exp()[..., None, None]
        s = s + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        outs.append(torch.matmul(q[:, t].unsqueeze(-2), s).squeeze(-2))
    return torch.stack(outs, 1) * q.shape[-1] ** -0.5, s


def _exact_grads(q, k, v, g, s0, do, ds):
    """One (batch, head): the whole masked product and its derivatives written out."""
    scale, L = q.shape[-1] ** -0.5, q.shape[0]
    c = g.cumsum(0)
    keep = torch.ones(L, L, dtype=torch.bool, device=q.device).tril()
    d = (c[:, None] - c[None, :]).masked_fill_(~keep, float("-inf")).exp_() * scale
    p, dp = (q @ k.T) * d, (do @ v.T)
    into, left = c.exp()[:, None] * scale, (c[-1] - c).exp()[:, None]
    out = p @ v + into * (q @ s0)
    last = c[-1].exp() * s0 + (k * left).T @ v
    w = p * dp
    dc = w.sum(1) - w.sum(0) + ((q @ s0) * do * into).sum(1) - ((k @ ds) * v * left).sum(1)
    dc[-1] += (ds * last).sum()
    dp *= d
    return {"out": out, "last_state": last, "dq": dp @ k + into * (do @ s0.T), "dk": dp.T @ q + left * (v @ ds.T),
            "dv": p.T @ do + left * (k @ ds), "dlog_decay": dc.flip(0).cumsum(0).flip(0),
            "dinitial_state": c[-1].exp() * ds + (q * into).T @ do}


def _exact_attention(case, t):
    f = {k: v.detach().double() for k, v in t.items()}
    b, h, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    R = h // case["groups"]
    if case["kind"] == "token":
        q, k = f["q"].repeat_interleave(R, 1), f["k"].repeat_interleave(R, 1)
        o, s = _exact_steps(q[:, None], k[:, None], f["v"][:, None], f["log_decay"].expand(b, h)[:, None], f["state"])
        return {"out": o[:, 0], "state": s}
    L = case["L"]
    g = f["log_decay"].expand(b, L, h)
    s0 = f.get("initial_state", torch.zeros(b, h, dk, dv, dtype=torch.float64, device="cuda"))
    if case["kind"] == "prompt":
        o, s = _exact_steps(f["q"].repeat_interleave(R, 2), f["k"].repeat_interleave(R, 2), f["v"], g, s0)
        return {"out": o, "last_state": s}
    if L > 4096:
        return None
    ds = f.get("dlast", torch.zeros_like(s0))
    got = [[_exact_grads(f["q"][i, :, j // R], f["k"][i, :, j // R], f["v"][i, :, j], g[i, :, j], s0[i, j],
                         f["dout"][i, :, j], ds[i, j]) for j in range(h)] for i in range(b)]

    def heads(name, dim):
        return torch.stack([torch.stack([x[name] for x in row], dim) for row in got], 0)

    res = {"out": heads("out", 1)}
    if case["states"]:
        res["last_state"] = heads("last_state", 0)
    res["dq"], res["dk"] = (heads(n, 1).unflatten(2, (case["groups"], R)).sum(3) for n in ("dq", "dk"))
    res["dv"] = heads("dv", 1)
    if case["decay"] == "token":
        res["dlog_decay"] = heads("dlog_decay", 1)
    if case["states"]:
        res["dinitial_state"] = heads("dinitial_state", 0)
    return res


def _exact_norm(case, t):
    f = {k: v.detach().double() for k, v in t.items()}
    x, w = f["x"], f["weight"]
    n, m = x.shape
    G, gate = case["groups"], case["gate"]
    sig = torch.sigmoid(f["z"]) if gate != "none" else None
    act = f["z"] * sig if gate != "none" else None
    h = (x * act if gate == "before" else x).view(n, G, m // G)
    mean = torch.zeros(n, G, 1, dtype=h.dtype, device=h.device) if case["rms"] else h.mean(-1, keepdim=True)
    rstd = ((h - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    y = (h - mean) * rstd
    a = y.view(n, m) * w + f.get("bias", 0.0)
    s = torch.sigmoid(a)
    res = {"out": a * act if gate == "after" else a * s if gate == "none" else a}
    if case["kind"] == "norm":
        return res
    dout = f["dout"]
    da = dout * act if gate == "after" else dout * s * (1 + a * (1 - s)) if gate == "none" else dout
    dy = (da * w).view(n, G, m // G)
    dh = dy - y * (dy * y).mean(-1, keepdim=True)
    if not case["rms"]:
        dh = dh - dy.mean(-1, keepdim=True)
    dh = (dh * rstd).view(n, m)
    res["dx"] = dh * act if gate == "before" else dh
    res["dweight"] = (da * y.view(n, m)).sum(0)
    if "bias" in f:
        res["dbias"] = da.sum(0)
    if gate != "none":
        res["dz"] = (dout * a if gate == "after" else dh * x) * sig * (1 + f["z"] * (1 - sig))
    return res


def exact(case, seed):
    t = prepare(case, seed)["t"]
    return _exact_norm(case, t) if case["kind"].startswith("norm") else _exact_attention(case, t)
