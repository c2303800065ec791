"""GPU tests of what the linear attention's texts promise beyond its results' bounds (tests/test_gpu_linattn.py): 16-bit results
are float32 ones rounded once."""
import sys

import pytest
import torch

from tests import linattn_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def _randn(r, *shape):
    return torch.randn(*shape, generator=r)


def _rounded_once(got, exact, size, what):
    """|got - exact| within half a unit of got's type at the exact value, and 2^-19 of the terms: each is a product of up to
    three factors within 2^-25 of their values, and of three exponentials of arguments up to 10 or so, 2^-24 (1 + 10 / 8) each
    at most; the sums' own roundings are smaller. A factor in 17 bits moves every few hundredth result past it."""
    g, e = got.detach().cpu().double(), exact.double()
    least, half = {BF16: (-126, -8), F16: (-14, -11)}[got.dtype]
    unit = torch.exp2(torch.floor(torch.log2(e.abs().clamp_min(2.0 ** least))) + half)
    bad = (g - e).abs() > unit + 2.0 ** -19 * size
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}"


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_are_float32(dtype):
    """Decays of e^-2 or so: every output is little more than its own token's score times v."""
    _say(f"linear attention scores {dtype}")
    from motif_mamba_amd import linear_attention_fn
    r = torch.Generator().manual_seed(1)
    t = {"q": _randn(r, 64, 64, 1, 1).to(dtype), "k": _randn(r, 64, 64, 1, 1).to(dtype), "v": _randn(r, 64, 64, 4, 64).to(dtype),
         "log_decay": -2 - torch.rand(64, 64, 4, generator=r)}
    out = linear_attention_fn(**{n: x.to(DEV) for n, x in t.items()}, scale=0.3)
    _rounded_once(out, ref.with_grads(t, 0.3)["out"], ref.magnitudes(t, 0.3)["out"], "out")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_states_are_float32(dtype):
    """Nothing but the state that was handed in."""
    _say(f"linear attention states {dtype}")
    from motif_mamba_amd import linear_attention_fn
    r = torch.Generator().manual_seed(2)
    t = {"q": _randn(r, 64, 64, 1, 1).to(dtype), "k": torch.zeros(64, 64, 1, 1, dtype=dtype), "v": _randn(r, 64, 64, 4, 64).to(dtype),
         "log_decay": -0.1 * torch.rand(64, 64, 4, generator=r), "initial_state": _randn(r, 64, 4, 1, 64)}
    out = linear_attention_fn(**{n: x.to(DEV) for n, x in t.items()}, scale=0.3)
    _rounded_once(out, ref.with_grads(t, 0.3)["out"], ref.magnitudes(t, 0.3)["out"], "out")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", [(1, 64), (64, 1)])
def test_gradients_are_float32(dtype, dk, dv):
    """Without a gradient of the decays or of a state, the states' gradient too is float32: few terms, most of them from behind
    the token's chunk."""
    _say(f"linear attention gradients {dk} {dv} {dtype}")
    from motif_mamba_amd import linear_attention_fn
    r = torch.Generator().manual_seed(3)
    b, L, H = 16, 130, 4
    t = {"q": _randn(r, b, L, H, dk).to(dtype), "k": _randn(r, b, L, H, dk).to(dtype), "v": _randn(r, b, L, H, dv).to(dtype)}
    dout = _randn(r, b, L, H, dv).to(dtype)
    dout[:, torch.arange(L) % 65 != 64] = 0
    g = {"log_decay": -0.02 * torch.rand(b, L, H, generator=r)}
    leaves = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
    got = torch.autograd.grad(linear_attention_fn(**leaves, log_decay=g["log_decay"].to(DEV), scale=0.3), list(leaves.values()), dout.to(DEV))
    exact, size = ref.with_grads({**t, **g}, 0.3, dout), ref.magnitudes({**t, **g}, 0.3, dout)
    for n, x in zip(leaves, got):
        _rounded_once(x, exact["d" + n], size["d" + n], "d" + n)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_heads(dtype):
    """No head uses q and k: their gradients are empty sums, 0, whatever stood in the memory they get."""
    _say(f"linear attention without heads {dtype}")
    from motif_mamba_amd import linear_attention_fn
    q, k = (torch.randn(2, 300, 1, 16, device=DEV).to(dtype).requires_grad_(True) for _ in range(2))
    v = torch.zeros(2, 300, 0, 8, device=DEV, dtype=dtype, requires_grad=True)
    out, last = linear_attention_fn(q, k, v, torch.zeros(2, 300, 0, device=DEV), return_last_state=True)
    assert out.shape == (2, 300, 0, 8) and last.shape == (2, 0, 16, 8)
    junk = [torch.full((2, 300, 1, 16), float("nan"), device=DEV, dtype=dtype) for _ in range(8)]
    del junk
    dq, dk, dv = torch.autograd.grad(out, [q, k, v], torch.zeros_like(out))
    assert dq.shape == q.shape and not dq.any() and not dk.any() and dv.shape == v.shape


def _token(seed=4):
    r = torch.Generator().manual_seed(seed)
    t = {"q": _randn(r, 2, 5, 1, 16), "k": _randn(r, 2, 5, 1, 16), "v": _randn(r, 2, 5, 2, 8), "log_decay": -torch.rand(2, 5, 2, generator=r)}
    return {n: x.to(DEV) for n, x in t.items()}, _randn(r, 2, 2, 16, 8).to(DEV)


def test_update_counts_as_a_change_of_the_state():
    """A state that a backward still needs is updated: an error, as with torch's own in-place operations."""
    _say("linear attention update: version")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    t, state = _token()
    q = t["q"].clone().requires_grad_(True)
    out = linear_attention_fn(q, t["k"], t["v"], t["log_decay"], initial_state=state)
    before = state._version
    linear_attention_update(state, *(t[n][:, 0] for n in ("q", "k", "v", "log_decay")))
    assert state._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with torch.inference_mode():
        s = torch.zeros_like(state)
        linear_attention_update(s, *(t[n][:, 0] for n in ("q", "k", "v", "log_decay")))
        assert s.any()


@pytest.mark.parametrize("which", ["state", "q", "k", "v", "log_decay"])
def test_update_refuses_derivatives(which):
    _say(f"linear attention update: {which} with a derivative")
    from torch.autograd import forward_ad
    from motif_mamba_amd import linear_attention_update
    t, state = _token()
    args = {"state": state, **{n: x[:, 0].clone() for n, x in t.items()}}
    leaf = {**args, which: args[which].clone().requires_grad_(True)}
    with pytest.raises(RuntimeError, match="derivatives"):
        linear_attention_update(**leaf)
    with torch.no_grad():
        assert not linear_attention_update(**leaf).requires_grad
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="derivatives"):
        linear_attention_update(**{**args, which: forward_ad.make_dual(args[which], torch.ones_like(args[which]))})


def test_block_step_refuses_derivatives():
    """In grad mode, before the cache is touched: the operators of one token have no derivatives."""
    _say("linear attention block: step in grad mode")
    from motif_mamba_amd import LinearAttentionBlock
    torch.manual_seed(5)
    b = LinearAttentionBlock(32, nheads=2, headdim=16, d_state=16).to(DEV)
    cache = b.allocate_inference_cache(2)
    with pytest.raises(RuntimeError, match="derivatives"):
        b.step(torch.randn(2, 32, device=DEV), cache)
    assert not cache[0].any() and not cache[1].any()
    with torch.no_grad():
        b.step(torch.randn(2, 32, device=DEV), cache)
    assert cache[0].any() and cache[1].any()
    for p in b.parameters():
        p.requires_grad_(False)
    b.step(torch.randn(2, 32, device=DEV), cache)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("grow", [88.8, 90.0, 1000.0, float("inf")])
def test_growing_states(dtype, grow):
    """A log decay whose exponential is infinite makes the state infinite, not NaN."""
    _say(f"linear attention log decay {grow} {dtype}")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    r = torch.Generator().manual_seed(6)
    t = {"q": _randn(r, 1, 1, 1, 1).abs().to(dtype), "k": _randn(r, 1, 1, 1, 1).to(dtype), "v": _randn(r, 1, 1, 2, 16).to(dtype),
         "log_decay": torch.full((1, 1, 2), grow), "initial_state": 1 + torch.rand(1, 2, 1, 16, generator=r)}
    d = {n: x.to(DEV) for n, x in t.items()}
    out, last = linear_attention_fn(**d, return_last_state=True)
    assert torch.isposinf(out).all() and torch.isposinf(last).all()
    state = d["initial_state"].clone()
    out = linear_attention_update(state, *(d[n][:, 0] for n in ("q", "k", "v", "log_decay")))
    assert torch.isposinf(out).all() and torch.isposinf(state).all()


def _infinite(dtype, L, dk, dv, which, bad, at, forget=(), states=True):
    """Inputs with one infinity (or a token of them) and what the definition makes of it, in float64."""
    r = torch.Generator().manual_seed(7 + L + dk)
    t = {"q": _randn(r, 1, L, 1, dk).to(dtype), "k": _randn(r, 1, L, 1, dk).to(dtype), "v": _randn(r, 1, L, 2, dv).to(dtype),
         "log_decay": -0.5 * torch.rand(1, L, 2, generator=r)}
    if states:
        t["initial_state"] = _randn(r, 1, 2, dk, dv)
    clean = {n: x.clone() for n, x in t.items()}
    for f in forget:
        t["log_decay"][:, f] = clean["log_decay"][:, f] = float("-inf")
    if which == "initial_state":
        t[which][0, 0, dk // 2, dv // 3] = bad
    elif which == "v":
        t[which][0, at, 1, dv // 2] = bad
    else:
        t[which][0, at, 0, dk // 3] = bad
    return t, clean


def _same_kinds(got, exact, what):
    g, e = got.cpu().double(), exact
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(g), kind(e)), (what, kind.__name__, int((kind(g) != kind(e)).sum()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("which", ["q", "k", "v", "initial_state"])
@pytest.mark.parametrize("L,dk,dv", [(1, 16, 16), (90, 64, 64), (150, 128, 128), (70, 37, 50), (1100, 64, 64), (1100, 128, 100)])
def test_infinite_values(L, dk, dv, which, dtype):
    """An infinity becomes what the recurrence makes of it, infinity or NaN, in outputs and states, in one segment and in several,
    and everything that it does not reach keeps its bits."""
    _say(f"linear attention infinite {which} {L} {dk} {dv} {dtype}")
    from motif_mamba_amd import linear_attention_fn
    for bad, at in ((float("inf"), 0), (float("-inf"), L // 3)):
        t, clean = _infinite(dtype, L, dk, dv, which, bad, at)
        out, last = linear_attention_fn(**{n: x.to(DEV) for n, x in t.items()}, scale=0.25, return_last_state=True)
        exact = ref.recurrence(*(t[n].double() for n in ("q", "k", "v", "log_decay")), 0.25, t["initial_state"].double())
        _same_kinds(out, exact[0], "out")
        _same_kinds(last, exact[1], "last_state")
        want = linear_attention_fn(**{n: x.to(DEV) for n, x in clean.items()}, scale=0.25, return_last_state=True)
        for x, y, e in zip((out, last), want, exact):
            assert torch.equal(x[e.isfinite().to(DEV)], y[e.isfinite().to(DEV)])


@pytest.mark.parametrize("L", [150, 1100])
def test_infinite_values_and_forgotten_states(L):
    """0 times infinity is NaN in the recurrence too: -inf does not forget an infinity."""
    _say(f"linear attention infinite v, -inf {L}")
    from motif_mamba_amd import linear_attention_fn
    t, _ = _infinite(BF16, L, 64, 64, "v", float("inf"), 40, forget=(20, 100))
    out, last = linear_attention_fn(**{n: x.to(DEV) for n, x in t.items()}, return_last_state=True)
    exact = ref.recurrence(*(t[n].double() for n in ("q", "k", "v", "log_decay")), 0.125, t["initial_state"].double())
    _same_kinds(out, exact[0], "out")
    _same_kinds(last, exact[1], "last_state")


def test_infinite_values_then_tokens():
    """The prompt and its tokens one by one agree."""
    _say("linear attention infinite v, tokens")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    t, _ = _infinite(F32, 40, 32, 32, "v", float("inf"), 10)
    d = {n: x.to(DEV) for n, x in t.items()}
    out, last = linear_attention_fn(**d, return_last_state=True)
    state = d["initial_state"].clone()
    for n in range(40):
        y = linear_attention_update(state, *(d[m][:, n] for m in ("q", "k", "v", "log_decay")))
        _same_kinds(out[:, n], y.cpu().double(), n)
    _same_kinds(last, state.cpu().double(), "state")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cuts", [(7,), (40, 90), (130, 300), (256,), (100, 101, 480)])
def test_documents_do_not_share_rounding(cuts, dtype):
    """Documents apart by -inf, every other one 30 times as large (its decays' gradients some 10^6 times): each one's results within
    the bound of its own terms. (Gradients of 30^3 and more pass float16's range.)"""
    _say(f"linear attention documents {cuts} {dtype}")
    from motif_mamba_amd import linear_attention_fn
    L, edges = 520, (0, *cuts, 520)
    r = torch.Generator().manual_seed(8)
    t = {"q": _randn(r, 1, L, 1, 32), "k": _randn(r, 1, L, 1, 32), "v": _randn(r, 1, L, 2, 32), "log_decay": -0.05 * torch.rand(1, L, 2, generator=r)}
    dout = _randn(r, 1, L, 2, 32)
    for n, (a, b) in enumerate(zip(edges, edges[1:])):
        for x in (t["q"], t["k"], t["v"], dout):
            x[:, a:b] *= 30.0 if n % 2 else 1.0
        if n:
            t["log_decay"][:, a] = float("-inf")
    t = {n: x if n == "log_decay" else x.to(dtype) for n, x in t.items()}
    dout = dout.to(dtype)
    leaves = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
    got = torch.autograd.grad(linear_attention_fn(**leaves, scale=0.2), list(leaves.values()), dout.to(DEV))
    for a, b in zip(edges, edges[1:]):
        part = {n: x[:, a:b].clone() for n, x in t.items()}
        part["log_decay"][:, 0] = 0.0   # nothing stands before it
        exact, size = ref.with_grads(part, 0.2, dout[:, a:b]), ref.magnitudes(part, 0.2, dout[:, a:b])
        for n, x in zip(leaves, got):
            x, e, z = x[:, a:b], exact["d" + n], size["d" + n]
            if n == "log_decay" and a:
                assert not x[:, 0].any()
                x, e, z = x[:, 1:], e[:, 1:], z[:, 1:]
                if not e.numel():
                    continue
            ref.check(x, e, z, F32, f"d{n} of {a} .. {b}", whole_row=n == "log_decay")


def test_block_cache_is_no_part_of_the_graph():
    """A prompt in grad mode fills the cache with values; the outputs still have their gradients."""
    _say("linear attention block: cache in grad mode")
    from motif_mamba_amd import LinearAttentionBlock
    torch.manual_seed(9)
    b = LinearAttentionBlock(32, nheads=2, headdim=16, d_state=16).to(DEV)
    hidden = torch.randn(2, 20, 32, device=DEV)
    cache, plain = b.allocate_inference_cache(2), b.allocate_inference_cache(2)
    out = b(hidden, cache)
    for x in cache:
        assert not x.requires_grad and x.grad_fn is None
    with torch.no_grad():
        assert torch.equal(b(hidden, plain), out)
        b.step(torch.randn(2, 32, device=DEV), cache)   # in place, while the graph is alive
    grads = torch.autograd.grad(out.sum(), list(b.parameters()))
    assert all(torch.isfinite(g).all() and g.any() for g in grads)
    assert torch.equal(b(hidden), out)


def test_most_pairs():
    """As many (batch row, head) pairs as the texts allow: prompts and their gradients, one token."""
    _say("linear attention most pairs")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    n = (1 << 23) - 1
    r = torch.Generator(device=DEV).manual_seed(10)
    q, k, v = (torch.randn(n, 1, 1, 1, generator=r, device=DEV).requires_grad_(True) for _ in range(3))
    g = -torch.rand(n, 1, 1, generator=r, device=DEV)
    out = linear_attention_fn(q, k, v, g, scale=0.5)
    torch.testing.assert_close(out, 0.5 * q * k * v, rtol=1e-6, atol=1e-30)
    got = torch.autograd.grad(out, [q, k, v], torch.ones_like(out))
    for x, y in zip(got, (k * v, q * v, q * k)):
        torch.testing.assert_close(x, 0.5 * y, rtol=1e-6, atol=1e-30)
    n = (1 << 24) - 1
    state, q, k, v = (torch.randn(n, 1, 1, generator=r, device=DEV) for _ in range(4))
    g = -torch.rand(n, 1, generator=r, device=DEV)
    want = g.exp()[..., None] * state + k * v
    y = linear_attention_update(state.unsqueeze(-1), q, k, v, g, scale=2.0)
    torch.testing.assert_close(state, want, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(y, 2 * q * want, rtol=1e-6, atol=1e-5)


def test_states_of_more_than_2_to_the_32_elements():
    """No tokens: the states are handed on, 17 GB of them."""
    _say("linear attention 2^32 elements of states")
    from motif_mamba_amd import linear_attention_fn
    heads = (1 << 18) + 3
    initial = torch.zeros(1, heads, 128, 128, device=DEV)
    for at in (0, heads // 2, heads - 1):
        initial[0, at] = torch.randn(128, 128, device=DEV)
    x = torch.zeros(1, 0, 1, 128, device=DEV)
    _, last = linear_attention_fn(x, x, torch.zeros(1, 0, heads, 128, device=DEV), torch.zeros(1, 0, heads, device=DEV), initial_state=initial,
                                  return_last_state=True)
    for at in (0, 1, heads // 2, heads - 2, heads - 1):
        assert torch.equal(last[0, at], initial[0, at]), at
    del initial, last
    torch.cuda.empty_cache()


def test_tokens_far_apart():
    """A layout with the tokens outermost, 2^22 elements and more from one to the next, and a single token with any stride."""
    _say("linear attention tokens far apart")
    from motif_mamba_amd import linear_attention_fn
    r = torch.Generator(device=DEV).manual_seed(11)
    for wide in (1 << 22, (1 << 22) - 1):
        buf = torch.randn(5, 1, wide, generator=r, device=DEV).to(BF16).transpose(0, 1)
        q, k, v, dout = (buf[..., n:n + 64].unflatten(-1, (2, 32)) for n in (0, 64, 128, 192))
        g = -torch.rand(1, 5, 2, generator=r, device=DEV)
        res = []
        for copy in (False, True):
            leaves = [(x.contiguous() if copy else x).detach().requires_grad_(True) for x in (q, k, v)]
            out = linear_attention_fn(*leaves, g)
            res.append((out, *torch.autograd.grad(out, leaves, dout.contiguous() if copy else dout)))
        for x, y in zip(*res):
            assert torch.equal(x, y)
        one = [x[:, :1] for x in (q, k, v)]
        assert torch.equal(linear_attention_fn(*one, g[:, :1]), res[0][0][:, :1])
