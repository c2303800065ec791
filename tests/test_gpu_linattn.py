"""GPU tests of the linear attention with one decay for each head (mm_linattn.hip) against the recurrence in float64
(tests/linattn_ref.py, which derives the bounds): lengths around the chunk, the block and the segments, odd sizes,
shared heads, strides, forgotten states, non-finite values in places a token does not see, gradients, refusals."""
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


def _inputs(seed, b, L, G, H, dk, dv, dtype, gdtype=F32, per_head=False, states=False, fast=0.3):
    r = torch.Generator().manual_seed(seed)
    t = {"q": torch.randn(b, L, G, dk, generator=r).to(dtype), "k": torch.randn(b, L, G, dk, generator=r).to(dtype),
         "v": torch.randn(b, L, H, dv, generator=r).to(dtype)}
    # Decays from 1 - 1e-3 to exp(-2) or so, by head.
    rate = torch.exp(torch.rand(H, generator=r) * 6 - 6.9) * (1 + fast)
    t["log_decay"] = (-rate if per_head else -rate * (0.2 + torch.rand(b, L, H, generator=r))).to(gdtype)
    if states:
        t["initial_state"] = torch.randn(b, H, dk, dv, generator=r)
    return t


def _to(t):
    return {n: x.to(DEV) for n, x in t.items()}


# (batch, seqlen, groups, heads, dk, dv)
SHAPES = [(2, 1, 1, 2, 16, 16), (1, 2, 1, 1, 1, 1), (1, 31, 1, 2, 32, 64), (2, 33, 2, 4, 64, 64), (1, 64, 1, 3, 128, 64),
          (1, 65, 1, 2, 64, 128), (2, 129, 1, 3, 37, 50), (1, 257, 3, 3, 128, 128), (1, 300, 2, 6, 80, 96), (1, 300, 1, 2, 72, 65)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    _say(f"linear attention forward {shape} {dtype}")
    from motif_mamba_amd import linear_attention_fn
    t = _inputs(sum(shape), *shape, dtype)
    scale = shape[4] ** -0.5
    exact, size = ref.with_grads(t, scale), ref.magnitudes(t, scale)
    out, last = linear_attention_fn(**_to(t), return_last_state=True)
    assert out.dtype == dtype and last.dtype == F32
    ref.check(out, exact["out"], size["out"], dtype, "out")
    ref.check(last, exact["last_state"], size["last_state"], dtype, "last_state")
    assert torch.equal(linear_attention_fn(**_to(t)), out)


def _grads(t, scale, dout, dlast=None):
    from motif_mamba_amd import linear_attention_fn
    leaves = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
    out, last = linear_attention_fn(**leaves, scale=scale, return_last_state=True)
    outs, douts = [out], [dout.to(DEV)]
    if dlast is not None:
        outs, douts = [out, last], [dout.to(DEV), dlast.to(DEV)]
    g = torch.autograd.grad(outs, list(leaves.values()), douts)
    return {"out": out, "last_state": last, **{"d" + n: x for n, x in zip(leaves, g)}}


def _check_all(got, t, scale, dout, dlast, dtype):
    exact, size = ref.with_grads(t, scale, dout, dlast), ref.magnitudes(t, scale, dout, dlast)
    for n, x in got.items():
        ref.check(x, exact[n], size[n], dtype, n, whole_row=n == "dlog_decay")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype):
    _say(f"linear attention gradients {shape} {dtype}")
    t = _inputs(100 + sum(shape), *shape, dtype)
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(5)).to(dtype)
    scale = shape[4] ** -0.5
    _check_all(_grads(t, scale, dout), t, scale, dout, None, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(2, 1, 1, 2, 16, 16), (1, 100, 2, 4, 64, 64), (1, 300, 1, 2, 128, 40), (1, 520, 1, 1, 40, 128)])
def test_states_and_their_gradients(shape, dtype):
    _say(f"linear attention states {shape} {dtype}")
    t = _inputs(200 + sum(shape), *shape, dtype, states=True)
    r = torch.Generator().manual_seed(6)
    dout = torch.randn(t["v"].shape, generator=r).to(dtype)
    dlast = torch.randn(t["initial_state"].shape, generator=r)
    _check_all(_grads(t, 0.7, dout, dlast), t, 0.7, dout, dlast, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("L", [1024, 1025, 1500])
def test_segments(dtype, L):
    """Few heads and a long row: cut into segments. The states' gradients cross them both ways."""
    _say(f"linear attention segments {L} {dtype}")
    t = _inputs(300 + L, 1, L, 1, 2, 64, 64, dtype, states=True)
    r = torch.Generator().manual_seed(7)
    dout, dlast = torch.randn(t["v"].shape, generator=r).to(dtype), torch.randn(1, 2, 64, 64, generator=r)
    _check_all(_grads(t, 0.125, dout, dlast), t, 0.125, dout, dlast, dtype)


@pytest.mark.parametrize("gdtype", [F32, BF16, F16])
@pytest.mark.parametrize("L", [3, 300])
def test_decay_per_head(gdtype, L):
    _say(f"linear attention, a decay per head {gdtype} {L}")
    t = _inputs(400 + L, 2, L, 1, 3, 32, 48, BF16, gdtype=gdtype, per_head=True)
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(8)).to(BF16)
    got = _grads(t, 0.2, dout)
    assert got["dlog_decay"].shape == (3,) and got["dlog_decay"].dtype == gdtype
    _check_all(got, t, 0.2, dout, None, BF16)


def test_strided_views():
    """q, k and v as slices of one projection (aligned and not), log_decay transposed, dout expanded."""
    _say("linear attention strided")
    from motif_mamba_amd import linear_attention_fn
    for off in (0, 8, 3):
        b, L, G, H, dk, dv = 2, 70, 2, 4, 32, 64
        r = torch.Generator().manual_seed(9)
        wide = torch.randn(b, L, off + 2 * G * dk + H * dv, generator=r).to(BF16).to(DEV)
        q, k, v = wide[..., off:].split([G * dk, G * dk, H * dv], -1)
        t = {"q": q.unflatten(-1, (G, dk)), "k": k.unflatten(-1, (G, dk)), "v": v.unflatten(-1, (H, dv)),
             "log_decay": (-torch.rand(b, H, L, generator=r)).to(DEV).transpose(1, 2)}
        want = {n: x.clone().contiguous() for n, x in t.items()}
        assert torch.equal(linear_attention_fn(**t), linear_attention_fn(**want))
        leaves = {n: x.detach().requires_grad_(True) for n, x in t.items()}
        dout = torch.randn(b, 1, H, dv, generator=r).to(BF16).to(DEV).expand(b, L, H, dv)
        got = torch.autograd.grad(linear_attention_fn(**leaves), list(leaves.values()), dout)
        leaves = {n: x.detach().requires_grad_(True) for n, x in want.items()}
        exp = torch.autograd.grad(linear_attention_fn(**leaves), list(leaves.values()), dout.contiguous())
        for n, x, y in zip(leaves, got, exp):
            assert torch.equal(x, y), n


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forgotten_states(dtype):
    """-inf starts a new document: nothing crosses it, forward or backward, whatever stands before."""
    _say(f"linear attention -inf {dtype}")
    t = _inputs(500, 1, 150, 1, 2, 32, 32, dtype, states=True)
    t["log_decay"][:, [0, 17, 18, 64, 100, 149]] = float("-inf")
    t["log_decay"][:, 40] = -1000.0
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(10)).to(dtype)
    got = _grads(t, 0.3, dout)
    exact, size = ref.with_grads(t, 0.3, dout), ref.magnitudes(t, 0.3, dout)
    for n, x in got.items():
        # autograd's gradient of exp at -inf is 0 * terms: 0 as well
        ref.check(x, torch.nan_to_num(exact[n], nan=0.0), size[n], dtype, n, whole_row=n == "dlog_decay")
    assert not got["dinitial_state"].any()
    for n in (0, 17, 18, 64, 100, 149, 40):
        assert not got["dlog_decay"][:, n].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_unseen_values_do_not_matter(dtype, bad, which):
    """Padding behind the last real token may hold anything: the tokens before it see none of it."""
    _say(f"linear attention unseen {bad} in {which} {dtype}")
    from motif_mamba_amd import linear_attention_fn
    for at in (1, 21, 63, 64, 75):
        t = _inputs(600, 1, 90, 1, 2, 64, 64, dtype)
        clean = linear_attention_fn(**_to(t))
        t[which][:, at:at + 3] = bad
        out = linear_attention_fn(**_to(t))
        assert torch.equal(out[:, :at], clean[:, :at]), at
        assert not torch.isfinite(out[:, at]).any(), at
        # one column of v: the others of that head stay finite
        t = _inputs(600, 1, 90, 1, 2, 64, 64, dtype)
        t["v"][:, at, 0, 5] = bad
        out = linear_attention_fn(**_to(t))
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[:, at:, 0, 5] = False
        assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_later_tokens_do_not_see_an_earlier_gradient(dtype):
    """An infinite dout reaches the tokens before it, not the ones behind."""
    _say(f"linear attention infinite dout {dtype}")
    t = _inputs(700, 1, 90, 1, 1, 64, 64, dtype)
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(11)).to(dtype)
    clean = _grads(t, 0.125, dout)
    for at in (3, 20, 64):
        d = dout.clone()
        d[:, at] = float("inf")
        got = _grads(t, 0.125, d)
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:, at + 1:], clean[n][:, at + 1:]), (n, at)
        assert torch.equal(got["dq"][:, :at], clean["dq"][:, :at])


def test_same_bits():
    """No atomics: a second call gives the same bits, and so does a graph's replay."""
    _say("linear attention same bits, graph")
    from motif_mamba_amd import linear_attention_fn
    t = _inputs(800, 2, 300, 1, 4, 64, 64, BF16, states=True)
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(12)).to(BF16)
    dlast = torch.randn(t["initial_state"].shape)
    first, second = _grads(t, 0.2, dout, dlast), _grads(t, 0.2, dout, dlast)
    for n in first:
        assert torch.equal(first[n], second[n]), n
    leaves = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
    d1, d2 = dout.to(DEV), dlast.to(DEV)

    def step():
        out, last = linear_attention_fn(**leaves, scale=0.2, return_last_state=True)
        return (out, last, *torch.autograd.grad([out, last], list(leaves.values()), [d1, d2]))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, first.values()):
            assert torch.equal(x, y)
        _grads(t, 0.2, dout)


def test_against_differences():
    """The gradients against central differences of the kernel's own forward, float32."""
    _say("linear attention differences")
    from motif_mamba_amd import linear_attention_fn
    t = _to(_inputs(900, 1, 40, 1, 2, 8, 8, F32, states=True))
    r = torch.Generator().manual_seed(13)
    dout, dlast = torch.randn(1, 40, 2, 8, generator=r).to(DEV), torch.randn(1, 2, 8, 8, generator=r).to(DEV)

    def loss(u):
        out, last = linear_attention_fn(**u, scale=0.5, return_last_state=True)
        return (out.double() * dout.double()).sum() + (last.double() * dlast.double()).sum()

    leaves = {n: x.clone().requires_grad_(True) for n, x in t.items()}
    out, last = linear_attention_fn(**leaves, scale=0.5, return_last_state=True)
    grads = torch.autograd.grad([out, last], list(leaves.values()), [dout, dlast])
    for (n, x), g in zip(t.items(), grads):
        way = torch.randn(x.shape, generator=r).to(DEV)
        h = 1e-3 if n == "log_decay" else 1e-2
        diff = (loss({**t, n: x + h * way}) - loss({**t, n: x - h * way})).item() / (2 * h)
        want = (g.double() * way.double()).sum().item()
        # The difference's own error: third derivatives (none for the bilinear ones) and float32 outputs, 3,000 terms.
        assert abs(diff - want) <= 2e-3 * max(1.0, (g.double() * way.double()).abs().sum().item()), n


@pytest.mark.parametrize("L", [0])
def test_empty(L):
    _say("linear attention empty")
    from motif_mamba_amd import linear_attention_fn
    t = _to(_inputs(1000, 2, L, 1, 2, 8, 8, BF16, states=True))
    out, last = linear_attention_fn(**t, return_last_state=True)
    assert out.shape == (2, 0, 2, 8) and torch.equal(last, t["initial_state"])
    t.pop("initial_state")
    out, last = linear_attention_fn(**t, return_last_state=True)
    assert not last.any()
    leaves = {n: x.requires_grad_(True) for n, x in _to(_inputs(1001, 2, L, 1, 2, 8, 8, BF16, states=True)).items()}
    out, last = linear_attention_fn(**leaves, return_last_state=True)
    dlast = torch.randn_like(last)
    g = torch.autograd.grad([last], list(leaves.values()), [dlast], allow_unused=True)
    assert torch.equal(g[4], dlast) and g[0].shape == (2, 0, 1, 8)
    empty = _to(_inputs(1002, 0, 5, 1, 2, 8, 8, BF16))
    assert linear_attention_fn(**empty).shape == (0, 5, 2, 8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 1, 2, 16, 16), (2, 2, 4, 128, 64), (1, 1, 3, 37, 50), (2, 1, 2, 64, 128), (1, 1, 2, 30, 6)])
def test_update(shape, dtype):
    _say(f"linear attention update {shape} {dtype}")
    from motif_mamba_amd import linear_attention_update
    b, G, H, dk, dv = shape
    t = _inputs(1100 + sum(shape), b, 3, G, H, dk, dv, dtype, states=True)
    scale = 0.3
    state = t["initial_state"].to(DEV)
    for n in range(3):
        u = {m: (x[:, :n + 1] if m != "initial_state" else x) for m, x in t.items()}
        exact, size = ref.with_grads(u, scale), ref.magnitudes(u, scale)
        out = linear_attention_update(state, *(t[m][:, n].to(DEV) for m in ("q", "k", "v", "log_decay")), scale=scale)
        ref.check(out, exact["out"][:, n], size["out"][:, n], F32, "out")
        ref.check(state, exact["last_state"], size["last_state"], F32, "state")


def test_update_strided_state_and_forgetting():
    """A slot of a larger cache, rows off 16 bytes, decay per head, -inf."""
    _say("linear attention update strided")
    from motif_mamba_amd import linear_attention_update
    for wide, off in ((70, 3), (72, 4)):
        r = torch.Generator().manual_seed(14)
        cache = torch.randn(5, 2, 20, wide, generator=r).to(DEV)
        before = cache.clone()
        state = cache[1:3, :, :16, off:off + 64]
        q, k, v = (torch.randn(2, n, d, generator=r).to(BF16).to(DEV) for n, d in ((1, 16), (1, 16), (2, 64)))
        g = torch.tensor([-0.5, float("-inf")], device=DEV)
        want = state.clone()
        out2 = linear_attention_update(want, q, k, v, g)
        out = linear_attention_update(state, q, k, v, g)
        assert torch.equal(out, out2) and torch.equal(state, want)
        inside = torch.zeros_like(cache, dtype=torch.bool)
        inside[1:3, :, :16, off:off + 64] = True
        assert torch.equal(cache[~inside], before[~inside])
        kv = k.float().unsqueeze(-1) * v.float().unsqueeze(-2)
        assert torch.equal(state[:, 1], kv[:, 1])


def test_prompt_then_tokens():
    """The prompt's last state continued token by token gives the whole sequence's outputs."""
    _say("linear attention prompt then tokens")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    t = _inputs(1200, 2, 80, 1, 3, 64, 32, BF16)
    exact, size = ref.with_grads(t, 0.125), ref.magnitudes(t, 0.125)
    d = _to(t)
    out, state = linear_attention_fn(**{n: x[:, :70] for n, x in d.items()}, return_last_state=True)
    for n in range(70, 80):
        y = linear_attention_update(state, *(d[m][:, n] for m in ("q", "k", "v", "log_decay")))
        ref.check(y, exact["out"][:, n], size["out"][:, n], BF16, f"token {n}")


def test_another_stream():
    _say("linear attention on another stream")
    from motif_mamba_amd import linear_attention_fn
    t = _to(_inputs(1300, 1, 1200, 1, 2, 64, 64, BF16))
    want = linear_attention_fn(**t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = linear_attention_fn(**t)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    _say("linear attention refusals")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    t = _to(_inputs(1400, 1, 8, 2, 4, 16, 16, BF16, states=True))

    def no(error, **over):
        with pytest.raises(error):
            linear_attention_fn(**{**t, **over})

    no(ValueError, v=t["v"][0])
    no(RuntimeError, q=t["q"].float())
    no(RuntimeError, k=t["k"][..., :8])
    no(RuntimeError, v=t["v"][:, :, :3])
    no(RuntimeError, v=t["v"][:, :4])
    no(RuntimeError, q=t["q"].cpu())
    no(RuntimeError, q=t["q"].double(), k=t["k"].double(), v=t["v"].double())
    no(RuntimeError, log_decay=t["log_decay"][..., :3])
    no(ValueError, log_decay=t["log_decay"][0, 0, :3])
    no(RuntimeError, log_decay=t["log_decay"].double())
    no(RuntimeError, initial_state=t["initial_state"].to(BF16))
    no(RuntimeError, initial_state=t["initial_state"][:, :2])
    wide = torch.zeros(1, 8, 2, 136, dtype=BF16, device=DEV)
    no(NotImplementedError, q=wide, k=wide, initial_state=None)
    u = {n: x[:, 0] for n, x in t.items() if n != "initial_state"}
    for bad in (t["initial_state"].to(BF16), t["initial_state"][:, :2], t["initial_state"].transpose(2, 3)[..., ::2, :]):
        with pytest.raises(RuntimeError):
            linear_attention_update(bad, **u)
    with pytest.raises(RuntimeError):
        linear_attention_update(t["initial_state"].transpose(2, 3), **u)
    with pytest.raises(ValueError):
        linear_attention_update(t["initial_state"], u["q"], u["k"], t["v"], u["log_decay"])


def test_many_short_rows():
    """More (batch row, head) pairs than one grid dimension of 65,535 holds."""
    _say("linear attention 70,000 pairs")
    from motif_mamba_amd import linear_attention_fn, linear_attention_update
    t = _inputs(1500, 17500, 3, 1, 4, 8, 8, BF16)
    d = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
    dout = torch.randn(t["v"].shape, generator=torch.Generator().manual_seed(16)).to(BF16)
    out = linear_attention_fn(**d, scale=0.4)
    got = dict(zip(["d" + n for n in d], torch.autograd.grad(out, list(d.values()), dout.to(DEV))), out=out)
    _check_all(got, t, 0.4, dout, None, BF16)
    state = torch.zeros(17500, 4, 8, 8, device=DEV)
    y = linear_attention_update(state, *(d[n].detach()[:, 0] for n in ("q", "k", "v", "log_decay")), scale=0.4)
    exact, size = ref.with_grads({n: x[:, :1] for n, x in t.items()}, 0.4), ref.magnitudes({n: x[:, :1] for n, x in t.items()}, 0.4)
    ref.check(y, exact["out"][:, 0], size["out"][:, 0], F32, "out")


def test_no_second_derivative():
    _say("linear attention, group norm: second derivatives refused")
    from motif_mamba_amd import group_norm_fn, linear_attention_fn
    t = {n: x.to(DEV).requires_grad_(True) for n, x in _inputs(1600, 1, 4, 1, 1, 8, 8, F32).items()}
    (g,) = torch.autograd.grad(linear_attention_fn(**t).sum(), [t["q"]], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(group_norm_fn(x, 2).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
