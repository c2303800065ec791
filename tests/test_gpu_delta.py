"""GPU tests of the gated delta rule (mm_delta.hip, mm_delta_api.hip) against the recurrence in float64: lengths around the chunk,
head sizes and layouts, states, forgotten states, infinities, gradients, single tokens, graphs, refusals. Bounds: tests/delta_ref.py."""
import sys

import pytest
import torch

from tests import delta_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def case(seed, b, L, H, G, dk, dv, dtype, decay="token", beta=1.0, states=True, gdtype=F32):
    r = torch.Generator().manual_seed(seed)
    t = {"q": _unit(torch.randn(b, L, G, dk, generator=r)).to(dtype), "k": _unit(torch.randn(b, L, G, dk, generator=r)).to(dtype),
         "v": torch.randn(b, L, H, dv, generator=r).to(dtype), "beta": (beta * torch.rand(b, L, H, generator=r)).to(gdtype)}
    if decay == "token":
        t["log_decay"] = (-0.2 * torch.rand(b, L, H, generator=r) ** 2).to(gdtype)
    elif decay == "head":
        t["log_decay"] = (-0.1 * torch.rand(H, generator=r)).to(gdtype)
    if states:
        t["initial_state"] = torch.randn(b, H, dk, dv, generator=r)
    return t


def _dev(t, grad=False):
    return {n: x.to(DEV).requires_grad_(grad) for n, x in t.items()}


def _forward(t, one_key=False, **kw):
    from motif_mamba_amd import delta_rule_fn
    _, L, _, dk = t["q"].shape
    exact = ref.with_grads(t, kw.get("scale", dk ** -0.5))
    out, last = delta_rule_fn(**_dev(t), return_last_state=True, **kw)
    for n, x in (("out", out), ("last_state", last)):
        ref.check(x, exact[n], t["v"].dtype, dk, L, n, one_key)


def _backward(t, seed, dlast=True, one_key=False, **kw):
    from motif_mamba_amd import delta_rule_fn
    _, L, _, dk = t["q"].shape
    r = torch.Generator().manual_seed(seed)
    dout = torch.randn(t["v"].shape, generator=r).to(t["v"].dtype)
    b, _, H, dv = t["v"].shape
    dl = torch.randn(b, H, dk, dv, generator=r) if dlast else None
    exact = ref.with_grads(t, kw.get("scale", dk ** -0.5), dout, dl)
    d = _dev(t, True)
    outs = delta_rule_fn(**d, return_last_state=dlast, **kw)
    outs, douts = ((list(outs), [dout.to(DEV), dl.to(DEV)]) if dlast else ([outs], [dout.to(DEV)]))
    got = dict(zip(["d" + n for n in d], torch.autograd.grad(outs, list(d.values()), douts)), out=outs[0])
    for n, x in got.items():
        assert x.dtype == (t[n[1:]].dtype if n != "out" else t["v"].dtype)
        ref.check(x, exact[n], t["v"].dtype, dk, L, n, one_key)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 129, 200])
def test_lengths(L, dtype):
    _say(f"delta L {L} {dtype}")
    _forward(case(L, 2, L, 4, 2, 64, 64, dtype))
    _backward(case(L, 2, L, 2, 2, 32, 48, dtype), L)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 128), (16, 16), (17, 33), (40, 48), (64, 80), (65, 64), (96, 96), (100, 37), (127, 127), (128, 128)])
def test_sizes(dk, dv, dtype):
    _say(f"delta sizes {dk} {dv} {dtype}")
    _forward(case(dk, 2, 70, 2, 1, dk, dv, dtype, beta=2.0))
    _backward(case(dv, 1, 70, 3, 3, dk, dv, dtype, beta=2.0), dk)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decay", ["none", "head", "token"])
@pytest.mark.parametrize("states", [False, True])
def test_decays_and_states(decay, states, dtype):
    _say(f"delta decay {decay} states {states} {dtype}")
    t = case(3, 2, 90, 4, 2, 48, 64, dtype, decay=decay, states=states)
    _forward(t)
    _backward(t, 5, dlast=states)


@pytest.mark.parametrize("gdtype", [BF16, F16])
def test_gate_types(gdtype):
    _say(f"delta gate types {gdtype}")
    t = case(4, 2, 70, 4, 1, 32, 32, F32, gdtype=gdtype)
    _forward(t)
    _backward(t, 6)
    _backward(case(5, 2, 70, 4, 1, 32, 32, BF16, decay="head", gdtype=gdtype), 7)


@pytest.mark.parametrize("H,G", [(1, 1), (5, 1), (6, 2), (8, 8), (12, 3)])
def test_groups(H, G):
    _say(f"delta groups {H} {G}")
    _backward(case(H, 2, 67, H, G, 64, 64, BF16), H)
    _backward(case(H, 1, 40, H, G, 30, 30, F16), H)


def test_scale_and_betas_at_their_ends():
    """beta 0 leaves the state alone, 1 puts v under k, 2 reflects."""
    _say("delta betas")
    t = case(8, 1, 80, 3, 1, 32, 40, F32)
    t["beta"][..., 0], t["beta"][..., 1], t["beta"][..., 2] = 0.0, 1.0, 2.0
    _forward(t, scale=0.3)
    _backward(t, 9, scale=-1.5)


def test_same_key_throughout():
    """Every token corrects the same row: the triangles' entries are as large as they get."""
    _say("delta one key")
    for beta in (1.0, 2.0):
        t = case(10, 1, 130, 2, 1, 64, 64, F32, decay="none")
        t["k"] = t["k"][:, :1].expand_as(t["k"]).contiguous()
        t["beta"] = torch.full_like(t["beta"], beta)
        _forward(t, one_key=True)
        _backward(t, 11, one_key=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forgotten_states(dtype):
    """-inf marks a document's first token: outputs and gradients of packed documents are those of each alone, and a document that
    overflows leaves the one before it alone."""
    _say(f"delta documents {dtype}")
    from motif_mamba_amd import delta_rule_fn
    t = case(12, 1, 150, 2, 1, 64, 64, dtype, states=False)
    cuts = [0, 5, 6, 64, 100, 150]
    for c in cuts[1:-1]:
        t["log_decay"][:, c] = float("-inf")
    _forward(t)
    r = torch.Generator().manual_seed(13)
    dout = torch.randn(t["v"].shape, generator=r).to(dtype).to(DEV)
    d = _dev(t, True)
    got = torch.autograd.grad(delta_rule_fn(**d), list(d.values()), dout)
    for a, b in zip(cuts, cuts[1:]):
        e = {n: x[:, a:b].detach().clone().requires_grad_(True) for n, x in d.items()}
        alone = torch.autograd.grad(delta_rule_fn(**e), list(e.values()), dout[:, a:b])
        for n, x, y in zip(d, got, alone):
            want = y.clone()
            if n == "log_decay":
                want[:, 0] = 0 if a else want[:, 0]
                assert not x[:, a].any() or a == 0
            err, m = (x[:, a:b].double() - want.double()).abs().max(), want.double().abs().max()
            # the same sums, grouped by other chunks; 16-bit results may round either way
            assert err <= (2 * ref.ROUND[x.dtype] + 2 ** -24 * 4 * 192 * 4) * m + 1e-30, (n, a, err, m)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_infinities_and_nan(dtype):
    """An input that is not finite changes what the recurrence says it changes, and nothing before it."""
    _say(f"delta not finite {dtype}")
    from motif_mamba_amd import delta_rule_fn
    inf, nan = float("inf"), float("nan")
    for name, at, bad in (("v", (0, 40, 1, 7), inf), ("v", (0, 70, 0, 3), nan), ("q", (0, 66, 0, 0), inf), ("q", (0, 1, 0, 5), nan),
                          ("k", (0, 50, 0, 9), nan), ("k", (0, 99, 0, 2), inf), ("beta", (0, 80, 1), nan), ("log_decay", (0, 33, 0), nan),
                          ("initial_state", (0, 1, 4, 5), -inf), ("log_decay", (0, 90, 1), inf)):
        t = case(14, 1, 100, 2, 1, 32, 24, dtype)
        t[name][at] = bad
        with torch.no_grad():
            exact = ref.recurrence(*(t[n].double() for n in ref.NAMES[:5]), 32 ** -0.5, t["initial_state"].double())
        got = delta_rule_fn(**_dev(t), return_last_state=True)
        for what, g, e in zip(("out", "last_state"), got, exact):
            g = g.cpu().double()
            if what == "out":
                assert torch.isfinite(g[:, :at[1] if name != "initial_state" else 0]).all()
            fin = torch.isfinite(e)
            assert torch.equal(torch.isnan(g), torch.isnan(e)), (name, what, torch.isnan(g).sum(), torch.isnan(e).sum())
            assert torch.equal(g[~fin & ~torch.isnan(e)], e[~fin & ~torch.isnan(e)]), (name, what)
            m = e[fin].abs().max() if fin.any() else 0.0
            assert ((g - e)[fin].abs() <= ref.ROUND[got[0].dtype] * e[fin].abs() + 4 * 1024 * 2 ** -24 * m).all(), (name, what)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (100, 72), (66, 33), (64, 128)])
def test_infinities_of_larger_heads(dk, dv, dtype):
    """As above, several at once, in whole and broken 16-byte pieces, of rows beside others that stay as they were."""
    _say(f"delta not finite {dk} {dv} {dtype}")
    from motif_mamba_amd import delta_rule_fn
    inf, nan = float("inf"), float("nan")
    plain = case(53, 2, 150, 2, 1, dk, dv, dtype)
    before = delta_rule_fn(**_dev(plain), return_last_state=True)
    t = {n: x.clone() for n, x in plain.items()}
    t["v"][0, 40, 1, 7] = inf
    t["v"][0, 130, 1, dv - 1] = -inf
    t["beta"][1, 149, 0] = nan
    t["initial_state"][1, 1, dk - 1, dv - 1] = inf
    with torch.no_grad():
        exact = ref.recurrence(*(t[n].double() for n in ref.NAMES[:5]), dk ** -0.5, t["initial_state"].double())
    got = delta_rule_fn(**_dev(t), return_last_state=True)
    assert torch.equal(got[0][0, :, 0], before[0][0, :, 0]) and torch.equal(got[1][0, 0], before[1][0, 0])
    assert torch.equal(got[0][1, :128, 0], before[0][1, :128, 0])   # (the chunks before its own, which goes token by token)
    for what, g, e in zip(("out", "last_state"), got, exact):
        g = g.cpu().double()
        fin = torch.isfinite(e)
        assert torch.equal(torch.isnan(g), torch.isnan(e)), (what, torch.isnan(g).sum(), torch.isnan(e).sum())
        assert torch.equal(g[~fin & ~torch.isnan(e)], e[~fin & ~torch.isnan(e)]), what
        assert ((g - e)[fin].abs() <= ref.ROUND[got[0].dtype] * e[fin].abs() + 4 * 1024 * 2 ** -24 * e[fin].abs().max()).all(), what


def test_one_row_s_values_stay_in_it():
    """NaN in one (batch row, head) reaches no other's outputs or gradients."""
    _say("delta NaN of another row")
    from motif_mamba_amd import delta_rule_fn
    t = case(15, 2, 100, 2, 2, 32, 32, BF16)
    dout = torch.randn(t["v"].shape).to(BF16).to(DEV)
    res = []
    for bad in (False, True):
        x = {n: y.clone() for n, y in t.items()}
        if bad:
            x["v"][1, 50, 0] = float("nan")
        d = _dev(x, True)
        out = delta_rule_fn(**d)
        res.append([out, *torch.autograd.grad(out, list(d.values()), dout)])
    for a, b, n in zip(*res, ["out", *t]):
        for i, h in ((0, 0), (0, 1), (1, 1)):
            x, y = ((z[i, h] if n == "initial_state" else z[i, :, h]) for z in (a, b))
            assert torch.equal(x, y), (n, i, h)
        # dv and the state's gradient hold nothing of v: outputs are linear in both together.
        assert torch.isnan(b[1]).any() or n in ("v", "initial_state")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("segs", [1, 2, 3, 7])
def test_segments(segs, dtype, monkeypatch):
    """Rows cut into segments, the last one shorter or of one token: outputs, states and gradients as without; heads of a group, one
    decay per head, no initial state."""
    _say(f"delta segments {segs} {dtype}")
    monkeypatch.setenv("MM_DELTA_SEGMENTS", str(segs))
    for L, dk, dv in ((449, 64, 48), (300, 128, 128), (200, 100, 72), (33, 16, 16)):
        _forward(case(segs, 1, L, 2, 1, dk, dv, dtype))
        _backward(case(dk, 2, L, 2, 1, dk, dv, dtype), L)
    t = case(44, 1, 257, 3, 3, 40, 40, dtype, decay="head", states=False)
    _forward(t)
    _backward(t, 45, dlast=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_segments_kept_and_computed_again(dtype, monkeypatch):
    """The backward gives the same bits with the forward's segment states as without them."""
    _say(f"delta kept segments {dtype}")
    from motif_mamba_amd._native import ext
    monkeypatch.setenv("MM_DELTA_SEGMENTS", "4")
    d = _dev(case(46, 2, 300, 2, 2, 64, 64, dtype))
    args = [d[n] for n in ref.NAMES[:5]] + [0.125, d["initial_state"]]
    *_, kept = ext().delta_fwd(*args, True, True)
    dout, dlast = torch.randn_like(d["v"]), torch.randn_like(d["initial_state"])
    a, b = (ext().delta_bwd(*args, dout, dlast, s, False, True, True) for s in (kept, None))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    monkeypatch.setenv("MM_DELTA_SEGMENTS", "5")
    with pytest.raises(RuntimeError, match="segment_states"):
        ext().delta_bwd(*args, dout, dlast, kept, False, True, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("segs", [2, 5])
def test_segments_not_finite(segs, dtype, monkeypatch):
    """As test_infinities_and_nan, in every segment, of one (batch row, head) beside others that stay as they were."""
    _say(f"delta segments not finite {segs} {dtype}")
    from motif_mamba_amd import delta_rule_fn
    monkeypatch.setenv("MM_DELTA_SEGMENTS", str(segs))
    inf, nan = float("inf"), float("nan")
    plain = case(47, 1, 330, 2, 1, 32, 24, dtype)
    before = delta_rule_fn(**_dev(plain), return_last_state=True)
    for name, at, bad in (("v", (0, 3, 1, 7), inf), ("v", (0, 200, 1, 7), nan), ("v", (0, 329, 1, 7), inf), ("beta", (0, 170, 1), nan), ("beta", (0, 70, 1), inf),
                          ("log_decay", (0, 100, 1), nan), ("log_decay", (0, 290, 1), inf), ("log_decay", (0, 2, 1), inf), ("initial_state", (0, 1, 4, 5), -inf),
                          ("initial_state", (0, 1, 4, 5), nan)):
        t = {n: x.clone() for n, x in plain.items()}
        t[name][at] = bad
        with torch.no_grad():
            exact = ref.recurrence(*(t[n].double() for n in ref.NAMES[:5]), 32 ** -0.5, t["initial_state"].double())
        got = delta_rule_fn(**_dev(t), return_last_state=True)
        assert torch.equal(got[0][:, :, 0], before[0][:, :, 0]) and torch.equal(got[1][:, 0], before[1][:, 0]), name
        for what, g, e in zip(("out", "last_state"), got, exact):
            g = g.cpu().double()
            fin = torch.isfinite(e)
            assert torch.equal(torch.isnan(g), torch.isnan(e)), (name, what, torch.isnan(g).sum(), torch.isnan(e).sum())
            assert torch.equal(g[~fin & ~torch.isnan(e)], e[~fin & ~torch.isnan(e)]), (name, what)
            m = e[fin].abs().max() if fin.any() else 0.0
            assert ((g - e)[fin].abs() <= ref.ROUND[got[0].dtype] * e[fin].abs() + 4 * 1024 * 2 ** -24 * m).all(), (name, what)


def test_segments_in_a_graph(monkeypatch):
    _say("delta segments graph")
    from motif_mamba_amd import delta_rule_fn
    monkeypatch.setenv("MM_DELTA_SEGMENTS", "3")
    t = case(48, 1, 400, 2, 1, 64, 64, BF16)
    d = _dev(t)
    dout = torch.randn(t["v"].shape).to(BF16).to(DEV)

    def go():
        x = {n: y.detach().requires_grad_(True) for n, y in d.items()}
        out, last = delta_rule_fn(**x, return_last_state=True)
        return [out, last, *torch.autograd.grad([out, last], list(x.values()), [dout, d["initial_state"]])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = go()
    for i in range(3):
        r = torch.Generator().manual_seed(50 + i)
        d["v"].copy_(torch.randn(t["v"].shape, generator=r))
        if i == 1:
            d["v"][0, 5, 1] = float("inf")   # the row goes in one piece, and in segments again after that
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in res]
        want = go()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(torch.nan_to_num(x.float(), 7.0), torch.nan_to_num(y.float(), 7.0)), i


def test_backward_twice_and_two_streams(monkeypatch):
    """A graph that is kept gives the same gradients again, and calls on two streams at once each their own."""
    _say("delta backward twice")
    from motif_mamba_amd import delta_rule_fn
    monkeypatch.setenv("MM_DELTA_SEGMENTS", "3")
    cases = [_dev(case(seed, 2, 500, 4, 2, 64, 128, BF16), True) for seed in (54, 55)]
    dout = torch.randn(cases[0]["v"].shape).to(BF16).to(DEV)

    def go(d):
        out, last = delta_rule_fn(**d, return_last_state=True)
        return [torch.autograd.grad([out, last], list(d.values()), [dout, d["initial_state"].detach()], retain_graph=True) for _ in range(2)]

    alone = []
    for d in cases:
        one, two = go(d)
        for x, y in zip(one, two):
            assert torch.equal(x, y)
        alone.append(one)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for s, d in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append([go(d) for _ in range(3)])
    torch.cuda.synchronize()
    for runs, want in zip(got, alone):
        for pair in runs:
            for grads in pair:
                for x, y in zip(grads, want):
                    assert torch.equal(x, y)


def test_a_token_that_sees_no_other():
    """Its decay has no gradient at all, and the state before it has none of what comes after a forgotten one."""
    _say("delta lone token")
    from motif_mamba_amd import delta_rule_fn
    for dtype in (BF16, F16, F32):
        d = _dev(case(49, 2, 1, 2, 1, 64, 64, dtype, states=False), True)
        (g,) = torch.autograd.grad(delta_rule_fn(**d).float().sum(), [d["log_decay"]])
        assert not g.any()
        t = case(51, 1, 90, 2, 1, 64, 64, dtype)
        t["log_decay"][:, 40] = float("-inf")
        d = _dev(t, True)
        out = delta_rule_fn(**d)
        (s,) = torch.autograd.grad(out[:, 40:].float().sum(), [d["initial_state"]])
        assert not s.any()


def test_update_many_pairs():
    """Pairs by the hundred thousand, more than fill the card several times over: each as alone."""
    _say("delta update many pairs")
    from motif_mamba_amd import delta_rule_update
    for dk, dv in ((8, 16), (16, 40), (8, 72)):
        t = {n: x[:, 0] if n != "initial_state" else x for n, x in _dev(case(52, 4, 1, 3, 1, dk, dv, F32)).items()}
        one = t["initial_state"].clone()
        out = delta_rule_update(one, *(t[n] for n in ref.NAMES[:5]))
        many = t["initial_state"].repeat(20000, 1, 1, 1)
        outs = delta_rule_update(many, *(t[n].repeat(20000, *[1] * (t[n].dim() - 1)) for n in ref.NAMES[:5]))
        assert torch.equal(outs, out.repeat(20000, 1, 1)) and torch.equal(many, one.repeat(20000, 1, 1, 1))


def test_layouts():
    """Slices of one projection, aligned and not, a transposed batch, one beta and decay for all tokens: the same values."""
    _say("delta layouts")
    from motif_mamba_amd import delta_rule_fn
    r = torch.Generator().manual_seed(16)
    b, L, H, G, dk, dv = 2, 75, 4, 2, 32, 24
    for off in (0, 1):
        wide = torch.randn(L, b, off + 2 * G * dk + H * dv, generator=r).to(BF16).to(DEV).transpose(0, 1)[..., off:]
        q, k, v = wide.split([G * dk, G * dk, H * dv], -1)
        q, k, v = (q * 0.15).unflatten(-1, (G, dk)), k.unflatten(-1, (G, dk)), v.unflatten(-1, (H, dv))
        wide[..., G * dk:2 * G * dk] *= 0.15
        beta, g = torch.rand(1, 1, H, generator=r).to(DEV).expand(b, L, H), -torch.rand(1, L, 1, generator=r).to(DEV).expand(b, L, H)
        res = []
        for f in (lambda x: x, lambda x: x.contiguous()):
            x = [f(y).detach().requires_grad_(True) for y in (q, k, v, beta, g)]
            out, last = delta_rule_fn(*x, return_last_state=True)
            res.append([out, last, *torch.autograd.grad([out, last], x, [f(v), torch.ones_like(last)])])
        for i, (x, y) in enumerate(zip(*res)):
            assert torch.allclose(x.float(), y.float(), rtol=2.0 ** -7, atol=1e-4 * y.float().abs().max().item()), i
        t = dict(zip(ref.NAMES, (y.cpu() for y in (q, k, v, beta, g))))
        ref.check(res[0][0], ref.with_grads(t, dk ** -0.5)["out"], BF16, dk, L, "out")


def test_far_tokens():
    """Tokens 2^22 elements apart and more are copied."""
    _say("delta far tokens")
    from motif_mamba_amd import delta_rule_fn
    t = case(17, 1, 3, 1, 1, 16, 16, F32)
    d = _dev(t)
    big = torch.zeros(3, 1 << 22, device=DEV)
    big[:, :16] = d["v"][0, :, 0]
    v = torch.as_strided(big, (1, 3, 1, 16), (1, 1 << 22, 1, 1))
    assert torch.equal(delta_rule_fn(**{**d, "v": v}), delta_rule_fn(**d))


def test_many_pairs():
    """More (batch row, head) pairs and chunks than a launch has workgroups."""
    _say("delta 70,000 pairs")
    from motif_mamba_amd import delta_rule_fn
    t = case(18, 7, 40, 2, 1, 16, 16, F32)
    d = _dev(t)
    many = {n: x.repeat(5000, *[1] * (x.dim() - 1)) for n, x in d.items()}
    for x in (d, many):
        for n in x:
            x[n].requires_grad_(True)
    res = []
    for x in (d, many):
        out, last = delta_rule_fn(**x, return_last_state=True)
        res.append([out, last, *torch.autograd.grad([out.sum() + last.sum()], list(x.values()))])
    for a, b in zip(*res):
        assert torch.equal(a.repeat(5000, *[1] * (a.dim() - 1)), b)


def test_long_row():
    _say("delta long row")
    t = case(19, 1, 3000, 1, 1, 32, 32, F32, states=False)
    _forward(t)
    _backward(t, 20, dlast=False)


def test_empty():
    _say("delta empty")
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = case(21, 2, 0, 2, 1, 16, 16, F32)
    d = _dev(t, True)
    out, last = delta_rule_fn(**d, return_last_state=True)
    assert out.shape == (2, 0, 2, 16) and torch.equal(last, d["initial_state"])
    (ds,) = torch.autograd.grad(last, [d["initial_state"]], torch.ones_like(last))
    assert torch.equal(ds, torch.ones_like(ds))
    d = {n: x[:0].detach().requires_grad_(True) for n, x in _dev(case(21, 2, 5, 2, 1, 16, 16, F32)).items()}
    out = delta_rule_fn(**d)
    assert out.shape == (0, 5, 2, 16)
    torch.autograd.grad(out.sum(), list(d.values()), allow_unused=True)
    q = torch.randn(2, 5, 1, 16, device=DEV, requires_grad=True)
    v = torch.zeros(2, 5, 0, 16, device=DEV, requires_grad=True)
    z = torch.zeros(2, 5, 0, device=DEV)
    out = delta_rule_fn(q, q, v, z, z)
    (dq,) = torch.autograd.grad(out, [q], torch.zeros_like(out))
    assert not dq.any()
    delta_rule_update(torch.zeros(0, 2, 16, 16, device=DEV), q[:0, 0].detach(), q[:0, 0].detach(), torch.zeros(0, 2, 16, device=DEV), torch.zeros(0, 2, device=DEV))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dk,dv", [(1, 1), (16, 32), (17, 30), (64, 64), (40, 80), (100, 37), (128, 128)])
@pytest.mark.parametrize("decay", ["token", "head", "none"])
def test_update(dk, dv, decay, dtype):
    """One token on a kept state, several in a row, against the recurrence."""
    _say(f"delta update {dk} {dv} {decay} {dtype}")
    from motif_mamba_amd import delta_rule_update
    t = case(dk + dv, 3, 4, 4, 2, dk, dv, dtype, decay=decay, beta=2.0)
    exact = ref.with_grads(t, dk ** -0.5)
    d = _dev(t)
    state = d["initial_state"].clone()
    outs = []
    for n in range(4):
        g = d["log_decay"] if decay == "head" else d["log_decay"][:, n] if decay == "token" else None
        outs.append(delta_rule_update(state, d["q"][:, n], d["k"][:, n], d["v"][:, n], d["beta"][:, n], g))
    ref.check(torch.stack(outs, 1), exact["out"], F32, dk, 4, "out")
    ref.check(state, exact["last_state"], F32, dk, 4, "last_state")


def test_update_states_of_other_strides():
    """A slice of a larger cache, rows of any alignment: what is not the state stays as it was."""
    _say("delta update strides")
    from motif_mamba_amd import delta_rule_update
    t = _dev(case(31, 3, 1, 4, 2, 20, 16, F32))
    args = [t[n][:, 0] for n in ("q", "k", "v", "beta", "log_decay")]
    plain = t["initial_state"].clone()
    out = delta_rule_update(plain, *args)
    for off, pitch in ((0, 16), (3, 19), (4, 24)):
        cache = torch.full((5, 4, 22, off + pitch), 7.0, device=DEV)
        view = cache[1:4, :, 1:21, off:off + 16]
        view.copy_(t["initial_state"])
        assert torch.equal(delta_rule_update(view, *args), out) and torch.equal(view, plain)
        view.fill_(7.0)
        assert (cache == 7.0).all()
    turned = t["initial_state"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(delta_rule_update(turned, *args), out) and torch.equal(turned, plain)


def test_update_infinities():
    _say("delta update not finite")
    from motif_mamba_amd import delta_rule_update
    inf = float("inf")
    for name, at, bad in (("v", (0, 0, 1, 7), inf), ("k", (0, 0, 0, 9), float("nan")), ("initial_state", (0, 1, 4, 5), -inf), ("log_decay", (0, 0, 0), -inf),
                          ("log_decay", (0, 0, 1), inf)):
        t = case(32, 1, 1, 2, 1, 32, 24, F32)
        t[name][at] = bad
        with torch.no_grad():
            e, es = ref.recurrence(*(t[n].double() for n in ref.NAMES[:5]), 32 ** -0.5, t["initial_state"].double())
        d = _dev(t)
        out = delta_rule_update(d["initial_state"], *(d[n][:, 0] for n in ref.NAMES[:5]))
        for g, x in ((out.cpu(), e[:, 0]), (d["initial_state"].cpu(), es)):
            assert torch.allclose(g.double(), x, rtol=1e-4, atol=1e-4, equal_nan=True), name


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 64), (24, 32), (40, 80), (64, 64), (65, 16), (100, 128), (128, 128)])
def test_infinite_growth(dk, dv, dtype):
    """An infinite decay factor under a negative beta: the state, what it gives and what a further token reads of it are infinite, and NaN
    only where the recurrence has one; rows that fill a head up to the kernel's size take no part."""
    _say(f"delta infinite growth {dk} {dv} {dtype}")
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = case(36, 1, 2, 2, 1, dk, dv, dtype)
    for n in ("q", "k", "initial_state"):
        t[n] = t[n].abs() + 0.25
    t["beta"] = -t["beta"] - 0.25
    t["initial_state"][0, 1] *= -1
    t["log_decay"][0, 0, 1] = t["log_decay"][0, 1, 0] = float("inf")
    with torch.no_grad():
        out, last = ref.recurrence(*(t[n].double() for n in ref.NAMES[:5]), dk ** -0.5, t["initial_state"].double())
    fin = torch.isfinite(out)
    assert torch.isinf(last).all() and fin[0, 0, 0].all() and fin.sum() == dv   # the first token of the head that grows at the second
    t["log_decay"][0, 1, 0] = 129.0   # counts as infinite
    d = _dev(t)
    state = d["initial_state"].clone()
    outs = [delta_rule_update(state, *(d[n][:, i] for n in ref.NAMES[:5])) for i in range(2)]
    for what, (o, s) in (("update", (torch.stack(outs, 1), state)), ("prompt", delta_rule_fn(**d, return_last_state=True))):
        o = o.cpu().double()
        assert torch.equal(s.cpu().double(), last) and torch.isfinite(o[fin]).all() and torch.equal(o[~fin], out[~fin]), what


def test_prompt_then_tokens():
    _say("delta prompt then tokens")
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = case(33, 2, 80, 4, 2, 64, 64, F32)
    d = _dev(t)
    exact = ref.with_grads(t, 64 ** -0.5)
    out, state = delta_rule_fn(**{n: x if n == "initial_state" else x[:, :70] for n, x in d.items()}, return_last_state=True)
    outs = [out] + [delta_rule_update(state, *(d[n][:, i] for n in ref.NAMES[:5])).unsqueeze(1) for i in range(70, 80)]
    ref.check(torch.cat(outs, 1), exact["out"], F32, 64, 80, "out")
    ref.check(state, exact["last_state"], F32, 64, 80, "last_state")


def test_against_differences():
    """The gradients against central differences of the kernels' own outputs along random ways."""
    _say("delta differences")
    from motif_mamba_amd import delta_rule_fn
    t = case(34, 1, 70, 2, 1, 16, 16, F32)
    r = torch.Generator().manual_seed(35)
    dout = torch.randn(t["v"].shape, generator=r).to(DEV).double()
    dl = torch.randn(t["initial_state"].shape, generator=r).to(DEV).double()
    d = _dev(t, True)

    def loss(x):
        out, last = delta_rule_fn(**x, return_last_state=True)
        return (out.double() * dout).sum() + (last.double() * dl).sum()

    grads = torch.autograd.grad(loss(d), list(d.values()))
    for (n, x), g in zip(d.items(), grads):
        way = torch.randn(x.shape, generator=r).to(DEV)
        with torch.no_grad():
            diff = (loss({**d, n: x + 1e-2 * way}) - loss({**d, n: x - 1e-2 * way})).item() / 2e-2
        # second-order differences: 1e-4 of a third derivative, some units of the terms' size
        terms = g.double() * way.double()
        assert abs(diff - terms.sum().item()) <= 2e-2 * max(1.0, terms.square().sum().sqrt().item()), n


def test_only_some_gradients():
    """Gradients of one input, of the last state alone, and of nothing."""
    _say("delta some gradients")
    from motif_mamba_amd import delta_rule_fn
    t = case(36, 1, 50, 2, 1, 32, 32, BF16)
    d = _dev(t, True)
    out, last = delta_rule_fn(**d, return_last_state=True)
    every = torch.autograd.grad(out.float().sum() + last.sum(), list(d.values()))
    for n, want in zip(t, every):
        x = {m: y.detach().requires_grad_(m == n) for m, y in d.items()}
        o, s = delta_rule_fn(**x, return_last_state=True)
        (got,) = torch.autograd.grad(o.float().sum() + s.sum(), [x[n]])
        assert torch.equal(got, want), n
    o, s = delta_rule_fn(**d, return_last_state=True)
    got = torch.autograd.grad(s.sum(), [d["v"], d["q"]])
    assert got[0].any() and not got[1].any()
    assert delta_rule_fn(**t_detached(d)).grad_fn is None


def t_detached(d):
    return {n: x.detach() for n, x in d.items()}


def test_same_bits_and_another_stream():
    _say("delta same bits")
    from motif_mamba_amd import delta_rule_fn
    t = case(37, 3, 150, 6, 2, 64, 128, BF16)
    dout = torch.randn(t["v"].shape).to(BF16).to(DEV)

    def go():
        d = _dev(t, True)
        out, last = delta_rule_fn(**d, return_last_state=True)
        return [out, last, *torch.autograd.grad([out, last], list(d.values()), [dout, torch.ones_like(last)])]

    a = go()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        b = go()
    with torch.cuda.stream(s2):
        c = go()
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_graph():
    """Forward, backward and the token's update captured and replayed, with eager work between the replays."""
    _say("delta graph")
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = case(38, 2, 100, 4, 1, 64, 64, BF16)
    d = _dev(t)
    state = torch.zeros_like(d["initial_state"])
    dout = torch.randn(t["v"].shape).to(BF16).to(DEV)

    def go():
        x = {n: y.detach().requires_grad_(True) for n, y in d.items()}
        out = delta_rule_fn(**x)
        grads = torch.autograd.grad(out, list(x.values()), dout)
        with torch.no_grad():
            tok = delta_rule_update(state, *(d[n][:, 0] for n in ref.NAMES[:5]))
        return [out, tok, state, *grads]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            go()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = go()
    for i in range(3):
        r = torch.Generator().manual_seed(40 + i)
        d["v"].copy_(torch.randn(t["v"].shape, generator=r))
        start = torch.randn(state.shape, generator=r).to(DEV)
        state.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in res]
        state.copy_(start)
        want = go()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y), i


def test_update_derivatives_and_version():
    _say("delta update derivatives")
    from torch.autograd import forward_ad
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = _dev(case(41, 2, 1, 2, 1, 16, 8, F32))
    args = {"state": t["initial_state"], **{n: t[n][:, 0].clone() for n in ref.NAMES[:5]}}
    for n in args:
        leaf = {**args, n: args[n].clone().requires_grad_(True)}
        with pytest.raises(RuntimeError, match="derivatives"):
            delta_rule_update(**leaf)
        with torch.no_grad():
            assert not delta_rule_update(**leaf).requires_grad
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="derivatives"):
            delta_rule_update(**{**args, n: forward_ad.make_dual(args[n], torch.ones_like(args[n]))})
    q = t["q"].clone().requires_grad_(True)
    out = delta_rule_fn(q, t["k"], t["v"], t["beta"], t["log_decay"], initial_state=args["state"])
    before = args["state"]._version
    delta_rule_update(**args)
    assert args["state"]._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_refusals():
    _say("delta refusals")
    from motif_mamba_amd import delta_rule_fn, delta_rule_update
    t = _dev(case(42, 2, 5, 4, 2, 16, 16, F32))

    def refused(error, **change):
        with pytest.raises(error):
            delta_rule_fn(**{**t, **change})

    refused(RuntimeError, q=t["q"].cpu())
    refused(RuntimeError, beta=t["beta"].cpu())
    refused(RuntimeError, q=t["q"].to(BF16))
    refused(RuntimeError, beta=t["beta"].double())
    refused(RuntimeError, beta=t["beta"][:, :4])
    refused(RuntimeError, beta=t["beta"][0])
    refused(ValueError, log_decay=t["log_decay"][0, 0, :3])
    refused(RuntimeError, log_decay=t["log_decay"][:, :, :3])
    refused(RuntimeError, k=t["k"][..., :8])
    refused(RuntimeError, v=t["v"][:, :, :3])
    refused(RuntimeError, initial_state=t["initial_state"].to(BF16))
    refused(RuntimeError, initial_state=t["initial_state"][:, :, :8])
    refused(ValueError, v=t["v"][0])
    big = torch.zeros(2, 5, 2, 129, device=DEV)
    refused(NotImplementedError, q=big, k=big, initial_state=None)
    refused(NotImplementedError, v=torch.zeros(2, 5, 4, 129, device=DEV), initial_state=None)
    one = [t[n][:, 0] for n in ref.NAMES[:5]]
    with pytest.raises(RuntimeError, match="overlap"):
        delta_rule_update(t["initial_state"][:1].expand(2, 4, 16, 16), *one)
    with pytest.raises(RuntimeError):
        delta_rule_update(t["initial_state"].transpose(2, 3), *one)
    with pytest.raises(RuntimeError):
        delta_rule_update(t["initial_state"].to(BF16), *one)
    d = {n: x.requires_grad_(True) for n, x in t.items()}
    (g,) = torch.autograd.grad(delta_rule_fn(**d).sum(), [d["q"]], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [d["k"]])
