"""GPU tests of the residual add with layer norm and RMS norm (mm_layer_norm.hip) against the formula in float64: row sizes from one
channel to the largest, odd and unaligned, residuals of both types, gradients, strides, graphs, refusals.

Bounds: half a unit of the result's type, plus float32 rounding of its terms. A normed value y is (h - mean) rstd: h is one addition
(2^-24 |h|), the mean and the squares' sum are sums of up to 64 additions in a thread, 6 steps in a wave and 4 waves, so
|dy| <= 80 * 2^-24 (max |h| rstd + |y|) at most and 16 * 2^-24 of it with signs as they come, which weight and bias multiply. Sums of
gradients: 2^-24 * 64 of the sum of the terms' absolute values (a few dozen additions in a row per thread, block and final run)."""
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def _plain(x, w, b, r, eps, rms):
    h = x if r is None else x + r
    m = torch.zeros_like(h[..., :1]) if rms else h.mean(-1, keepdim=True)
    y = (h - m) * ((h - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    return y * (1.0 if w is None else w) + (0.0 if b is None else b), h


def _case(seed, rows, n, dtype, residual=None, wdtype=F32, weights="wb"):
    g = torch.Generator().manual_seed(seed)
    t = {"x": (torch.randn(rows, n, generator=g) * 2 + 0.5).to(dtype)}
    t["weight"] = (1 + 0.2 * torch.randn(n, generator=g)).to(wdtype) if "w" in weights else None
    t["bias"] = (0.3 * torch.randn(n, generator=g)).to(wdtype) if "b" in weights else None
    t["residual"] = None if residual is None else torch.randn(rows, n, generator=g).to(residual)
    return t


def _check(t, rms, prenorm, seed=1, eps=1e-5, wide=False):
    from motif_mamba_amd import layer_norm_fn
    g = torch.Generator().manual_seed(seed)
    dtype = t["x"].dtype
    rtype = t["residual"].dtype if t["residual"] is not None else F32 if wide else dtype
    douts = [torch.randn(t["x"].shape, generator=g).to(dtype)] + ([torch.randn(t["x"].shape, generator=g).to(rtype)] if prenorm else [])
    names = [n for n, x in t.items() if x is not None]
    dev = {n: None if x is None else x.to(DEV).requires_grad_(True) for n, x in t.items()}
    outs = layer_norm_fn(**dev, eps=eps, prenorm=prenorm, residual_in_fp32=wide, is_rms_norm=rms)
    outs = list(outs) if prenorm else [outs]
    got = dict(zip(["d" + n for n in names], torch.autograd.grad(outs, [dev[n] for n in names], [d.to(DEV) for d in douts])))
    got.update(zip(("out", "residual_out"), outs))
    f = {n: None if x is None else x.double().requires_grad_(True) for n, x in t.items()}
    eo = list(_plain(f["x"], f["weight"], f["bias"], f["residual"], eps, rms))[:len(outs)]
    exact = dict(zip(["d" + n for n in names], torch.autograd.grad(eo, [f[n] for n in names], [d.double() for d in douts], allow_unused=True)))
    exact.update(zip(("out", "residual_out"), (o.detach() for o in eo)))
    # What float32 rounding is a fraction of.
    x, w = t["x"].double(), 1.0 if f["weight"] is None else f["weight"].detach().abs()
    b = 0.0 if f["bias"] is None else f["bias"].detach().abs()
    h = x if t["residual"] is None else x + t["residual"].double()
    habs = x.abs() if t["residual"] is None else x.abs() + t["residual"].double().abs()
    m = 0.0 if rms else h.mean(-1, keepdim=True)
    rstd = ((h - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    ymax = (habs.amax(-1, keepdim=True) * rstd).expand(h.shape)
    d = douts[0].double().abs()
    dn = d * w
    dh = rstd * (dn + 2 * dn.mean(-1, keepdim=True) * (1 + ymax * ymax)) * (1 + ymax) + (douts[1].double().abs() if prenorm else 0.0)
    size = {"out": ymax * w + b, "residual_out": habs, "dx": dh, "dresidual": dh, "dweight": (d * ymax).sum(0), "dbias": d.sum(0)}
    for n, y in got.items():
        e, z = exact[n], y.detach().cpu().double()
        assert z.shape == e.shape and y.dtype == {"out": dtype, "residual_out": rtype}.get(n, None if n[0] != "d" else t[n[1:]].dtype), n
        tol = ROUND[y.dtype] * e.abs() + 64 * 2.0 ** -24 * size[n] + 6e-8 * (y.dtype == F16)
        bad = ~((z - e).abs() <= tol)
        assert not bool(bad.any()), f"{n}: {int(bad.sum())} of {bad.numel()} off by up to {(z - e).abs()[bad].max().item():.3g}"


@pytest.mark.parametrize("dtype,residual", [(BF16, None), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32), (F32, None)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (5, 64), (2, 513), (9, 1000), (4, 1001), (3, 2560)])
def test_layer_norm(rows, n, rms, dtype, residual):
    _say(f"layer norm {rows} x {n} rms={rms} {dtype} {residual}")
    t = _case(rows + n, rows, n, dtype, residual)
    if n > 1 or rms:
        _check(t, rms, prenorm=False)
    _check(t, rms, prenorm=n % 2 == 0)
    if residual is None:
        _check(t, rms, prenorm=True, wide=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [255, 256, 257, 511, 1024, 1536, 2049, 3000, 4095, 4096, 4097, 5120, 8200, 9001, 16383, 16384])
def test_row_sizes(n, dtype):
    """Every number of pieces per thread, one wave and four, to the largest row."""
    _say(f"layer norm row {n} {dtype}")
    _check(_case(n, 5, n, dtype, F32), False, True)
    _check(_case(n, 3, n, dtype, None, weights="w"), True, False)


@pytest.mark.parametrize("rows", [300, 2000, 5000])
def test_many_rows(rows):
    """More rows than waves, which take several each."""
    _say(f"layer norm rows {rows}")
    _check(_case(rows, rows, 520, BF16, F32), True, True)
    _check(_case(rows, rows, 64, F32), False, False)
    _check(_case(rows, rows // 4, 4200, F16, F16), False, True)


@pytest.mark.parametrize("wdtype", [BF16, F16, F32])
@pytest.mark.parametrize("weights", ["", "w", "b", "wb"])
def test_weights(weights, wdtype):
    _say(f"layer norm weights {weights} {wdtype}")
    _check(_case(9, 6, 100, BF16, F32, wdtype, weights), False, True)


def test_constant_and_zero_rows():
    """A row without variance: y = 0 (0.5 / sqrt(0.25 + eps) with is_rms), finite gradients."""
    _say("layer norm constant rows")
    from motif_mamba_amd import layer_norm_fn
    x = torch.full((2, 64), 0.5, device=DEV)
    x[1] = 0
    assert not layer_norm_fn(x, None, eps=1e-5).any()
    assert torch.allclose(layer_norm_fn(x, None, eps=1e-5, is_rms_norm=True)[0], torch.full((64,), 0.5 / (0.25 + 1e-5) ** 0.5, device=DEV))
    x = x.requires_grad_(True)
    (g,) = torch.autograd.grad(layer_norm_fn(x, None, eps=1e-5).sum(), [x])
    assert torch.isfinite(g).all()


def test_one_row_s_values_stay_in_it():
    """An infinity or NaN reaches its own row alone; a large mean costs no digits of the variance."""
    _say("layer norm non-finite")
    from motif_mamba_amd import layer_norm_fn
    t = _case(11, 6, 70, F32)
    w = t["weight"].to(DEV)
    clean = layer_norm_fn(t["x"].to(DEV), w)
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[2, 40] = bad
        d = x.to(DEV).requires_grad_(True)
        out = layer_norm_fn(d, w)
        (g,) = torch.autograd.grad(out, [d], torch.ones_like(out))
        keep = torch.arange(6) != 2
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[2]).any() and torch.isfinite(g[keep]).all()
    x = (t["x"] + 1000).to(DEV)
    exact = _plain(x.cpu().double(), None, None, None, 1e-6, False)[0]
    assert (layer_norm_fn(x, None).cpu().double() - exact).abs().max() < 16 * 2.0 ** -24 * 1010


def test_strides_and_shapes():
    """x, residual and gradients as slices (aligned and not), more leading dimensions, a transposed x; the same values, and what lies
    beside them untouched."""
    _say("layer norm strides")
    from motif_mamba_amd import layer_norm_fn
    r = torch.Generator().manual_seed(15)
    for off in (0, 8, 1):
        wide = torch.randn(2, 9, off + 256, generator=r).to(BF16).to(DEV)
        res = torch.randn(2, 9, off + 256, generator=r).to(DEV)
        w = torch.randn(128, generator=r).to(DEV)
        got = []
        for f in (lambda x: x, lambda x: x.contiguous()):
            a, b = f(wide[..., off:off + 128]).detach().requires_grad_(True), f(res[..., off + 128:]).detach().requires_grad_(True)
            y, z = layer_norm_fn(a, w, residual=b, prenorm=True)
            assert y.shape == a.shape and y.is_contiguous() and z.dtype == F32 and z.is_contiguous()
            got.append((y, z, *torch.autograd.grad([y, z], [a, b], [f(wide[..., off + 128:]), f(res[..., off:off + 128])])))
        for i, (a, b) in enumerate(zip(*got)):
            assert torch.equal(a, b), i
    x = torch.randn(64, 6, generator=r).to(DEV).t()
    assert torch.equal(layer_norm_fn(x, None), layer_norm_fn(x.contiguous(), None))


def test_norm_is_of_the_unrounded_sum():
    """residual_out is h rounded; y is the norm of h, and its gradient too."""
    _say("layer norm rounding")
    t = _case(21, 40, 600, BF16, BF16)
    t["residual"] = t["residual"] * 100   # a sum whose rounding would show
    _check(t, False, True)
    _check(t, True, True)


def test_only_some_gradients():
    _say("layer norm some gradients")
    from motif_mamba_amd import layer_norm_fn
    for residual, prenorm in ((F32, True), (BF16, True), (F32, False), (None, True)):
        t = {n: None if x is None else x.to(DEV).requires_grad_(True) for n, x in _case(22, 30, 200, BF16, residual).items()}

        def loss(x):
            outs = layer_norm_fn(**x, prenorm=prenorm)
            return sum(o.float().sum() * (i + 1) for i, o in enumerate(outs)) if prenorm else outs.float().square().sum()

        names = [n for n in t if t[n] is not None]
        every = dict(zip(names, torch.autograd.grad(loss(t), [t[n] for n in names])))
        for n in names:
            x = {m: None if y is None else y.detach().requires_grad_(m == n) for m, y in t.items()}
            (g,) = torch.autograd.grad(loss(x), [x[n]])
            assert torch.equal(g, every[n]), n
    # Of the residual that is handed on alone.
    t = {n: x.to(DEV).requires_grad_(True) for n, x in _case(23, 30, 200, BF16, F32).items()}
    _, z = layer_norm_fn(**t, prenorm=True)
    dx, dr, dw = torch.autograd.grad(z, [t["x"], t["residual"], t["weight"]], torch.ones_like(z))
    assert (dx == 1).all() and (dr == 1).all() and not dw.any()
    assert layer_norm_fn(**{n: x.detach() for n, x in t.items()}).grad_fn is None


def test_same_bits_and_another_stream():
    _say("layer norm same bits")
    from motif_mamba_amd import layer_norm_fn
    t = _case(16, 3000, 600, BF16, F32)
    dout = torch.randn(3000, 600).to(BF16).to(DEV)

    def go():
        d = {n: x.to(DEV).requires_grad_(True) for n, x in t.items()}
        y, z = layer_norm_fn(**d, prenorm=True)
        return [y, z, *torch.autograd.grad([y, z], list(d.values()), [dout, torch.ones_like(z)])]

    a = go()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        b = go()
    s.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,residual", [(BF16, F32), (F32, F32)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("n", [4104, 5001])
def test_rows_of_four_waves_many_to_a_block(n, rms, dtype, residual):
    """Waves that exchange their sums through LDS, row after row: the formula's values, and the same bits on every call."""
    _say(f"layer norm four waves {n} rms={rms} {dtype} {residual}")
    from motif_mamba_amd import layer_norm_fn
    t = _case(n, 1300, n, dtype, residual)
    _check(t, rms, True)
    dev = {k: x.to(DEV) for k, x in _case(n + 1, 2000, n, dtype, residual).items()}
    douts = [torch.randn(2000, n, device=DEV).to(x) for x in (dtype, residual)]

    def go():
        d = {k: x.detach().requires_grad_(True) for k, x in dev.items()}
        outs = layer_norm_fn(**d, prenorm=True, is_rms_norm=rms)
        return [*outs, *torch.autograd.grad(outs, list(d.values()), douts)]

    one = go()
    for _ in range(3):
        for i, (x, y) in enumerate(zip(one, go())):
            assert torch.equal(x, y), i


def test_graph():
    _say("layer norm graph")
    from motif_mamba_amd import layer_norm_fn
    t = {n: x.to(DEV) for n, x in _case(17, 700, 300, BF16, F32).items()}
    dout = torch.randn(700, 300).to(BF16).to(DEV)

    def go():
        d = {n: x.detach().requires_grad_(True) for n, x in t.items()}
        y, z = layer_norm_fn(**d, prenorm=True)
        return [y, z, *torch.autograd.grad([y, z], list(d.values()), [dout, torch.ones_like(z)])]

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
        t["x"].copy_(torch.randn(700, 300))
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in res]
        for x, y in zip(got, go()):
            assert torch.equal(x, y), i


def test_backward_twice_and_a_changed_residual():
    """A graph that is kept gives the same gradients again; the residual stream that it holds may not change before that."""
    _say("layer norm backward twice")
    from motif_mamba_amd import layer_norm_fn
    r = torch.Generator().manual_seed(61)
    x = torch.randn(70, 96, generator=r).to(torch.bfloat16).to(DEV).requires_grad_(True)
    res = torch.randn(70, 96, generator=r).to(DEV).requires_grad_(True)
    w = torch.randn(96, generator=r).to(DEV).requires_grad_(True)
    y, h = layer_norm_fn(x, w, residual=res, prenorm=True, is_rms_norm=True)
    dy, dh = torch.ones_like(y), torch.ones_like(h)
    one, two = (torch.autograd.grad([y, h], [x, res, w], [dy, dh], retain_graph=True) for _ in range(2))
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, [x], dy)


def test_against_differences():
    _say("layer norm differences")
    from motif_mamba_amd import layer_norm_fn
    r = torch.Generator().manual_seed(17)
    t = {n: x.to(DEV) for n, x in _case(18, 4, 32, F32, F32).items()}
    da, db = (torch.randn(4, 32, generator=r).to(DEV).double() for _ in range(2))
    for rms in (True, False):
        def loss(u):
            y, z = layer_norm_fn(**u, prenorm=True, is_rms_norm=rms)
            return (y.double() * da).sum() + (z.double() * db).sum()
        leaves = {n: x.clone().requires_grad_(True) for n, x in t.items()}
        grads = torch.autograd.grad(loss(leaves), list(leaves.values()))
        for (n, x), g in zip(t.items(), grads):
            way = torch.randn(x.shape, generator=r).to(DEV)
            diff = (loss({**t, n: x + 1e-2 * way}) - loss({**t, n: x - 1e-2 * way})).item() / 2e-2
            terms = (g.double() * way.double())
            # second-order differences: h^2 times a third derivative, 1e-4 of the terms or so, 128 of them
            assert abs(diff - terms.sum().item()) <= 1e-2 * max(1.0, terms.abs().sum().item()), n


def test_module_and_import_path():
    _say("layer norm module")
    from mamba_ssm.ops.triton.layer_norm import RMSNorm, layer_norm_fn, rms_norm_fn
    m = RMSNorm(48, eps=1e-5).to(DEV)
    x, r = torch.randn(2, 5, 48, device=DEV), torch.randn(2, 5, 48, device=DEV)
    y, z = m(x, r, prenorm=True, residual_in_fp32=True)
    assert torch.equal(z, x + r) and torch.equal(y, layer_norm_fn(x, m.weight, m.bias, residual=r, eps=1e-5, is_rms_norm=True))
    assert torch.equal(y, rms_norm_fn(x, m.weight, residual=r, eps=1e-5))


def test_empty():
    _say("layer norm empty")
    from motif_mamba_amd import layer_norm_fn
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y, z = layer_norm_fn(x, w, prenorm=True)
    assert y.shape == z.shape == (0, 32)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == (0, 32) and not dw.any()
    assert layer_norm_fn(torch.zeros(3, 0, device=DEV), None).shape == (3, 0)


def test_refusals():
    _say("layer norm refusals")
    from motif_mamba_amd import layer_norm_fn
    x = torch.zeros(4, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    with pytest.raises(ValueError):
        layer_norm_fn(x, w, residual=x[:2])
    with pytest.raises(NotImplementedError):
        layer_norm_fn(torch.zeros(1, 16385, device=DEV), None)
    for bad in (dict(weight=w[:16]), dict(weight=w.cpu()), dict(weight=w, bias=w.to(BF16)), dict(weight=w.double()), dict(weight=w, eps=-1.0),
                dict(weight=w, residual=x.to(BF16)), dict(weight=w, residual=x.double()), dict(weight=w, residual=x.cpu())):
        with pytest.raises(RuntimeError):
            layer_norm_fn(x, **bad)
    with pytest.raises(RuntimeError):
        layer_norm_fn(x.double(), w)
    with pytest.raises(RuntimeError):
        layer_norm_fn(x.cpu(), w)
    y = layer_norm_fn(x.requires_grad_(True), w)
    (g,) = torch.autograd.grad(y.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [x])
