"""GPU tests of the gated group norm (mm_group_norm.hip) against its formula in float64: group sizes from one channel
to several waves' worth, odd and unaligned ones, both gates, the activation, gradients, strides, refusals.

Bounds: half a unit of the result's type, plus float32 rounding of its terms. A normed value y is (h - mean) rstd: the
mean and h carry 2^-24 |h| and the sums' rounding, so |dy| <= 16 * 2^-24 (max |h| rstd + |y|), which the affine part
and the gate multiply; their own operations and the exponential add 16 * 2^-24 of the result. Sums of gradients: 2^-24
* 64 of the sum of the terms' absolute values (a few dozen additions in a row per thread, block and final run)."""
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


def _plain(x, groups, w, b, z, eps, act, rms, before):
    h = x * torch.nn.functional.silu(z) if before and z is not None else x
    h = h.unflatten(-1, (groups, -1))
    m = torch.zeros_like(h[..., :1]) if rms else h.mean(-1, keepdim=True)
    rstd = ((h - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    y = ((h - m) * rstd).flatten(-2)
    a = y * (1.0 if w is None else w) + (0.0 if b is None else b)
    if z is not None and not before:
        return a * torch.nn.functional.silu(z)
    return torch.nn.functional.silu(a) if act else a


def _case(seed, rows, groups, size, dtype, wdtype=F32, gate="after", weights="wb"):
    r = torch.Generator().manual_seed(seed)
    m = groups * size
    t = {"x": (torch.randn(rows, m, generator=r) * 2 + 0.5).to(dtype)}
    t["w"] = (1 + 0.2 * torch.randn(m, generator=r)).to(wdtype) if "w" in weights else None
    t["b"] = (0.3 * torch.randn(m, generator=r)).to(wdtype) if "b" in weights else None
    t["z"] = torch.randn(rows, m, generator=r).to(dtype) if gate in ("after", "before") else None
    return t


def _both(t, groups, gate, rms, dout, eps=1e-5):
    """The kernel's and the float64 results: out and gradients by name."""
    from motif_mamba_amd import group_norm_fn
    dev = {n: None if x is None else x.to(DEV).requires_grad_(True) for n, x in t.items()}
    out = group_norm_fn(dev["x"], groups, dev["w"], dev["b"], z=dev["z"], eps=eps, activation="silu" if gate == "act" else None,
                        is_rms_norm=rms, norm_before_gate=gate != "before")
    names = [n for n, x in t.items() if x is not None]
    got = dict(zip(["d" + n for n in names], torch.autograd.grad(out, [dev[n] for n in names], dout.to(DEV))), out=out)
    f = {n: None if x is None else x.double().requires_grad_(True) for n, x in t.items()}
    o = _plain(f["x"], groups, f["w"], f["b"], f["z"], eps, gate == "act", rms, gate == "before")
    exact = dict(zip(["d" + n for n in names], torch.autograd.grad(o, [f[n] for n in names], dout.double())), out=o.detach())
    return got, exact


def _bounds(t, groups, gate, rms, dout, eps=1e-5):
    """The magnitudes that float32 rounding is a fraction of, for every result."""
    f = {n: None if x is None else x.double() for n, x in t.items()}
    x, w, b = f["x"], 1.0 if f["w"] is None else f["w"].abs(), 0.0 if f["b"] is None else f["b"].abs()
    s = torch.nn.functional.silu(f["z"]).abs() if f["z"] is not None else 1.0
    # silu'(z) is at most 1.1, and |silu(z)| at most |z|
    h = (x * s if gate == "before" else x).unflatten(-1, (groups, -1))
    m = 0.0 if rms else h.mean(-1, keepdim=True)
    rstd = ((h - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    ymax = (h.abs().amax(-1, keepdim=True) * rstd).expand(h.shape).flatten(-2)   # |y| and its error's scale
    rs = rstd.expand(h.shape).flatten(-2)
    a = ymax * w + b
    d = dout.double().abs()
    z = f["z"].abs() if f["z"] is not None else 1.0
    da = d * (s if gate == "after" else 1.1 * (1 + a) if gate == "act" else 1.0)
    dn = (da * w).unflatten(-1, (groups, -1))
    mean_dn = dn.mean(-1, keepdim=True).expand(h.shape).flatten(-2)
    dh = rs * (dn.flatten(-2) + 2 * mean_dn * (1 + ymax * ymax)) * (1 + ymax)
    out = {"out": a * (s if gate == "after" else 1.0), "dx": dh * (s if gate == "before" else 1.0),
           "dw": (da * ymax).sum(0), "db": da.sum(0)}
    if f["z"] is not None:
        out["dz"] = 1.1 * (1 + z) * (d * a if gate == "after" else dh * x.abs())
    return out


def _check(t, groups, gate, rms, dtype, seed=1, eps=1e-5):
    dout = torch.randn(t["x"].shape, generator=torch.Generator().manual_seed(seed)).to(dtype)
    got, exact = _both(t, groups, gate, rms, dout, eps)
    size = _bounds(t, groups, gate, rms, dout, eps)
    for n, x in got.items():
        e, g = exact[n], x.detach().cpu().double()
        assert g.shape == e.shape
        tol = ROUND[x.dtype] * e.abs() + 64 * 2.0 ** -24 * size[n] + 6e-8 * (x.dtype == F16)
        bad = ~((g - e).abs() <= tol)
        assert not bool(bad.any()), f"{n}: {int(bad.sum())} of {bad.numel()} off by up to {(g - e).abs()[bad].max().item():.3g}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("gate,rms", [("after", False), ("before", True), ("act", False), ("none", True), ("before", False)])
@pytest.mark.parametrize("rows,groups,size", [(1, 1, 1), (3, 2, 8), (5, 24, 64), (7, 8, 125), (2, 3, 40), (4, 1, 512), (3, 2, 1000)])
def test_group_norm(rows, groups, size, gate, rms, dtype):
    _say(f"group norm {rows} x {groups} x {size} {gate} rms={rms} {dtype}")
    _check(_case(rows + size, rows, groups, size, dtype, gate=gate), groups, gate, rms, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1024, 1030, 2049, 4096, 5120, 8200, 9001, 16384])
def test_large_groups(size, dtype):
    """Groups of more than one wave, up to the largest, in vectors and one by one."""
    _say(f"group norm large group {size} {dtype}")
    _check(_case(size, 5, 1, size, dtype, gate="before"), 1, "before", True, dtype)
    _check(_case(size, 3, 2, size, dtype, gate="after"), 2, "after", False, dtype)


@pytest.mark.parametrize("rows", [300, 2000])
def test_many_rows(rows):
    _say(f"group norm rows {rows}")
    _check(_case(rows, rows, 4, 64, BF16), 4, "after", False, BF16)


@pytest.mark.parametrize("wdtype", [BF16, F16])
@pytest.mark.parametrize("weights", ["", "w", "wb"])
def test_weights(weights, wdtype):
    _say(f"group norm weights {weights} {wdtype}")
    _check(_case(9, 6, 2, 48, BF16, wdtype, "after", weights), 2, "after", False, BF16)


def test_constant_and_zero_rows():
    """A group without variance: y = 0 (0.5 / sqrt(0.25 + eps) with is_rms), finite gradients."""
    _say("group norm constant rows")
    from motif_mamba_amd import group_norm_fn
    x = torch.full((2, 64), 0.5, device=DEV)
    x[1] = 0
    assert not group_norm_fn(x, 2).any()
    assert torch.allclose(group_norm_fn(x, 2, is_rms_norm=True)[0], torch.full((64,), 0.5 / (0.25 + 1e-5) ** 0.5, device=DEV))
    x = x.requires_grad_(True)
    (g,) = torch.autograd.grad(group_norm_fn(x, 2).sum(), [x])
    assert torch.isfinite(g).all()


def test_one_group_s_values_stay_in_it():
    """An infinity or NaN reaches its own group alone; a large mean costs no digits of the variance."""
    _say("group norm non-finite")
    from motif_mamba_amd import group_norm_fn
    t = _case(11, 4, 4, 32, F32)
    clean = group_norm_fn(t["x"].to(DEV), 4, z=t["z"].to(DEV))
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[1, 40] = bad
        out = group_norm_fn(x.to(DEV), 4, z=t["z"].to(DEV))
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1, 32:64] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[1, 32:64]).any()
    x = (t["x"] + 1000).to(DEV)
    exact = _plain(x.cpu().double(), 4, None, None, None, 1e-5, False, False, False)
    assert (group_norm_fn(x, 4).cpu().double() - exact).abs().max() < 16 * 2.0 ** -24 * 1010


def test_strides_and_shapes():
    """x, z and dout as slices (aligned and not), more leading dimensions, a transposed x; the same bits."""
    _say("group norm strides")
    from motif_mamba_amd import group_norm_fn
    r = torch.Generator().manual_seed(15)
    for off in (0, 8, 1):
        wide = torch.randn(2, 9, off + 256, generator=r).to(BF16).to(DEV)
        x, z = wide[..., off:off + 128], wide[..., off + 128:]
        w = torch.randn(128, generator=r).to(DEV)
        res = []
        for a, b in ((x, z), (x.contiguous(), z.contiguous())):
            a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
            y = group_norm_fn(a, 2, w, z=b)
            assert y.shape == x.shape and y.is_contiguous()
            res.append((y, *torch.autograd.grad(y, [a, b], wide[..., off:off + 128])))
        exact = _plain(x.cpu().double(), 2, w.cpu().double(), None, z.cpu().double(), 1e-5, False, False, False)
        assert (res[0][0].cpu().double() - exact).abs().max() < 2.0 ** -8 * exact.abs().max()
        for i, (a, b) in enumerate(zip(*res)):
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-5), i
    x = torch.randn(64, 6, generator=r).to(DEV).t()
    assert torch.equal(group_norm_fn(x, 2), group_norm_fn(x.contiguous(), 2))


def test_same_bits_and_another_stream():
    _say("group norm same bits")
    t = _case(16, 700, 2, 96, BF16)
    dout = torch.randn(700, 192).to(BF16)
    a, _ = _both(t, 2, "after", False, dout)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b, _ = _both(t, 2, "after", False, dout)
    s.synchronize()
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_against_differences():
    _say("group norm differences")
    from motif_mamba_amd import group_norm_fn
    r = torch.Generator().manual_seed(17)
    t = {n: x.to(DEV) for n, x in _case(18, 4, 2, 16, F32).items()}
    dout = torch.randn(4, 32, generator=r).to(DEV)
    for before in (True, False):
        def loss(u):
            return (group_norm_fn(u["x"], 2, u["w"], u["b"], z=u["z"], norm_before_gate=before).double() * dout.double()).sum()
        leaves = {n: x.clone().requires_grad_(True) for n, x in t.items()}
        grads = torch.autograd.grad(loss(leaves), list(leaves.values()))
        for (n, x), g in zip(t.items(), grads):
            way = torch.randn(x.shape, generator=r).to(DEV)
            diff = (loss({**t, n: x + 1e-2 * way}) - loss({**t, n: x - 1e-2 * way})).item() / 2e-2
            terms = (g.double() * way.double())
            # second-order differences: h^2 times a third derivative, 1e-4 of the terms or so, 128 of them
            assert abs(diff - terms.sum().item()) <= 1e-2 * max(1.0, terms.abs().sum().item()), n


def test_empty():
    _say("group norm empty")
    from motif_mamba_amd import group_norm_fn
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y = group_norm_fn(x, 2, w)
    assert y.shape == (0, 32)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == (0, 32) and not dw.any()


def test_refusals():
    _say("group norm refusals")
    from motif_mamba_amd import group_norm_fn
    x = torch.zeros(4, 32, device=DEV)
    with pytest.raises(NotImplementedError):
        group_norm_fn(x, 2, activation="gelu")
    with pytest.raises(ValueError):
        group_norm_fn(x, 2, z=x, activation="silu")
    with pytest.raises(ValueError):
        group_norm_fn(x, 2, z=x[:2])
    for bad in (dict(n_groups=3), dict(n_groups=0), dict(n_groups=2, weight=torch.ones(16, device=DEV)), dict(n_groups=2, z=x.to(BF16)),
                dict(n_groups=2, weight=torch.ones(32)), dict(n_groups=2, eps=-1.0),
                dict(n_groups=2, weight=torch.ones(32, device=DEV), bias=torch.ones(32, device=DEV, dtype=BF16))):
        with pytest.raises(RuntimeError):
            group_norm_fn(x, **bad)
    with pytest.raises(RuntimeError):
        group_norm_fn(x.double(), 2)
    with pytest.raises(RuntimeError):
        group_norm_fn(x.cpu(), 2)
    with pytest.raises(NotImplementedError):
        group_norm_fn(torch.zeros(1, 16385, device=DEV), 1)
