"""CPU tests of how the linear attention's and the group norm's entry points treat autograd, with a stand-in for the extension
where a call would reach it, and of requests that their C entries refuse."""
import pytest
import torch
from torch.autograd import forward_ad

from tests.test_linattn_capi import PTRS, SIZES, _call, _fill, blocks  # noqa: F401


class _Ext:
    """Outputs of the right shapes."""

    def linattn_fwd(self, q, k, v, g, scale, initial, last, keep):
        return [torch.zeros_like(v), *([torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3])] if last else []),
                *([None] if keep else [])]

    def group_norm_fwd(self, x, *rest):
        return torch.zeros_like(x)


def _calls(monkeypatch):
    from motif_mamba_amd import group_norm, linear_attention, selective_scan
    monkeypatch.setattr(linear_attention, "ext", _Ext)
    monkeypatch.setattr(group_norm, "ext", _Ext)

    monkeypatch.setattr(selective_scan, "_infer", lambda u, *rest: torch.zeros_like(u))
    x, s = torch.randn(1, 4, 2, 8), torch.randn(1, 2, 8, 8)
    g = -torch.rand(1, 4, 2)
    at = [dict(q=x, k=x, v=x, log_decay=g, initial_state=s)] * 5
    for n, t in zip(("q", "k", "v", "log_decay", "initial_state"), at):
        yield f"linear attention {n}", t[n], lambda y, n=n, t=t: linear_attention.linear_attention_fn(**{**t, n: y})
    r, w = torch.randn(3, 8), torch.randn(8)
    for n, y in (("x", r), ("weight", w), ("bias", w), ("z", r)):
        args = dict(x=r, n_groups=2, weight=w, bias=w, z=r)
        yield f"group norm {n}", y, lambda y, n=n, args=args: group_norm.group_norm_fn(**{**args, n: y})
    u, A, B = torch.randn(1, 2, 4), -torch.rand(2, 3), torch.randn(1, 3, 4)
    yield "scan u", u, lambda y: selective_scan.selective_scan_fn(y, u, A, B, B)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(monkeypatch, grad):
    """A tangent needs no requires_grad: without this the call returned outputs that had none."""
    for what, x, call in _calls(monkeypatch):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            try:
                call(dual)
            except (RuntimeError, NotImplementedError):
                continue
            pytest.fail(what)


def test_without_derivatives_the_call_goes_past_autograd(monkeypatch):
    for what, x, call in _calls(monkeypatch):
        if what.startswith("scan"):
            continue
        assert call(x).grad_fn is None, what
        with forward_ad.dual_level():
            assert call(x).grad_fn is None, what
        with torch.no_grad():
            assert call(x.clone().requires_grad_(True)).grad_fn is None, what
        assert call(x.clone().requires_grad_(True)).grad_fn is not None, what


TOKEN = {**{n: x for n, x in {**SIZES, **PTRS}.items() if n != "seqlen"}, "state": 4096, "out": 4096}


@pytest.mark.parametrize("strides", [(0, 256, 16), (512, 0, 16), (512, 256, 0), (512, 256, 15), (512, 255, 16), (256, 512, 8), (500, 256, 16),
                                     (-256, 256, 16)])
def test_update_refuses_states_that_overlap(blocks, strides):
    """batch 2, 2 heads, 16 x 16: an expanded state would be written by several workgroups at once."""
    names = ("state_batch_stride", "state_head_stride", "state_dk_stride")
    rc, msg = _call("mm_linattn_update", _fill(blocks, "mm_linattn_update_params", **TOKEN, **dict(zip(names, strides))))
    assert rc == -1 and "overlap" in msg, (rc, msg)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block_rounds_a_value_once(dtype):
    """A token's value enters as v dt with the dt that its decay uses, in float32, rounded once."""
    from motif_mamba_amd import LinearAttentionBlock
    torch.manual_seed(2)
    b = LinearAttentionBlock(32, nheads=4, headdim=16, d_state=8)
    xbc, dt = torch.randn(3, 50, b.d_xbc).to(dtype), torch.randn(3, 50, 4).to(dtype)
    with torch.no_grad():
        _, _, v, g = b._operands(xbc, dt)
    exact_dt = torch.nn.functional.softplus(dt.double() + b.dt_bias.double())
    exact = xbc[..., :64].double().unflatten(-1, (4, 16)) * exact_dt.unsqueeze(-1)
    assert v.dtype == dtype and g.dtype == torch.float32
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    unit = torch.exp2(torch.floor(torch.log2(exact.detach().abs().clamp_min(2.0 ** -14)))) * half
    # softplus and the product in float32: a few 2^-24
    assert ((v.double() - exact).abs() <= unit + 2.0 ** -21 * exact.abs()).all()
    assert torch.allclose(g.double(), -torch.exp(b.A_log.double()) * exact_dt, rtol=2.0 ** -20)


@pytest.mark.parametrize("name,change", [("mm_linattn_fwd", dict(batch=1 << 23, nheads=1)), ("mm_linattn_bwd", dict(batch=1 << 23, nheads=1)),
                                         ("mm_linattn_update", dict(batch=1 << 24, nheads=1))])
def test_more_pairs_than_a_launch_takes(blocks, name, change):
    base = {"mm_linattn_fwd": {**SIZES, **PTRS, "out": 4096}, "mm_linattn_update": {**TOKEN, "state_batch_stride": 256, "state_dk_stride": 16},
            "mm_linattn_bwd": {**SIZES, **PTRS, "dout": 4096, "dq": 4096, "dk_out": 4096, "dv_out": 4096}}[name]
    rc, msg = _call(name, _fill(blocks, name + "_params", **{**base, **change}))
    assert rc == -2 and "too large" in msg, (rc, msg)
