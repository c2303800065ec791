"""GPU tests of GatedDeltaBlock, the operators of a delta-rule layer run together with the norm at its entry and the residual stream:
outputs and gradients of two layers in a row against the same in float64 on the CPU, and a prompt continued token by token.

Bounds: float32 throughout, two layers of projections of 96 and 256 terms, a conv, three norms; some hundreds of roundings of 2^-24
behind every value, taken as 2^-14 of the largest one (the norms' divisions and the state's memory amplify)."""
import sys

import pytest
import torch
from torch import nn
from torch.nn import functional as F

from tests import delta_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


class _Two(nn.Module):
    def __init__(self, n_groups=2):
        super().__init__()
        from motif_mamba_amd import GatedDeltaBlock, RMSNorm
        self.layers = nn.ModuleList(GatedDeltaBlock(96, nheads=4, headdim=64, d_state=32, n_groups=n_groups) for _ in range(2))
        self.norm = RMSNorm(96)
        for m in (*self.layers, self):
            nn.init.normal_(m.norm.weight, 1.0, 0.1)

    def forward(self, x, caches=(None, None)):
        r = None
        for m, c in zip(self.layers, caches):
            x, r = m(x, r, c)
        return self.norm(x, r)

    def step(self, x, caches):
        r = None
        for m, c in zip(self.layers, caches):
            x, r = m.step(x, r, c)
        return self.norm(x, r)


def _two(seed, **kw):
    torch.manual_seed(seed)
    return _Two(**kw)


def _rms(x, w, eps):
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w


def _plain(m, x):
    """The same in plain float64."""
    r = torch.zeros_like(x)
    for b in m.layers:
        r = r + x
        z, qkv, beta, a = (_rms(r, b.norm.weight, b.eps) @ b.in_proj.weight.t()).split([b.d_inner, b.d_qkv, b.nheads, b.nheads], -1)
        conv = F.silu(F.conv1d(F.pad(qkv.transpose(1, 2), (b.d_conv - 1, 0)), b.conv_weight.unsqueeze(1), b.conv_bias, groups=b.d_qkv)).transpose(1, 2)
        v, q, k = conv.split([b.d_inner, b.d_qk, b.d_qk], -1)
        q, k = (y.unflatten(-1, (b.n_groups, b.d_state)) for y in (q, k))
        q, k = (y / (y.square().sum(-1, keepdim=True) + 1e-6).sqrt() for y in (q, k))
        y, _ = ref.recurrence(q, k, v.unflatten(-1, (b.nheads, b.headdim)), torch.sigmoid(beta),
                              -torch.exp(b.A_log) * F.softplus(a + b.dt_bias), b.d_state ** -0.5)
        y = (_rms(y, 1.0, b.eps)).flatten(-2) * b.norm_weight * F.silu(z)
        x = y @ b.out_proj.weight.t()
    return _rms(r + x, m.norm.weight, m.norm.eps)


@pytest.mark.parametrize("L", [1, 5, 100])
def test_outputs_and_gradients(L):
    _say(f"gated delta blocks L {L}")
    m = _two(L)
    x = torch.randn(2, L, 96)
    dout = torch.randn(2, L, 96)
    f = _two(L).double()
    exact = _plain(f, x.double())
    want = torch.autograd.grad(exact, list(f.parameters()), dout.double())
    m = m.to(DEV)
    out = m(x.to(DEV))
    got = torch.autograd.grad(out, list(m.parameters()), dout.to(DEV))
    for n, a, e in [("out", out, exact), *((n, a, e) for (n, _), a, e in zip(m.named_parameters(), got, want))]:
        err = (a.detach().cpu().double() - e.detach()).abs().max().item()
        assert err <= 2.0 ** -14 * max(1e-3, e.abs().max().item()), (n, err)


@pytest.mark.parametrize("split", [1, 2, 40, 69])
def test_prompt_then_steps(split):
    """The prompt and the tokens after it give what the whole text gives."""
    _say(f"gated delta blocks, prompt of {split} and steps")
    m = _two(7, n_groups=1).to(DEV)
    x = torch.randn(3, 70, 96, device=DEV)
    with torch.no_grad():
        whole = m(x)
        caches = [b.allocate_inference_cache(3) for b in m.layers]
        out = [m(x[:, :split], caches)]
        out += [m.step(x[:, t], caches).unsqueeze(1) for t in range(split, 70)]
    err = (torch.cat(out, 1) - whole).abs().max().item()
    assert err <= 2.0 ** -14 * whole.abs().max().item(), err


def test_bf16_runs():
    _say("gated delta blocks bf16")
    m = _two(9).to(DEV)
    x = torch.randn(2, 130, 96, device=DEV)
    exact = m(x)
    for b in m.layers:
        b.in_proj.to(torch.bfloat16), b.out_proj.to(torch.bfloat16)
        b.conv_weight.data, b.conv_bias.data = b.conv_weight.data.bfloat16(), b.conv_bias.data.bfloat16()
    out = m(x.bfloat16())
    out.sum().backward()
    assert out.dtype == torch.bfloat16 and all(torch.isfinite(p.grad).all() for p in m.parameters())
    # two layers of eight roundings of 2^-8 each, of a sum's terms; the stream between them is float32
    assert (out.float() - exact).norm() <= 16 * 2.0 ** -8 * exact.norm()


def test_step_refuses_derivatives():
    """In grad mode, before the cache is touched."""
    _say("gated delta block: step in grad mode")
    m = _two(5).to(DEV).layers[0]
    cache = m.allocate_inference_cache(2)
    x = torch.randn(2, 96, device=DEV)
    with pytest.raises(RuntimeError, match="derivatives"):
        m.step(x, None, cache)
    assert not any(c.any() for c in cache)
    with torch.no_grad():
        out, res = m.step(x, None, cache)
    assert out.shape == x.shape and res.dtype == torch.float32 and all(c.any() for c in cache)


def test_steps_in_a_graph():
    _say("gated delta blocks: captured step")
    m = _two(6).to(DEV)
    x = torch.randn(2, 96, device=DEV)
    caches = [b.allocate_inference_cache(2) for b in m.layers]
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                m.step(x, caches)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = m.step(x, caches)
        for c in (*caches[0], *caches[1]):
            c.zero_()
        eager = [b.allocate_inference_cache(2) for b in m.layers]
        for i in range(4):
            x.copy_(torch.randn(2, 96))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, m.step(x, eager)), i
