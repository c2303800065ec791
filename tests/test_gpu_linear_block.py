"""GPU tests of LinearAttentionBlock, the operators of a linear-attention layer run together: its outputs and gradients
against the same layer in float64 on the CPU, and a prompt continued token by token.

Bounds: float32 throughout, projections of 96 and 256 terms, a conv, a norm; a few hundred roundings of 2^-24 behind every
value, taken as 2^-14 of the largest one (the sums over the state's memory and the norm's division amplify)."""
import sys

import pytest
import torch
from torch.nn import functional as F

from tests import linattn_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def _block(seed, n_groups=2):
    from motif_mamba_amd import LinearAttentionBlock
    torch.manual_seed(seed)
    return LinearAttentionBlock(96, nheads=4, headdim=64, d_state=32, n_groups=n_groups)


def _plain(b, hidden):
    """The layer in plain float64."""
    z, xbc, dt = (hidden @ b.in_proj.weight.t()).split([b.d_inner, b.d_xbc, b.nheads], -1)
    w = b.conv_weight.unsqueeze(1)
    conv = F.silu(F.conv1d(F.pad(xbc.transpose(1, 2), (b.d_conv - 1, 0)), w, b.conv_bias, groups=b.d_xbc)).transpose(1, 2)
    v, q, k = conv.split([b.d_inner, b.d_qk, b.d_qk], -1)
    dt = F.softplus(dt + b.dt_bias)
    y, _ = ref.recurrence(q.unflatten(-1, (b.n_groups, b.d_state)), k.unflatten(-1, (b.n_groups, b.d_state)),
                          v.unflatten(-1, (b.nheads, b.headdim)) * dt.unsqueeze(-1), -torch.exp(b.A_log) * dt, 1.0)
    h = (y.flatten(-2) * F.silu(z)).unflatten(-1, (b.n_groups, -1))
    h = (h * (h.square().mean(-1, keepdim=True) + b.eps).rsqrt()).flatten(-2) * b.norm_weight
    return h @ b.out_proj.weight.t()


@pytest.mark.parametrize("L", [1, 5, 100])
def test_outputs_and_gradients(L):
    _say(f"linear attention block L {L}")
    b = _block(L)
    hidden = torch.randn(2, L, 96)
    dout = torch.randn(2, L, 96)
    f = _block(L).double()
    exact = _plain(f, hidden.double())
    want = torch.autograd.grad(exact, list(f.parameters()), dout.double())
    b = b.to(DEV)
    out = b(hidden.to(DEV))
    got = torch.autograd.grad(out, list(b.parameters()), dout.to(DEV))
    for n, x, y in [("out", out, exact), *((n, x, y) for (n, _), x, y in zip(b.named_parameters(), got, want))]:
        err = (x.detach().cpu().double() - y.detach()).abs().max().item()
        assert err <= 2.0 ** -14 * max(1e-3, y.abs().max().item()), (n, err)


@pytest.mark.parametrize("split", [1, 2, 40, 69])
def test_prompt_then_steps(split):
    """The prompt and the tokens after it give what the whole text gives."""
    _say(f"linear attention block, prompt of {split} and steps")
    b = _block(7, n_groups=1).to(DEV)
    hidden = torch.randn(3, 70, 96, device=DEV)
    with torch.no_grad():
        whole = b(hidden)
        cache = b.allocate_inference_cache(3)
        out = [b(hidden[:, :split], cache)]
        out += [b.step(hidden[:, t], cache).unsqueeze(1) for t in range(split, 70)]
    err = (torch.cat(out, 1) - whole).abs().max().item()
    assert err <= 2.0 ** -14 * whole.abs().max().item(), err


def test_bf16_runs():
    _say("linear attention block bf16")
    b = _block(9).to(DEV)
    hidden = torch.randn(2, 130, 96, device=DEV)
    exact = b(hidden)
    for p in (b.in_proj, b.out_proj):
        p.to(torch.bfloat16)
    b.conv_weight.data, b.conv_bias.data = b.conv_weight.data.bfloat16(), b.conv_bias.data.bfloat16()
    out = b(hidden.bfloat16())
    out.sum().backward()
    assert out.dtype == torch.bfloat16 and all(torch.isfinite(p.grad).all() for p in b.parameters())
    # six roundings of 2^-8 in a row, each of a sum's terms
    assert (out.float() - exact).norm() <= 6 * 2.0 ** -8 * exact.norm()
