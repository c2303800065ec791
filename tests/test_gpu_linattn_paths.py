"""GPU tests of the linear attention on the ways through its kernels that tests/test_gpu_linattn.py does not take: the backward
where the decays need no gradient, and rows cut into segments at dk above 64, at odd sizes, unaligned and with one decay per head.
Against the recurrence in float64; states, scores and sums are float32 for every input type, so the terms' error is float32's."""
import sys

import pytest
import torch

from tests import linattn_ref as ref
from tests.test_gpu_linattn import SHAPES, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _say(msg):
    print(f"\n[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def _dout(t, seed):
    r = torch.Generator().manual_seed(seed)
    return torch.randn(t["v"].shape, generator=r).to(t["v"].dtype), r


def _check(t, scale, dout, dlast, wanted, views=None):
    """Outputs and the gradients of `wanted` against float64. views: the device tensors to use instead of copies of t."""
    from motif_mamba_amd import linear_attention_fn
    dev = {n: (views or {}).get(n, x.to(DEV)) for n, x in t.items()}
    dev = {n: x.detach().requires_grad_(n in wanted) for n, x in dev.items()}
    out, last = linear_attention_fn(**dev, scale=scale, return_last_state=True)
    outs, douts = ([out], [dout.to(DEV)]) if dlast is None else ([out, last], [dout.to(DEV), dlast.to(DEV)])
    got = torch.autograd.grad(outs, [dev[n] for n in wanted], douts)
    exact, size = ref.with_grads(t, scale, dout, dlast), ref.magnitudes(t, scale, dout, dlast)
    ref.check(out, exact["out"], size["out"], F32, "out")
    ref.check(last, exact["last_state"], size["last_state"], F32, "last_state")
    for n, x in zip(wanted, got):
        ref.check(x, exact["d" + n], size["d" + n], F32, "d" + n, whole_row=n == "log_decay")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_without_the_decays(shape, per_head, dtype):
    _say(f"linear attention gradients without the decays' {shape} {per_head} {dtype}")
    t = _inputs(2000 + sum(shape), *shape, dtype, per_head=per_head)
    dout, _ = _dout(t, 1)
    _check(t, shape[4] ** -0.5, dout, None, ["q", "k", "v"])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("wanted", [["q", "k", "v", "initial_state"], ["v"], ["initial_state"], ["log_decay"]])
@pytest.mark.parametrize("shape", [(1, 100, 2, 4, 64, 64), (1, 300, 1, 2, 128, 40), (2, 129, 3, 3, 40, 128)])
def test_some_gradients_and_states(shape, wanted, dtype):
    _say(f"linear attention gradients of {wanted} {shape} {dtype}")
    t = _inputs(2100 + sum(shape), *shape, dtype, states=True)
    dout, r = _dout(t, 2)
    _check(t, 0.3, dout, torch.randn(t["initial_state"].shape, generator=r), wanted)


def _segmented(t):
    from motif_mamba_amd._native import ext
    d = {n: x.to(DEV) for n, x in t.items()}
    g = d["log_decay"].expand(*d["v"].shape[:3])
    return ext().linattn_fwd(d["q"], d["k"], d["v"], g, 1.0, None, False, True)[1] is not None


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("wanted", [["q", "k", "v", "log_decay", "initial_state"], ["q", "k", "v"]])
@pytest.mark.parametrize("L,G,H,dk,dv", [(1100, 1, 2, 128, 128), (1280, 2, 2, 80, 96), (1101, 1, 2, 37, 50), (1500, 1, 1, 128, 48), (1201, 1, 3, 24, 72)])
def test_segments(L, G, H, dk, dv, wanted, dtype):
    _say(f"linear attention segments {L} {G} {H} {dk} {dv} {len(wanted)} {dtype}")
    t = _inputs(2200 + L, 1, L, G, H, dk, dv, dtype, states=True)
    assert _segmented(t)
    dout, r = _dout(t, 3)
    _check(t, dk ** -0.5, dout, torch.randn(t["initial_state"].shape, generator=r), wanted)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("wanted", [["q", "k", "v", "log_decay"], ["q", "k", "v"]])
def test_segments_of_a_decay_per_head(wanted, dtype):
    _say(f"linear attention segments, a decay per head {len(wanted)} {dtype}")
    t = _inputs(2300, 1, 1100, 1, 2, 72, 64, dtype, per_head=True)
    assert _segmented(t)
    dout, _ = _dout(t, 4)
    _check(t, 0.1, dout, None, wanted)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("off", [0, 3])
def test_segments_of_slices(off, dtype):
    """q, k and v slices of one tensor, aligned and not."""
    _say(f"linear attention segments of slices {off} {dtype}")
    L, dk, dv = 1100, 96, 64
    t = _inputs(2400, 1, L, 1, 2, dk, dv, dtype)
    wide = torch.cat([torch.zeros(1, L, off, dtype=dtype), t["q"].flatten(2), t["k"].flatten(2), t["v"].flatten(2)], -1).to(DEV)
    q, k, v = wide[..., off:].split([dk, dk, 2 * dv], -1)
    views = {"q": q.unflatten(-1, (1, dk)), "k": k.unflatten(-1, (1, dk)), "v": v.unflatten(-1, (2, dv))}
    assert _segmented(t)
    dout, _ = _dout(t, 5)
    _check(t, 0.1, dout, None, ["q", "k", "v", "log_decay"], views)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("wanted", [["q", "k", "v", "log_decay", "initial_state"], ["q", "k", "v"]])
@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("dk,dv", [(48, 40), (48, 104), (112, 40), (112, 104), (37, 33), (37, 101), (107, 33), (107, 101)])
def test_every_kernel(dk, dv, heads, wanted, dtype):
    """The kernels are built for dk and dv up to 64 and up to 128, aligned rows and others, heads of their own and shared q and k,
    and with and without the decays' gradient: each of them."""
    _say(f"linear attention {dk} {dv} {heads} heads {len(wanted)} {dtype}")
    t = _inputs(2500 + dk + dv, 1, 150, 1, heads, dk, dv, dtype, states=True)
    dout, r = _dout(t, 6)
    _check(t, dk ** -0.5, dout, torch.randn(t["initial_state"].shape, generator=r), wanted)
