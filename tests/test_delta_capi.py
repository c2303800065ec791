"""CPU checks of the C ABI of the gated delta rule and the layer norm (include/mm_delta.h, include/mm_layer_norm.h): what the library
exports, requests refused before anything is launched, and how the Python entry points treat autograd, with a stand-in for the
extension where a call would reach it. The parameter blocks are filled by name through offsets taken from the headers."""
import ctypes
import os
import re
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from tests import capi

HEADERS = {"mm_delta.h": ["mm_delta_fwd", "mm_delta_fwd_workspace_size", "mm_delta_bwd", "mm_delta_bwd_workspace_size", "mm_delta_update",
                          "mm_delta_segment_states_size"],
           "mm_layer_norm.h": ["mm_layer_norm_fwd", "mm_layer_norm_bwd", "mm_layer_norm_bwd_workspace_size"]}
INC = os.path.join(capi.REPO, "include")


def _lib():
    from motif_mamba_amd import _native
    return _native.lib()


def test_exports():
    for h, names in HEADERS.items():
        text = open(os.path.join(INC, h)).read()
        assert sorted(set(re.findall(r"^\w[\w ]*?\b(mm_\w+)\(", text, re.M))) == sorted(names)
        for n in names:
            assert hasattr(_lib(), n), n


@pytest.fixture(scope="module")
def blocks(tmp_path_factory):
    """struct name -> (size, {field: (offset, size)})"""
    d = tmp_path_factory.mktemp("layout")
    text = "".join(open(os.path.join(INC, h)).read() for h in HEADERS)
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    found = {}
    for body, name in re.findall(r"typedef struct \w+ \{(.*?)\} (\w+);", text, re.S):
        found[name] = [re.sub(r".*[ *]", "", f.strip()) for line in body.split(";") for f in line.split(",") if f.strip()]
    src = ['#include <stdio.h>', '#include <stddef.h>', *(f'#include "{h}"' for h in HEADERS), 'int main(void) {']
    for name, fields in found.items():
        src.append(f'printf("{name} . %zu 0\\n", sizeof({name}));')
        src += [f'printf("{name} {f} %zu %zu\\n", offsetof({name}, {f}), sizeof((({name} *)0)->{f}));' for f in fields]
    (d / "l.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.check_call(["gcc", "-std=c11", f"-I{INC}", str(d / "l.c"), "-o", str(d / "l")])
    res = {}
    for line in subprocess.check_output([str(d / "l")]).decode().split("\n"):
        if line:
            name, f, off, size = line.split()
            if f == ".":
                res[name] = (int(off), {})
            else:
                res[name][1][f] = (int(off), int(size))
    return res


def _fill(blocks, name, **values):
    size, fields = blocks[name]
    buf = bytearray(size)
    for f, v in values.items():
        off, n = fields[f]
        raw = ctypes.c_float(v) if isinstance(v, float) else {4: ctypes.c_int32, 8: ctypes.c_int64}[n](v)
        buf[off:off + n] = bytes(raw)
    return (ctypes.c_char * size).from_buffer(buf)


def _call(name, block):
    fn = getattr(_lib(), name)
    fn.restype = ctypes.c_int
    rc = fn(block, None)
    return rc, _lib().mm_last_error().decode()


SIZES = dict(batch=2, seqlen=5, n_groups=1, nheads=2, dk=16, dv=16, itype=2, gtype=0, btype=0)
PTRS = dict(q=4096, k=4096, v=4096, beta=4096, log_decay=4096)
ROOM = dict(workspace=4096, workspace_bytes=1 << 40)
FWD = {**SIZES, **PTRS, **ROOM, "out": 4096}
BWD = {**SIZES, **PTRS, **ROOM, "dout": 4096, "dq": 4096, "dk_out": 4096, "dv_out": 4096, "dbeta": 4096}
TOKEN = {n: x for n, x in {**SIZES, **PTRS, "state": 4096, "out": 4096}.items() if n != "seqlen"}
SHARED = [
    (dict(itype=7), -1, "dtype"), (dict(gtype=9), -1, "dtype"), (dict(btype=3), -1, "dtype"), (dict(seqlen=-1), -1, "negative"),
    (dict(n_groups=0), -1, "multiple"), (dict(nheads=3, n_groups=2), -1, "multiple"), (dict(dk=0), -1, "at least 1"), (dict(dk=129), -2, "128"),
    (dict(dv=200), -2, "128"), (dict(batch=1 << 20), -2, "too large"), (dict(batch=1 << 62, nheads=8), -2, "too large"),
    (dict(seqlen=(1 << 23) + 1), -2, "2^23"), (dict(q=0), -1, "required"), (dict(beta=0), -1, "required"),
    (dict(workspace=0), -1, "workspace"), (dict(workspace_bytes=64), -1, "workspace"), (dict(q_seq_stride=1 << 22), -2, "strides"),
    (dict(v_seq_stride=-4), -2, "strides")]


@pytest.mark.parametrize("change,code,needle", [*SHARED, (dict(out=0), -1, "required"), (dict(out_seq_stride=1 << 22), -2, "strides")])
def test_fwd_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_delta_fwd", _fill(blocks, "mm_delta_fwd_params", **{**FWD, **change}))
    assert rc == code and needle in msg, (rc, msg)


@pytest.mark.parametrize("change,code,needle", [*SHARED, (dict(dq=0), -1, "required"), (dict(dout=0), -1, "required"), (dict(dbeta=0), -1, "required"),
                                                (dict(do_seq_stride=1 << 22), -2, "strides"), (dict(log_decay=0, dlog_decay=4096), -1, "goes with")])
def test_bwd_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_delta_bwd", _fill(blocks, "mm_delta_bwd_params", **{**BWD, **change}))
    assert rc == code and needle in msg, (rc, msg)


@pytest.mark.parametrize("change,code,needle", [
    (dict(itype=7), -1, "dtype"), (dict(dk=129), -2, "128"), (dict(batch=1 << 23, nheads=1), -2, "too large"), (dict(state=0), -1, "required"),
    (dict(beta=0), -1, "required"), *((dict(zip(("state_batch_stride", "state_head_stride", "state_dk_stride"), s)), -1, "overlap") for s in (
        (0, 256, 16), (512, 0, 16), (512, 256, 0), (512, 256, 15), (512, 255, 16), (256, 512, 8), (500, 256, 16), (-256, 256, 16)))])
def test_update_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_delta_update", _fill(blocks, "mm_delta_update_params", **{**TOKEN, **change}))
    assert rc == code and needle in msg, (rc, msg)


def test_workspaces_are_enough_by_a_byte(blocks):
    """What the query says is what the call accepts."""
    for name, base in (("mm_delta_fwd", FWD), ("mm_delta_bwd", {**BWD, "nheads": 4, "dlog_decay": 4096, "decay_per_head": 1})):
        for t in (0, 1, 2):
            block = {**base, "itype": t, "seqlen": 77}
            size = getattr(_lib(), name + "_workspace_size")
            size.restype = ctypes.c_int64
            n = size(_fill(blocks, name + "_params", **block))
            assert n > 0
            rc, msg = _call(name, _fill(blocks, name + "_params", **{**block, "workspace_bytes": n - 1}))
            assert rc == -1 and "workspace" in msg
            assert size(_fill(blocks, name + "_params", **{**block, "seqlen": 0})) == 0 == size(None)


def test_segment_states_of_another_size_are_refused(blocks, monkeypatch):
    """The forward's and backward's cuts of a row are the same, or the call is refused (MM_DELTA_SEGMENTS may change between the two)."""
    monkeypatch.setenv("MM_DELTA_SEGMENTS", "3")
    size = _lib().mm_delta_segment_states_size
    size.restype = ctypes.c_int64
    sizes = {t: size(_fill(blocks, "mm_delta_fwd_params", **{**FWD, "itype": t, "seqlen": 200})) for t in (0, 1, 2)}
    assert all(sizes.values())
    for name, base in (("mm_delta_fwd", FWD), ("mm_delta_bwd", BWD)):
        for t, n in sizes.items():
            block = {**base, "itype": t, "seqlen": 200, "segment_states": 4096}
            work = getattr(_lib(), name + "_workspace_size")
            work.restype = ctypes.c_int64
            least = work(_fill(blocks, name + "_params", **{**block, "segment_states_bytes": n}))
            assert least < work(_fill(blocks, name + "_params", **{**block, "segment_states": 0}))
            for bytes_ in (0, n - 16, n + 16):
                rc, msg = _call(name, _fill(blocks, name + "_params", **{**block, "segment_states_bytes": bytes_}))
                assert rc == -1 and "segment_states" in msg, (rc, msg)
            rc, msg = _call(name, _fill(blocks, name + "_params", **{**block, "segment_states_bytes": n, "workspace_bytes": least - 1}))
            assert rc == -1 and "workspace" in msg, (rc, msg)
            monkeypatch.setenv("MM_DELTA_SEGMENTS", "1")
            rc, msg = _call(name, _fill(blocks, name + "_params", **{**block, "segment_states_bytes": n}))
            assert rc == -1 and "segment_states" in msg, (rc, msg)
            monkeypatch.setenv("MM_DELTA_SEGMENTS", "3")


@pytest.mark.parametrize("segments", [None, "1", "4"])
@pytest.mark.parametrize("change", [dict(batch=1 << 20, nheads=2), dict(batch=1 << 62, nheads=8), dict(batch=1 << 32, nheads=1 << 32), dict(dk=129), dict(dv=0),
                                    dict(seqlen=(1 << 23) + 1), dict(n_groups=0), dict(itype=7)])
def test_sizes_of_refused_calls(blocks, change, segments):
    """The size queries, which come before the call that refuses, need nothing for it and end as they should, with any number of segments
    asked for. (In a process of its own, which a division by zero would end.)"""
    work = []
    for name, base in (("mm_delta_fwd", FWD), ("mm_delta_bwd", BWD)):
        block = bytes(_fill(blocks, name + "_params", **{**base, "seqlen": 200, **change})).hex()
        work += [(f, block) for f in ([name + "_workspace_size"] + (["mm_delta_segment_states_size"] if name == "mm_delta_fwd" else []))]
    code = f"""
import ctypes, sys
lib = ctypes.CDLL({_lib()._name!r})
for name, block in {work!r}:
    f = getattr(lib, name)
    f.restype = ctypes.c_int64
    raw = bytes.fromhex(block)
    print(name, f((ctypes.c_char * len(raw)).from_buffer_copy(raw)), flush=True)
"""
    env = {n: x for n, x in os.environ.items() if n != "MM_DELTA_SEGMENTS"}
    res = subprocess.run([sys.executable, "-c", code], env={**env, **({"MM_DELTA_SEGMENTS": segments} if segments else {})}, stdout=subprocess.PIPE, timeout=120)
    assert res.returncode == 0, (res.returncode, res.stdout)
    assert res.stdout.decode().split("\n")[:-1] == [f"{f} 0" for f, _ in work]


def test_nothing_to_do(blocks):
    assert _call("mm_delta_fwd", _fill(blocks, "mm_delta_fwd_params", **{**SIZES, "batch": 0}))[0] == 0
    assert _call("mm_delta_fwd", _fill(blocks, "mm_delta_fwd_params", **{**SIZES, "seqlen": 0}))[0] == 0
    assert _call("mm_delta_bwd", _fill(blocks, "mm_delta_bwd_params", **{**SIZES, "seqlen": 0}))[0] == 0
    token = {n: x for n, x in SIZES.items() if n != "seqlen"}
    assert _call("mm_delta_update", _fill(blocks, "mm_delta_update_params", **{**token, "batch": 0}))[0] == 0
    for name in ("mm_delta_fwd", "mm_delta_bwd", "mm_delta_update", "mm_layer_norm_fwd", "mm_layer_norm_bwd"):
        assert _call(name, None)[0] == -1


NORM = dict(rows=2, channels=32, itype=2, rtype=2, wtype=0, eps=1e-5, x=4096, out=4096)


@pytest.mark.parametrize("change,code,needle", [
    (dict(itype=3), -1, "dtype"), (dict(rtype=5), -1, "dtype"), (dict(wtype=-1), -1, "dtype"), (dict(rtype=1), -2, "residual"), (dict(itype=0, rtype=2), -2, "residual"),
    (dict(rows=-1), -1, "negative"), (dict(channels=16385), -2, "16384"), (dict(rows=1 << 24), -2, "rows"), (dict(eps=-1.0), -1, "eps"),
    (dict(eps=float("nan")), -1, "eps"), (dict(x=0), -1, "required"), (dict(out=0), -1, "required")])
def test_norm_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_layer_norm_fwd", _fill(blocks, "mm_layer_norm_params", **{**NORM, **change}))
    assert rc == code and needle in msg, (rc, msg)


def test_norm_bwd_refusals(blocks):
    rc, msg = _call("mm_layer_norm_bwd", _fill(blocks, "mm_layer_norm_params", **NORM))
    assert rc == -1 and "dout" in msg
    rc, msg = _call("mm_layer_norm_bwd", _fill(blocks, "mm_layer_norm_params", **{**NORM, "x": 0, "dout": 4096}))
    assert rc == -1 and "residual" in msg
    rc, msg = _call("mm_layer_norm_bwd", _fill(blocks, "mm_layer_norm_params", **{**NORM, "dout": 4096, "dx": 4096, "dweight": 4096}))
    assert rc == -1 and "workspace" in msg
    assert _call("mm_layer_norm_fwd", _fill(blocks, "mm_layer_norm_params", **{**NORM, "rows": 0}))[0] == 0


def test_python_refusals_without_a_gpu():
    from motif_mamba_amd import delta_rule_fn, delta_rule_update, layer_norm_fn
    x, b = torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1)
    with pytest.raises(RuntimeError):
        delta_rule_fn(x, x, x, b)
    with pytest.raises(ValueError):
        delta_rule_fn(x, x, x[0], b)
    with pytest.raises(RuntimeError):
        delta_rule_update(torch.zeros(1, 1, 8, 8), x[:, 0], x[:, 0], x[:, 0], b[:, 0])
    with pytest.raises(RuntimeError):
        layer_norm_fn(torch.zeros(2, 8), None)
    with pytest.raises(ValueError):
        layer_norm_fn(torch.zeros(2, 8), None, residual=torch.zeros(3, 8))


class _Ext:
    """Outputs of the right shapes."""

    def delta_fwd(self, q, k, v, beta, g, scale, initial, last, keep):
        return [torch.zeros_like(v), *([torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3])] if last else []),
                *([None] if keep else [])]

    def layer_norm_fwd(self, x, residual, weight, bias, eps, rms, want, wide):
        return [torch.zeros_like(x), torch.zeros_like(x) if want else None]


def _calls(monkeypatch):
    from motif_mamba_amd import delta_rule, layer_norm
    monkeypatch.setattr(delta_rule, "ext", _Ext)
    monkeypatch.setattr(layer_norm, "ext", _Ext)
    x, s, g = torch.randn(1, 4, 2, 8), torch.randn(1, 2, 8, 8), -torch.rand(1, 4, 2)
    at = dict(q=x, k=x, v=x, beta=g, log_decay=g, initial_state=s)
    for n in at:
        yield f"delta rule {n}", at[n], lambda y, n=n: delta_rule.delta_rule_fn(**{**at, n: y})
    r, w = torch.randn(3, 8), torch.randn(8)
    args = dict(x=r, weight=w, bias=w, residual=r)
    for n in args:
        yield f"layer norm {n}", args[n], lambda y, n=n: layer_norm.layer_norm_fn(**{**args, n: y})


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(monkeypatch, grad):
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
        assert call(x).grad_fn is None, what
        with torch.no_grad():
            assert call(x.clone().requires_grad_(True)).grad_fn is None, what
        assert call(x.clone().requires_grad_(True)).grad_fn is not None, what
