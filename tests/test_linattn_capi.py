"""CPU checks of the C ABI of the linear attention and the group norm (include/mm_linattn.h, include/mm_group_norm.h): what the
library exports, and requests refused before anything is launched. The parameter blocks are filled by name through offsets
taken from the headers."""
import ctypes
import os
import re
import subprocess

import pytest

from tests import capi

HEADERS = {"mm_linattn.h": ["mm_linattn_fwd", "mm_linattn_fwd_workspace_size", "mm_linattn_bwd", "mm_linattn_bwd_workspace_size",
                            "mm_linattn_update"],
           "mm_group_norm.h": ["mm_group_norm_fwd", "mm_group_norm_bwd", "mm_group_norm_bwd_workspace_size"]}
INC = os.path.join(capi.REPO, "include")


def _lib():
    from motif_mamba_amd import _native
    return _native.lib()


def test_exports():
    lib = _lib()
    for h, names in HEADERS.items():
        text = open(os.path.join(INC, h)).read()
        assert sorted(set(re.findall(r"^\w[\w ]*?\b(mm_\w+)\(", text, re.M))) == sorted(names)
        for n in names:
            assert hasattr(lib, n), n


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


SIZES = dict(batch=2, seqlen=5, n_groups=1, nheads=2, dk=16, dv=16, itype=2, gtype=0)
PTRS = dict(q=4096, k=4096, v=4096, log_decay=4096)


@pytest.mark.parametrize("change,code,needle", [
    (dict(itype=7), -1, "dtype"), (dict(gtype=9), -1, "dtype"), (dict(seqlen=-1), -1, "negative"), (dict(n_groups=0), -1, "multiple"),
    (dict(nheads=3, n_groups=2), -1, "multiple"), (dict(dk=0), -1, "at least 1"), (dict(dk=129), -2, "128"), (dict(dv=200), -2, "128"),
    (dict(batch=1 << 23), -2, "too large"), (dict(seqlen=1 << 24), -2, "2^23"), (dict(q=0), -1, "required"), (dict(out=0), -1, "required"),
    (dict(q_seq_stride=1 << 23), -2, "strides"), (dict(v_seq_stride=-4), -2, "strides")])
def test_fwd_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_linattn_fwd", _fill(blocks, "mm_linattn_fwd_params", **{**SIZES, **PTRS, "out": 4096, **change}))
    assert rc == code and needle in msg, (rc, msg)


@pytest.mark.parametrize("change,code,needle", [
    (dict(dk=129), -2, "128"), (dict(dq=0), -1, "required"), (dict(dout=0), -1, "required"), (dict(dlog_decay=4096), -1, "workspace"),
    (dict(nheads=4, n_groups=2, workspace=4096, workspace_bytes=16), -1, "workspace"), (dict(do_seq_stride=1 << 22), -2, "strides")])
def test_bwd_refusals(blocks, change, code, needle):
    full = {**SIZES, **PTRS, "nheads": 1, "dout": 4096, "dq": 4096, "dk_out": 4096, "dv_out": 4096, **change}
    rc, msg = _call("mm_linattn_bwd", _fill(blocks, "mm_linattn_bwd_params", **full))
    assert rc == code and needle in msg, (rc, msg)


def test_nothing_to_do(blocks):
    assert _call("mm_linattn_fwd", _fill(blocks, "mm_linattn_fwd_params", **{**SIZES, "batch": 0}))[0] == 0
    assert _call("mm_linattn_fwd", _fill(blocks, "mm_linattn_fwd_params", **{**SIZES, "seqlen": 0}))[0] == 0
    size = {k: v for k, v in SIZES.items() if k != "seqlen"}
    assert _call("mm_linattn_update", _fill(blocks, "mm_linattn_update_params", **{**size, "batch": 0}))[0] == 0
    rc, msg = _call("mm_linattn_update", _fill(blocks, "mm_linattn_update_params", **size))
    assert rc == -1 and "required" in msg
    for name in ("mm_linattn_fwd", "mm_linattn_bwd", "mm_linattn_update", "mm_group_norm_fwd", "mm_group_norm_bwd"):
        assert _call(name, None)[0] == -1


NORM = dict(rows=2, channels=32, n_groups=2, itype=2, wtype=0, eps=1e-5, gate=0, x=4096, out=4096)


@pytest.mark.parametrize("change,code,needle", [
    (dict(itype=3), -1, "dtype"), (dict(rows=-1), -1, "negative"), (dict(n_groups=3), -1, "multiple"), (dict(n_groups=0), -1, "multiple"),
    (dict(channels=32770), -2, "16384"), (dict(eps=-1.0), -1, "eps"), (dict(gate=4), -1, "gate"), (dict(gate=1), -1, "z goes"),
    (dict(gate=3, z=4096), -1, "z goes"), (dict(x=0), -1, "required")])
def test_norm_refusals(blocks, change, code, needle):
    rc, msg = _call("mm_group_norm_fwd", _fill(blocks, "mm_group_norm_params", **{**NORM, **change}))
    assert rc == code and needle in msg, (rc, msg)


def test_norm_bwd_refusals(blocks):
    rc, msg = _call("mm_group_norm_bwd", _fill(blocks, "mm_group_norm_params", **NORM))
    assert rc == -1 and "dout" in msg
    rc, msg = _call("mm_group_norm_bwd", _fill(blocks, "mm_group_norm_params", **{**NORM, "dout": 4096, "dx": 4096, "dweight": 4096}))
    assert rc == -1 and "workspace" in msg
    assert _call("mm_group_norm_fwd", _fill(blocks, "mm_group_norm_params", **{**NORM, "rows": 0}))[0] == 0


def test_python_refusals_without_a_gpu():
    import torch
    from motif_mamba_amd import group_norm_fn, linear_attention_fn, linear_attention_update
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError):
        linear_attention_fn(x, x, x, torch.zeros(1, 2, 1))
    with pytest.raises(ValueError):
        linear_attention_fn(x, x, x[0], torch.zeros(1, 2, 1))
    with pytest.raises(RuntimeError):
        linear_attention_update(torch.zeros(1, 1, 8, 8), x[:, 0], x[:, 0], x[:, 0], torch.zeros(1, 1))
    with pytest.raises(RuntimeError):
        group_norm_fn(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        group_norm_fn(torch.zeros(2, 8), 2, z=torch.zeros(2, 8), activation="silu")
