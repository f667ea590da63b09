"""The training operators' refusals and host logic (no GPU): the Python layer's checks
raise before any launch, the C ABI's return SRBCRS_EINVAL with a message, struct layouts and constants
match include/srbcrs.h, and workspace sizes follow the shapes."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from mask_amd import _capi

ROOT = Path(__file__).resolve().parent.parent
INF, NAN = float("inf"), float("nan")


def _norm(**kw):
    d = dict(batch=2, length=10, channels=32, groups=4, batch_x=320, ld_x=32, batch_dy=320, ld_dy=32, dtype=0,
             param_dtype=0, activation=0, eps=1e-5)
    d.update(kw)
    return _capi.NormDesc(*(d[f] for f, _ in _capi.NormDesc._fields_))


def _xent(**kw):
    d = dict(rows=10, dim=64, classes=100, ld_h=64, ld_w=64, ignore_index=-100, dtype=0, reduction=1)
    d.update(kw)
    return _capi.XentDesc(*(d[f] for f, _ in _capi.XentDesc._fields_))


def _ortho(**kw):
    d = dict(batch=1, rows=20, cols=30, batch_g=600, ld_g=30, dtype=0, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7)
    d.update(kw)
    return _capi.OrthoDesc(*(d[f] for f, _ in _capi.OrthoDesc._fields_))


def _size_of(fn, *args):
    n = ctypes.c_size_t(0)
    rc = fn(*args, ctypes.byref(n))
    return rc, n.value


def _norm_size(d, backward=0):
    return _size_of(_capi.lib().srbcrs_group_norm_workspace, ctypes.byref(d), backward)


def _xent_size(d, backward=0, h=0, w=0):
    return _size_of(_capi.lib().srbcrs_linear_xent_workspace, ctypes.byref(d), h, w, backward)


def _ortho_size(d):
    return _size_of(_capi.lib().srbcrs_orthogonalize_workspace, ctypes.byref(d))


def _error():
    return _capi.lib().srbcrs_last_error().decode()


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=3), "dtype"), (dict(param_dtype=-1), "param_dtype"), (dict(groups=0), "groups"), (dict(groups=5), "groups"),
    (dict(groups=-4), "groups"), (dict(batch=-1), "batch"), (dict(length=-1), "length"), (dict(channels=1 << 21, groups=1), "channels"),
    (dict(batch=1 << 30, length=1 << 30), "too many"), (dict(activation=4), "activation"), (dict(eps=-1.0), "eps"),
    (dict(eps=NAN), "eps"), (dict(eps=INF), "eps"), (dict(ld_x=-32), "ld_x"), (dict(batch_x=-1), "batch_x")])
def test_group_norm_descriptions_are_refused(kw, message):
    rc, _ = _norm_size(_norm(**kw))
    assert rc == _capi.SRBCRS_EINVAL and message in _error()


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(classes=0), "class"),
    (dict(classes=1 << 31), "classes"), (dict(dim=0), "feature"), (dict(dim=1 << 25), "dim"), (dict(reduction=3), "reduction"),
    (dict(ld_h=-1), "ld_h"), (dict(ld_w=-1), "ld_w")])
def test_cross_entropy_descriptions_are_refused(kw, message):
    rc, _ = _xent_size(_xent(**kw))
    assert rc == _capi.SRBCRS_EINVAL and message in _error()


@pytest.mark.parametrize("kw, message", [
    (dict(dtype=-1), "dtype"), (dict(batch=65536), "batch"), (dict(rows=-1), "rows"), (dict(cols=1 << 25), "cols"),
    (dict(steps=0), "steps"), (dict(steps=101), "steps"), (dict(a=NAN), "coefficients"), (dict(a=0, b=0, c=0), "coefficients"),
    (dict(c=INF), "coefficients"), (dict(a=2000.0), "coefficients"), (dict(eps=-1e-9), "eps"), (dict(ld_g=-30), "strides")])
def test_orthogonalize_descriptions_are_refused(kw, message):
    rc, _ = _ortho_size(_ortho(**kw))
    assert rc == _capi.SRBCRS_EINVAL and message in _error()


def test_null_and_short_arguments_are_refused():
    """Before any HIP call: null pointers, misaligned ones, workspaces that are
    missing, misaligned or a byte short."""
    L = _capi.lib()
    p = 1 << 20     # an aligned address that is never touched

    def refused(rc, message):
        assert rc == _capi.SRBCRS_EINVAL and message in _error(), _error()

    d = _norm()
    n = _norm_size(d)[1]
    r = ctypes.byref(d)
    refused(L.srbcrs_group_norm(None, p, p, p, p, p, p, n, None), "desc is NULL")
    refused(L.srbcrs_group_norm(r, None, p, p, p, p, p, n, None), "x is NULL")
    refused(L.srbcrs_group_norm(r, p, p, p, None, p, p, n, None), "y is NULL")
    refused(L.srbcrs_group_norm(r, p, p, p, p, None, p, n, None), "stats is NULL")
    refused(L.srbcrs_group_norm(r, p + 2, p, p, p, p, p, n, None), "aligned")
    assert n == 1                                # a short sample needs no workspace
    d = _norm(batch=1, length=100000)
    n = _norm_size(d)[1]
    r = ctypes.byref(d)
    refused(L.srbcrs_group_norm(r, p, p, p, p, p, None, n, None), "workspace is NULL")
    refused(L.srbcrs_group_norm(r, p, p, p, p, p, p + 128, n, None), "256-byte")
    refused(L.srbcrs_group_norm(r, p, p, p, p, p, p, n - 1, None), "too small")
    n = _norm_size(d, 1)[1]
    refused(L.srbcrs_group_norm_backward(r, None, p, p, p, p, p, p, p, p, n, None), "dy is NULL")
    refused(L.srbcrs_group_norm_backward(r, p, p, p, p, p, None, p, p, p, n, None), "dx is NULL")
    refused(L.srbcrs_group_norm_backward(r, p, p, p, p, p, p, p, p, p, n - 1, None), "too small")
    d = _xent()
    r = ctypes.byref(d)
    n = _xent_size(d)[1]
    refused(L.srbcrs_linear_xent(r, None, p, p, p, p, p, n, None), "h is NULL")
    refused(L.srbcrs_linear_xent(r, p, p, None, p, p, p, n, None), "target is NULL")
    refused(L.srbcrs_linear_xent(r, p, p + 1, p, p, p, p, n, None), "aligned")
    refused(L.srbcrs_linear_xent(r, p, p, p, p, p, p, n - 1, None), "too small")
    n = _xent_size(d, 1)[1]
    refused(L.srbcrs_linear_xent_backward(r, p, p, p, p, None, p, p, p, n, None), "dloss is NULL")
    refused(L.srbcrs_linear_xent_backward(r, p, p, p, p, p, p, p, p, n - 1, None), "too small")
    assert L.srbcrs_linear_xent_backward(r, p, p, p, p, p, None, None, p, n, None) == _capi.SRBCRS_OK   # nothing is wanted
    d = _ortho()
    r = ctypes.byref(d)
    n = _ortho_size(d)[1]
    refused(L.srbcrs_orthogonalize(r, None, p, p, n, None), "g is NULL")
    refused(L.srbcrs_orthogonalize(r, p, None, p, n, None), "out is NULL")
    assert n == 1                                # a small matrix needs no workspace
    d = _ortho(rows=100, cols=3000, ld_g=3000, batch_g=300000)
    r = ctypes.byref(d)
    n = _ortho_size(d)[1]
    refused(L.srbcrs_orthogonalize(r, p, p, None, n, None), "workspace is NULL")
    refused(L.srbcrs_orthogonalize(r, p, p, p, n - 1, None), "too small")
    refused(L.srbcrs_orthogonalize_workspace(r, None), "bytes is NULL")


def test_empty_shapes_need_no_pointer():
    L = _capi.lib()
    for kw in (dict(batch=0), dict(length=0), dict(channels=0)):
        d = _norm(**kw)
        assert _norm_size(d) == (_capi.SRBCRS_OK, 1)
        assert L.srbcrs_group_norm(ctypes.byref(d), None, None, None, None, None, None, 0, None) == _capi.SRBCRS_OK
    d = _ortho(rows=0)
    assert L.srbcrs_orthogonalize(ctypes.byref(d), None, None, None, 0, None) == _capi.SRBCRS_OK
    assert _xent_size(_xent(rows=0))[1] == 1


def test_cross_entropy_workspace_stays_below_the_logits():
    """The point of the operator: 64 thousand rows over 128 thousand classes have
    34 GB of logits in 32 bits.  16-bit operands that can be read where they are need no copy."""
    logits = 4 * 65536 * 131072
    for dtype in (0, 1, 2):
        for backward in (0, 1):
            rc, n = _xent_size(_xent(rows=65536, classes=131072, dim=1024, ld_h=1024, ld_w=1024, dtype=dtype), backward)
            assert rc == 0 and n < logits / 8
    d = _xent(rows=512, classes=131072, dim=1024, ld_h=1024, ld_w=1024, dtype=1)
    assert _xent_size(d)[1] + 131072 * 1024 * 2 <= _xent_size(d, w=8)[1]      # 8 bytes off: a copy of the weight


def test_descriptions_match_the_header(tmp_path):
    """Field offsets, sizes and constants against a compiled program."""
    structs = {"srbcrs_norm_desc": _capi.NormDesc, "srbcrs_xent_desc": _capi.XentDesc, "srbcrs_ortho_desc": _capi.OrthoDesc}
    lines = []
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "srbcrs.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{ROOT / 'include'}", "-o", str(exe), str(src)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(got[f"{c} size"]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{c} {f}"]) == getattr(py, f).offset, (c, f)
    text = (ROOT / "include" / "srbcrs.h").read_text()
    defs = {k: int(v) for k, v in re.findall(r"#define (SRBCRS_[A-Z_0-9]+) \(?(-?\d+)\)?", text)}
    assert (defs["SRBCRS_F32"], defs["SRBCRS_BF16"], defs["SRBCRS_F16"]) == tuple(_capi.DTYPE_CODES[k] for k in ("float32", "bfloat16", "float16"))
    for k, v in _capi.ACTIVATIONS.items():
        assert defs[f"SRBCRS_ACT_{k.upper()}"] == v
    for k, v in _capi.REDUCTIONS.items():
        assert defs[f"SRBCRS_REDUCE_{k.upper()}"] == v


def test_host_tensors_are_refused():
    """There is no other implementation: a host tensor's address would reach the GPU."""
    torch = pytest.importorskip("torch")
    from mask_amd import ops
    x = torch.ones(4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.orthogonalize(x)
    with pytest.raises(TypeError, match="torch tensor"):
        ops.orthogonalize([[1.0]])


def test_group_norm_workspace_of_many_short_samples():
    """Split samples of one chunk each have few parts a group, however many of them the parameters' gradients are
    joined from: the parts, two means a group and at most 64 shares of the parameters."""
    batch, length, channels, groups = 8192, 100, 320, 32
    d = _norm(batch=batch, length=length, channels=channels, groups=groups, batch_x=length * channels, ld_x=channels,
              batch_dy=length * channels, ld_dy=channels)
    rc, n = _norm_size(d, 1)
    assert rc == 0 and n <= 8 * (batch * channels + 2 * batch * groups + 64 * channels) + 4 * 256
