"""Host side of layer norm and linear cross entropy on the CPU: the C entry
points' checks (before anything is enqueued), workspace sizes, the Python
layer's refusals, and the float64 forms the GPU tests compare with."""
import ctypes
import os
import re

import pytest
import torch

from tests._ops_util import lce_ref, norm_ref
from testtimeideas_amd import _lib
from testtimeideas_amd.ttt_e2e import LayerNorm, layer_norm, linear_cross_entropy

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "ttt_ops.h")
P = 0x100000  # an aligned address that is never read


class Norm(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("param_dtype", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("eps", ctypes.c_float)]


class Lce(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("reduction", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ignore_index", ctypes.c_int64)]


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64)]


def _c():
    lib = _lib.load()
    for n in ("ttt_norm_workspace_size", "ttt_lce_workspace_size"):
        getattr(lib, n).restype = ctypes.c_int64
    return lib


def _rows(stride, at=P):
    return ctypes.byref(Rows(at, stride))


def _vp(x):
    return None if x is None else ctypes.c_void_p(x)


def _i(n):
    return ctypes.c_int64(n)


def test_library_exports_the_declared_entry_points():
    text = open(HEADER).read()
    names = set(re.findall(r"^[A-Za-z_][\w\s\*]*?\b(ttt_\w+)\s*\(", text, flags=re.M))
    assert {"ttt_norm_fwd", "ttt_norm_bwd", "ttt_norm_gg", "ttt_lce_fwd", "ttt_lce_bwd", "ttt_lce_gg"} <= names
    assert all(hasattr(_c(), n) for n in names)


def _norm_fwd(x=None, y=None, mean=P, rstd=P, w=P, b=P, **kw):
    d = dict(dtype=1, param_dtype=1, rows=4, cols=64, eps=1e-5)
    d.update(kw)
    pr = Norm(**d)
    s = d["cols"]
    return _c().ttt_norm_fwd(ctypes.byref(pr), x or _rows(s), _vp(w), _vp(b), y or _rows(s), _vp(mean), _vp(rstd), None)


def test_norm_refusals():
    lib = _c()
    assert _norm_fwd(dtype=5) == 2 and b"dtype" in lib.ttt_last_error()
    assert _norm_fwd(param_dtype=0) == 2
    assert _norm_fwd(rows=0) == 1
    assert _norm_fwd(rows=1 << 31) == 1
    assert _norm_fwd(cols=0) == 2
    assert _norm_fwd(cols=32769) == 2
    assert _norm_fwd(dtype=2, param_dtype=2, cols=16385) == 2
    assert _norm_fwd(x=_rows(63)) == 1 and b"stride" in lib.ttt_last_error()
    assert _norm_fwd(x=_rows(64, 0)) == 1
    assert _norm_fwd(x=_rows(64, P + 1)) == 1
    assert _norm_fwd(mean=None) == 1
    assert lib.ttt_norm_fwd(None, None, None, None, None, None, None, None) == 1
    pr = ctypes.byref(Norm(1, 1, 4, 64, 1e-5))
    r = _rows(64)
    # no statistics; no workspace for the parameters' sums
    assert lib.ttt_norm_bwd(pr, r, None, r, None, _vp(P), r, None, None, None, _i(0), None) == 1
    assert lib.ttt_norm_bwd(pr, r, None, r, _vp(P), _vp(P), r, _vp(P), None, None, _i(0), None) == 4
    assert lib.ttt_norm_gg(pr, r, None, r, _vp(P), _vp(P), r, None, None, r, _vp(P), r, _vp(P), _i(8), None) == 4
    # nothing asked for: nothing is enqueued
    assert lib.ttt_norm_bwd(pr, r, None, r, _vp(P), _vp(P), None, None, None, None, _i(0), None) == 0


def test_norm_workspace():
    lib = _c()
    size = lambda *a: lib.ttt_norm_workspace_size(ctypes.byref(Norm(*a, 1e-5)))  # noqa: E731
    assert size(1, 1, 1, 64) == 2 * 64 * 4
    assert size(1, 1, 1 << 20, 64) == size(1, 1, 1 << 24, 64)  # bounded by the workgroups
    assert size(9, 1, 1, 64) == -1


def _lce(name, ws=P, wsn=1 << 50, x=None, w=None, **kw):
    d = dict(dtype=1, reduction=2, rows=4, cols=64, vocab=100, ignore_index=-100)
    d.update(kw)
    pr, s, lib = ctypes.byref(Lce(**d)), d["cols"], _c()
    x, w = x or _rows(s), w or _rows(s)
    t = _vp(P)
    if name == "fwd":
        return lib.ttt_lce_fwd(pr, x, w, t, None, _vp(P), _vp(P), _vp(ws), _i(wsn), None)
    if name == "bwd":
        return lib.ttt_lce_bwd(pr, x, w, t, None, _vp(P), _vp(P), _rows(s), _rows(s), None, _vp(ws), _i(wsn),
                               None)
    return lib.ttt_lce_gg(pr, x, w, t, None, _vp(P), _vp(P), None, None, None, _rows(s), _rows(s), None, _vp(ws),
                          _i(wsn), None)


def test_lce_refusals():
    lib = _c()
    for name in ("fwd", "bwd", "gg"):
        assert _lce(name, dtype=4) == 2
        assert _lce(name, reduction=3) == 1
        assert _lce(name, rows=0) == 1
        assert _lce(name, rows=(1 << 22) + 1) == 1
        assert _lce(name, vocab=0) == 1
        assert _lce(name, vocab=(1 << 22) + 1) == 1
        assert _lce(name, cols=0) == 1
        assert _lce(name, cols=(1 << 16) + 8) == 1
        assert _lce(name, x=_rows(60)) == 1
        assert _lce(name, x=_rows(68)) == 1 and b"aligned" in lib.ttt_last_error()
        assert _lce(name, w=_rows(64, P + 8)) == 1
        assert _lce(name, w=_rows((1 << 22) + 8)) == 1
    assert _lce("fwd", ws=None) == 4 and _lce("bwd", wsn=64) == 4
    assert _lce("gg") == 1 and b"cotangent" in lib.ttt_last_error()
    assert lib.ttt_lce_fwd(None, None, None, None, None, None, None, None, _i(0), None) == 1


def test_lce_workspace_does_not_grow_with_the_logits():
    """Past a piece's size, the workspace is that of a piece."""
    size = lambda v, e: _c().ttt_lce_workspace_size(ctypes.byref(Lce(1, 2, 8192, 512, v, -100)), e)  # noqa: E731
    assert all(size(1 << 22, e) <= 1.1 * size(1 << 18, e) for e in (0, 1, 2))
    assert size(1 << 22, 1) < 8192 * (1 << 22) * 2 / 64
    assert size(0, 1) == -1 and size(64, 3) == -1


def test_python_refusals():
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear_cross_entropy(x, w, t)
    m = torch.device("meta")
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        LayerNorm(8)(torch.zeros(4, 8, device=m))
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm((4, 8))
    with pytest.raises(ValueError, match="does not end in"):
        LayerNorm(8)(torch.zeros(4, 9))


def test_float64_forms_are_the_definitions_gradients():
    """norm_ref and lce_ref against autograd of the definitions."""
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy, a, cw, cb = rn(5, 9), rn(9), rn(9), rn(5, 9), rn(5, 9), rn(9), rn(9)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, dy)]
    y = torch.nn.functional.layer_norm(leaves[0], (9,), leaves[1], leaves[2], 1e-5)
    first = torch.autograd.grad(y, leaves[:3], leaves[3], create_graph=True)
    second = torch.autograd.grad(first, (leaves[0], leaves[1], leaves[3]), (a, cw, cb))
    ref, _ = norm_ref(x, w, b, 1e-5, dy, a, cw, cb)
    for name, v in zip(("y", "dx", "dw", "db", "gx", "gw", "gdy"), (y, *first, *second)):
        assert torch.allclose(ref[name], v, rtol=1e-10, atol=1e-12), name

    x, w, a, b = rn(6, 5), rn(11, 5), rn(6, 5), rn(11, 5)
    t = torch.randint(0, 11, (6,), generator=g)
    wt = torch.tensor([1.0, 0.0, 0.5, 1.0, 0.0, 2.0], dtype=torch.float64)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    up = torch.tensor(1.7, dtype=torch.float64, requires_grad=True)
    loss = (torch.nn.functional.cross_entropy(lx @ lw.t(), t, reduction="none") * wt).sum() / wt.sum()
    first = torch.autograd.grad(loss, (lx, lw), up, create_graph=True)
    second = torch.autograd.grad(first, (lx, lw, up), (a, b))
    ref, _ = lce_ref(x, w, t, wt, 1.7, 1 / float(wt.sum()), torch.float32, a, b)
    for name, v in zip(("loss", "dx", "dw", "gx", "gw", "gloss"), (loss, *first, *second)):
        assert torch.allclose(ref[name], v, rtol=1e-10, atol=1e-12), name
