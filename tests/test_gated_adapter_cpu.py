"""CPU tests of the C entry points of the gated layer, the row quantisation, the 8-bit
layer and the orthogonalised update: refusals, workspace sizes, structures."""
import ctypes as C
import os
import re

import pytest

from fusiongpu_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(4096)  # stands for a device pointer; refused calls never use it
OFF = C.c_void_p(4096 + 8)


def _status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def _linear(**kw):
    v = dict(rows=10, in_dim=8, out_dim=4, dtype=1, activation=0, x_stride=0, w_stride=0, residual_stride=0,
             pre_stride=0, y_stride=0, unaligned=0)
    v.update(kw)
    return _lib.LinearParams(*v.values())


def _orth(**kw):
    v = dict(batch=1, rows=10, cols=8, dtype=0, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, row_stride=0, batch_stride=0)
    v.update(kw)
    return _lib.OrthogonalizeParams(*v.values())


def test_structure_matches_the_header():
    h = open(os.path.join(ROOT, "include", "fusiongpu.h")).read()
    h = re.sub(r"/\*.*?\*/", "", h, flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} fg_orthogonalize_params;", h).group(1)
    types = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
    assert list(_lib.OrthogonalizeParams._fields_) == [(f, types[t]) for t, f in re.findall(r"(\w+)\s+(\w+);", body)]


def _gated(p, x=P, w=P, bias=None, pre=None, y=P, ws=P, n=1 << 40):
    return _status("fg_gated_linear", C.byref(p), x, w, bias, pre, y, ws, n, None)


def _gated_backward(p, dy=P, x=P, w=P, pre=P, dx=P, dw=P, db=P, ws=P, n=1 << 40):
    return _status("fg_gated_linear_backward", C.byref(p), dy, x, w, pre, dx, dw, db, ws, n, None)


BAD = [dict(rows=-1), dict(in_dim=0), dict(out_dim=0), dict(dtype=3), dict(activation=4), dict(x_stride=7), dict(w_stride=7),
       dict(y_stride=3), dict(unaligned=8)]


@pytest.mark.parametrize("kw", BAD + [dict(pre_stride=7), dict(residual_stride=8)])
def test_gated_refuses(kw):
    p, n = _linear(**kw), C.c_size_t()
    assert _gated(p) == 1 and _gated_backward(p) == 1
    for name in ("fg_gated_linear_workspace_size", "fg_gated_linear_backward_workspace_size"):
        assert _status(name, C.byref(p), C.byref(n)) == 1


def test_gated_arguments():
    for kw in (dict(in_dim=32769), dict(out_dim=(1 << 29) + 1)):
        p, n = _linear(**kw), C.c_size_t()
        assert _gated(p) == 4 and _gated_backward(p) == 4
        assert _status("fg_gated_linear_workspace_size", C.byref(p), C.byref(n)) == 4
    p = _linear()
    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(x=OFF), dict(w=OFF)):
        assert _gated(p, **kw) == 1, kw
    for kw in (dict(dy=None), dict(pre=None), dict(x=None), dict(w=None), dict(x=OFF), dict(w=OFF)):
        assert _gated_backward(p, **kw) == 1, kw
    big = _linear(rows=500, in_dim=72, out_dim=40)
    n = _lib.size_query("fg_gated_linear_backward_workspace_size", C.byref(big))
    assert n >= 500 * 80 * 2 * 2  # two parts of dz and dp
    for ws, b in ((None, n), (P, n - 1), (OFF, n)):
        assert _gated_backward(big, ws=ws, n=b) == 3
    odd = _linear(rows=500, in_dim=71, out_dim=40)
    n = _lib.size_query("fg_gated_linear_workspace_size", C.byref(odd))
    assert n >= (500 + 80) * 72 * 2
    assert _gated(odd, ws=None, n=0) == 3
    # the activation's place next to 16 bytes is asked for by name
    named = _lib.size_query("fg_gated_linear_workspace_size", C.byref(_linear(rows=500, in_dim=72, out_dim=40, unaligned=3)))
    assert named >= (500 + 80) * 72 * 2 and _lib.size_query("fg_gated_linear_workspace_size", C.byref(big)) == 0
    empty = _linear(rows=0)
    assert _gated(empty, x=None, w=None, y=None) == 0
    for name in ("fg_gated_linear_workspace_size", "fg_gated_linear_backward_workspace_size"):
        assert _status(name, C.byref(p), None) == 1


def _int8(p, x=P, xs=P, w=P, ws=P, bias=None, res=None, y=P, room=P, n=1 << 40):
    return _status("fg_linear_int8", C.byref(p), x, xs, w, ws, bias, res, y, room, n, None)


@pytest.mark.parametrize("kw", BAD + [dict(residual_stride=3), dict(pre_stride=4)])
def test_int8_refuses(kw):
    p, n = _linear(**kw), C.c_size_t()
    assert _int8(p) == 1
    assert _status("fg_linear_int8_workspace_size", C.byref(p), C.byref(n)) == 1


def test_int8_arguments():
    p = _linear(rows=500, in_dim=80, out_dim=40)
    assert _lib.size_query("fg_linear_int8_workspace_size", C.byref(p)) == 0
    for kw in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(x=OFF), dict(w=OFF)):
        assert _int8(p, **kw) == 1, kw
    assert _int8(_linear(in_dim=131072)) == 4
    off = _linear(rows=500, in_dim=81, out_dim=40)
    n = _lib.size_query("fg_linear_int8_workspace_size", C.byref(off))
    assert n >= 540 * 96
    assert _int8(off, room=None, n=0) == 3 and _int8(off, n=n - 1) == 3
    assert _int8(_linear(rows=0), x=None, xs=None, w=None, ws=None, y=None) == 0


def test_quantize_refuses():
    ok = dict(x=P, dtype=0, rows=4, dim=8, ldx=0, q=P, ldq=0, scale=P, s=None)

    def st(**kw):
        return _status("fg_quantize_rows", *{**ok, **kw}.values())

    for kw in (dict(dtype=3), dict(rows=-1), dict(dim=0), dict(ldx=7), dict(ldq=7), dict(x=None), dict(q=None), dict(scale=None)):
        assert st(**kw) == 1, kw
    assert st(dim=(1 << 30) + 1) == 4
    assert st(rows=0, x=None, q=None, scale=None) == 0


@pytest.mark.parametrize("kw,want", [(dict(batch=-1), 1), (dict(rows=0), 1), (dict(cols=0), 1), (dict(dtype=3), 1),
                                     (dict(steps=-1), 1), (dict(steps=101), 1), (dict(eps=-1.0), 1),
                                     (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1), (dict(a=float("nan")), 1),
                                     (dict(b=-16.5), 1), (dict(c=float("inf")), 1), (dict(row_stride=7), 1),
                                     (dict(batch_stride=-1), 1), (dict(batch=65536), 4), (dict(rows=32769), 4),
                                     (dict(cols=32769), 4)])
def test_orthogonalize_refuses(kw, want):
    p, n = _orth(**kw), C.c_size_t()
    assert _status("fg_orthogonalize", C.byref(p), P, P, P, 1 << 40, None) == want
    assert _status("fg_orthogonalize_workspace_size", C.byref(p), C.byref(n)) == want


def test_orthogonalize_arguments():
    p = _orth(rows=300, cols=200)
    n = _lib.size_query("fg_orthogonalize_workspace_size", C.byref(p))
    assert n >= 4 * (2 * 300 * 200 + 2 * 200 * 200)
    for g, out in ((None, P), (P, None)):
        assert _status("fg_orthogonalize", C.byref(p), g, out, P, n, None) == 1
    for ws, b in ((None, n), (P, n - 1), (OFF, n)):
        assert _status("fg_orthogonalize", C.byref(p), P, P, ws, b, None) == 3
    assert _status("fg_orthogonalize", None, P, P, P, n, None) == 1
    assert _status("fg_orthogonalize_workspace_size", C.byref(p), None) == 1
    assert _status("fg_orthogonalize", C.byref(_orth(batch=0)), None, None, None, 0, None) == 0


def test_new_operators_take_their_tensors_by_name():
    torch = pytest.importorskip("torch")
    from fusiongpu_b200 import adapter
    x = torch.zeros(2, 4)
    calls = {"gated_linear": dict(x=x, w=x), "gated_linear_backward": dict(dy=x, x=x, w=x, pre=x), "quantize_rows": dict(x=x),
             "linear_int8": dict(x=x, x_scale=x[0], w=x, w_scale=x[0]), "orthogonalize": dict(g=x)}
    for name, kw in calls.items():
        with pytest.raises(ValueError, match="CUDA"):
            getattr(adapter, name)(**kw)
        with pytest.raises(ValueError, match="CUDA"):
            getattr(adapter, name)(*kw.values())
        first = next(iter(kw))
        with pytest.raises(TypeError, match=first):
            getattr(adapter, name)(**{k: v for k, v in kw.items() if k != first})


def test_vector_stores_of_the_update_are_aligned():
    src = open(os.path.join(ROOT, "fusiongpu_b200", "csrc", "orth.cu")).read()
    found = re.findall(r"extern __shared__ (.*?)\w+\[\];", src)
    assert found and all("__align__" in d for d in found)
