"""CPU tests of the query adapter's C entry points: refusals and workspace
sizes (host logic; nothing is launched) and the ctypes structures."""
import ctypes as C
import os
import re

import pytest

from fusiongpu_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = C.c_void_p(4096)  # stands for a device pointer; refused calls never use it


def _struct_fields(name):
    h = open(os.path.join(ROOT, "include", "fusiongpu.h")).read()
    h = re.sub(r"/\*.*?\*/", "", h, flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", h).group(1)
    types = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
    return [(f, types[t]) for t, f in re.findall(r"(\w+)\s+(\w+);", body)]


@pytest.mark.parametrize("name,cls", [("fg_linear_params", _lib.LinearParams),
                                      ("fg_preference_params", _lib.PreferenceParams)])
def test_structures_match_the_header(name, cls):
    assert list(cls._fields_) == _struct_fields(name)


def _linear(**kw):
    v = dict(rows=10, in_dim=8, out_dim=4, dtype=0, activation=0, x_stride=0, w_stride=0, residual_stride=0,
             pre_stride=0, y_stride=0)
    v.update(kw)
    return _lib.LinearParams(*v.values())


def _status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def _message():
    return _lib.lib().fg_last_error().decode()


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(in_dim=0), dict(out_dim=0), dict(dtype=3), dict(dtype=-1),
                                dict(activation=4), dict(x_stride=7), dict(w_stride=7), dict(y_stride=3),
                                dict(pre_stride=3), dict(residual_stride=-4)])
def test_linear_refuses(kw):
    p, n = _linear(**kw), C.c_size_t()
    assert _status("fg_linear", C.byref(p), P, P, None, None, None, P, None, 0, None) == 1 and _message()
    assert _status("fg_linear_workspace_size", C.byref(p), C.byref(n)) == 1
    assert _status("fg_linear_backward", C.byref(p), P, P, P, P, P, P, P, None, 0, None) == 1
    assert _status("fg_linear_backward_workspace_size", C.byref(p), C.byref(n)) == 1


def test_linear_null_arguments():
    p = _linear(activation=2)
    assert _status("fg_linear", None, P, P, None, None, None, P, None, 0, None) == 1
    for x, w, y in ((None, P, P), (P, None, P), (P, P, None)):
        assert _status("fg_linear", C.byref(p), x, w, None, None, None, y, None, 0, None) == 1
    assert _status("fg_linear_workspace_size", C.byref(p), None) == 1
    # dy; pre with an activation; w for dx; x for dw
    for dy, x, w, pre in ((None, P, P, P), (P, P, P, None), (P, P, None, P), (P, None, P, P)):
        assert _status("fg_linear_backward", C.byref(p), dy, x, w, pre, P, P, P, P, 1 << 40, None) == 1
    n = _lib.size_query("fg_linear_backward_workspace_size", C.byref(p))
    assert n >= 10 * 4 * 4  # dz
    for ws, b in ((None, n), (P, n - 1), (C.c_void_p(4096 + 8), n)):
        assert _status("fg_linear_backward", C.byref(p), P, P, P, P, P, P, P, ws, b, None) == 3
    empty = _linear(rows=0)
    assert _status("fg_linear", C.byref(empty), None, None, None, None, None, None, None, 0, None) == 0


def test_layer_norm_refuses():
    ok = dict(x=P, dtype=0, rows=4, dim=8, ldx=0, w=None, b=None, pd=0, eps=1e-5, y=P, ldy=0, m=None, r=None, s=None)

    def st(**kw):
        return _status("fg_layer_norm", *{**ok, **kw}.values())

    for kw in (dict(dtype=3), dict(pd=1), dict(dtype=1, pd=2), dict(rows=-1), dict(dim=0), dict(ldx=7), dict(ldy=-8),
               dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None), dict(m=P), dict(r=P)):
        assert st(**kw) == 1, kw
    assert st(dim=16385) == 4
    assert st(rows=0, x=None, y=None) == 0
    n = _lib.size_query("fg_layer_norm_backward_workspace_size", 1000, 768)
    assert n >= 2 * 768 * 4
    ok = dict(dy=P, lddy=0, x=P, dtype=1, rows=4, dim=8, ldx=0, w=P, pd=0, m=P, r=P, dx=P, lddx=0, dw=P, db=P, ws=P,
              wb=1 << 40, s=None)

    def st(**kw):
        return _status("fg_layer_norm_backward", *{**ok, **kw}.values())

    for kw in (dict(dtype=7), dict(pd=2), dict(rows=-1), dict(dim=-3), dict(ldx=3), dict(lddy=3), dict(lddx=3),
               dict(dy=None), dict(x=None), dict(m=None), dict(r=None)):
        assert st(**kw) == 1, kw
    assert st(dim=20000) == 4
    for kw in (dict(ws=None), dict(wb=8), dict(ws=C.c_void_p(4097))):
        assert st(**kw) == 3, kw


def test_preference_refuses():
    base = dict(nq=4, dim=8, dtype=0, base_dtype=3, nbase=10, n_pairs=6, metric=0, beta=1.0, label_smoothing=0.0,
                query_stride=0, ref_stride=0, dq_stride=0)

    def st(args=(P, P, P, P, P, P, P, P, P, P), **kw):
        p = _lib.PreferenceParams(*{**base, **kw}.values())
        return _status("fg_preference_loss", C.byref(p), *args, None)

    for kw in (dict(nq=-1), dict(dim=0), dict(dtype=3), dict(base_dtype=4), dict(nbase=-1), dict(n_pairs=-1),
               dict(metric=2), dict(beta=0.0), dict(beta=-1.0), dict(beta=float("inf")), dict(beta=float("nan")),
               dict(label_smoothing=0.51), dict(label_smoothing=-0.01), dict(query_stride=7), dict(ref_stride=7),
               dict(dq_stride=-1)):
        assert st(**kw) == 1, kw
    assert st(dim=16385) == 4
    full = [P] * 10
    for k in (0, 2, 3, 4, 5, 7):  # queries, base, offsets, pos, neg, losses
        assert st(full[:k] + [None] + full[k + 1:]) == 1, k
    assert st([None] * 10, nq=0) == 0
    assert _status("fg_preference_loss", None, *full, None) == 1


def test_vector_stores_to_shared_memory_are_aligned():
    """Dynamic shared memory that kernels access 16 bytes at a time is declared so: the
    compiler places an array of float on 4 bytes where nothing asks for more."""
    for name in ("norm.cu", "linear_tc.cu"):
        src = open(os.path.join(ROOT, "fusiongpu_b200", "csrc", name)).read()
        found = re.findall(r"extern __shared__ (.*?)\w+\[\];", src)
        assert found and all("__align__" in d for d in found), (name, found)


@pytest.mark.parametrize("out_dim,in_dim", [(1536, 768), (2048, 2048), (264, 520), (64, 64)])
def test_deep_products_are_cut_into_parts(out_dim, in_dim):
    """dw of 16-bit layers sums over the rows: 32,768 to an accumulator at most, in up to
    eight parts of a cluster, which need no workspace, or in parts that lie in it."""
    deep = 512 * 64
    rows = sorted({deep * 2 ** e + d for e in range(0, 13) for d in (-1, 0, 1, 56, 63, 64, 65, 448, 449, 960, 1000)} |
                  {deep * m + 1 for m in range(1, 40)})
    for r in rows:
        p = _linear(rows=r, in_dim=in_dim, out_dim=out_dim, dtype=2)
        n = _lib.size_query("fg_linear_backward_workspace_size", C.byref(p))
        parts = n // ((out_dim + 255) // 256 * 256 * in_dim * 4)
        blocks = (r + 63) // 64
        assert blocks <= 512 * (parts if parts else 8), (r, parts)
        assert parts <= max(32, 2 * blocks / 512), (r, parts)  # and no more than that asks for


def test_linear_room_for_operands_off_16_bytes():
    """Their copies lie in the workspace; strides off 16 bytes and float32 are copied anyway."""
    for name, bits in (("fg_linear_workspace_size", 3), ("fg_linear_backward_workspace_size", 7)):
        for dtype in (1, 2):
            size = [_lib.size_query(name, C.byref(_linear(rows=500, in_dim=72, out_dim=40, dtype=dtype, unaligned=b)))
                    for b in range(bits + 1)]
            for b in range(bits + 1):
                room = sum(n for k, n in enumerate((500 * 72 * 2, 40 * 72 * 2, 500 * 40 * 2)) if b >> k & 1)
                assert room <= size[b] - size[0] <= room + 3 * 256
        both = [_lib.size_query(name, C.byref(_linear(rows=500, in_dim=72, out_dim=40, dtype=1, x_stride=73, w_stride=75,
                                                      y_stride=41, unaligned=b))) for b in (0, bits)]
        assert both[0] == both[1]
    for bits in (8, -1):
        p, n = _linear(unaligned=bits), C.c_size_t()
        assert _status("fg_linear_workspace_size", C.byref(p), C.byref(n)) == 1


def test_operators_take_their_tensors_by_name():
    """Called with keywords alone, each operator gets as far as its tensors, which here are
    not on a GPU; a missing one is named."""
    torch = pytest.importorskip("torch")
    from fusiongpu_b200 import adapter
    x = torch.zeros(2, 4)
    calls = {"layer_norm": dict(x=x), "layer_norm_backward": dict(dy=x, x=x, mean=x[:, 0], rstd=x[:, 0]),
             "linear": dict(x=x, w=x), "linear_backward": dict(dy=x, x=x, w=x),
             "preference_loss": dict(queries=x, base=x, offsets=x, pos_ids=x, neg_ids=x)}
    for name, kw in calls.items():
        with pytest.raises(ValueError, match="CUDA"):
            getattr(adapter, name)(**kw)
        with pytest.raises(ValueError, match="CUDA"):
            getattr(adapter, name)(*kw.values())
        first = next(iter(kw))
        with pytest.raises(TypeError, match=first):
            getattr(adapter, name)(**{k: v for k, v in kw.items() if k != first})
