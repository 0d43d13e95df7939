"""Query adapter: a small model between an embedding model and the search, and
its training on preferences over the index's documents.

The reference searches the queries as they are given (search_pipeline.cu:594);
this is what a user of an index puts before that call to fit it to other
queries without re-embedding and re-building it.  :class:`QueryAdapter` is the
residual block

    adapted = q + w2 act(w1 layer_norm(q) + b1) + b2

or, gated, with act(z) * p for [z p] = w1 layer_norm(q) + b1 in the inner layer's
place.  Its operators (:func:`layer_norm`, :func:`linear`, :func:`gated_linear`,
:func:`preference_loss` and the gradients) are the package's own sm_100a kernels
behind the C ABI (fg_layer_norm, fg_linear, fg_gated_linear, fg_preference_loss in
``include/fusiongpu.h``), as are :func:`orthogonalize`, from which :class:`Muon`
makes the matrices' updates, and :func:`quantize_rows` and :func:`linear_int8`,
with which :meth:`QueryAdapter.quantized` serves in 8 bits.
Tensors are CUDA tensors of float32, float16 or bfloat16; the documents may be
uint8.  Rows may be strided; a tensor whose last dimension is not contiguous
is copied.  Every call takes ``stream=`` (default: the current stream of its
first tensor's device), runs and allocates its results and workspace there, and
does not synchronise: as with any work on another stream, its tensors are ready
there before the call and stay until it is done.  Results are no part of an
autograd graph, whether or not a tensor requires gradients; the backward
functions are called by hand.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
import inspect
import math

import torch

from . import _lib
from .graph import METRICS

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
BASE_DTYPES = {**DTYPES, torch.uint8: 3}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _matrix(t: torch.Tensor, name: str, like: torch.Tensor | None = None, rows: int = -1, cols: int = -1):
    """(a CUDA matrix with unit column stride, its row stride), checked against
    `like`'s type and device and the shape where given."""
    if not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if like is None:
        if t.dtype not in DTYPES:
            raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    elif t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, not {t.dtype} on {t.device}")
    n, d = t.shape
    if (rows >= 0 and n != rows) or (cols >= 0 and d != cols):
        raise ValueError(f"{name} has shape {(n, d)}, not {(rows if rows >= 0 else n, cols if cols >= 0 else d)}")
    s0, s1 = t.stride()
    if (s1 != 1 and d > 1) or (s0 < d and n > 1):
        t = t.contiguous()
        s0 = d
    return t, s0 if n > 1 else 0


def _vector(t: torch.Tensor | None, name: str, n: int, dtype, device) -> int | None:
    if t is None:
        return None
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, not {t.dtype} on {t.device}")
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n}")
    return t.data_ptr()


def _rows(like: torch.Tensor, n: int, d: int) -> torch.Tensor:
    return torch.empty_strided((n, d), (d, 1), dtype=like.dtype, device=like.device)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


@contextlib.contextmanager
def _entered(device, stream):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _on(fn):
    """Runs the function with its `stream` argument and its first tensor's device
    current, so that results and workspace are allocated for that stream; they
    already are in the usual call."""
    first = next(iter(inspect.signature(fn).parameters))

    @functools.wraps(fn)
    def call(*args, stream: torch.cuda.Stream | None = None, **kw):
        x = args[0] if args else kw.get(first)
        if x is None:
            raise TypeError(f"{fn.__name__}() needs {first}")
        if stream is None and x.is_cuda and x.device.index == torch.cuda.current_device():
            return fn(*args, **kw)
        if not x.is_cuda:
            raise ValueError("CUDA tensors are needed")
        with _entered(x.device, stream if stream is not None else torch.cuda.current_stream(x.device)):
            return fn(*args, **kw)
    return call


# the current stream's handle; torch.cuda.current_stream() builds an object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(x: torch.Tensor) -> int:
    if _raw_stream is not None:
        return _raw_stream(x.device.index)
    return torch.cuda.current_stream(x.device).cuda_stream


@functools.lru_cache(maxsize=1024)
def _norm_ws(n: int, d: int, device: int) -> int:
    return _lib.size_query("fg_layer_norm_backward_workspace_size", n, d)


@functools.lru_cache(maxsize=1024)
def _linear_ws(query: str, n: int, i: int, o: int, dtype: int, act: int, ldx: int, ldw: int, ldy: int, off: int,
               device: int) -> int:
    return _lib.size_query(query, C.byref(_lib.LinearParams(n, i, o, dtype, act, ldx, ldw, 0, 0, ldy, off)))


@functools.lru_cache(maxsize=1024)
def _orthogonalize_ws(batch: int, m: int, n: int, dtype: int, steps: int, device: int) -> int:
    return _lib.size_query("fg_orthogonalize_workspace_size",
                           C.byref(_lib.OrthogonalizeParams(batch, m, n, dtype, steps, 0, 0, 0, 0, 0, 0)))


@functools.lru_cache(maxsize=1024)
def _orthogonalize_check(m: int, n: int, dtype: int, steps: int, a: float, b: float, c: float, eps: float) -> None:
    _lib.size_query("fg_orthogonalize_workspace_size", C.byref(_lib.OrthogonalizeParams(1, m, n, dtype, steps, a, b, c, eps, 0, 0)))


def _off16(*pointers: int) -> int:
    """fg_linear_operand bits of the pointers (x, w, dy) that are off 16 bytes."""
    off = 0
    for k, p in enumerate(pointers):
        if p & 15:
            off |= 1 << k
    return off


@_on
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, return_stats: bool = False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension
    of x [rows][dim]; weight and bias of x's type or both float32.  With
    return_stats also the rows' mean and 1 / sqrt(variance + eps), which
    :func:`layer_norm_backward` takes."""
    x, ld = _matrix(x, "x")
    n, d = x.shape
    t, dev = x.dtype, x.device
    p = weight if weight is not None else bias
    pd = torch.float32 if p is not None and p.dtype == torch.float32 else t
    w, b = _vector(weight, "weight", d, pd, dev), _vector(bias, "bias", d, pd, dev)
    y = _rows(x, n, d)
    mean = rstd = None
    if return_stats:
        mean, rstd = torch.empty(n, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().fg_layer_norm(x.data_ptr(), DTYPES[t], n, d, ld, w, b, DTYPES[pd], eps, y.data_ptr(), 0,
                                        _ptr(mean), _ptr(rstd), _stream(x)), "fg_layer_norm")
    return (y, mean, rstd) if return_stats else y


@_on
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None, param_grads: bool = True):
    """Gradients (dx, dweight, dbias) of :func:`layer_norm`; the parameters'
    are of weight's type (x's without one), None when param_grads is false."""
    x, ld = _matrix(x, "x")
    n, d = x.shape
    t, dev = x.dtype, x.device
    dy, lddy = _matrix(dy, "dy", x, n, d)
    if mean is None or rstd is None:
        raise ValueError("mean and rstd of the forward pass are needed")
    m, r = _vector(mean, "mean", n, torch.float32, dev), _vector(rstd, "rstd", n, torch.float32, dev)
    pd = torch.float32 if weight is not None and weight.dtype == torch.float32 else t
    w = _vector(weight, "weight", d, pd, dev)
    dx = _rows(x, n, d)
    dw = db = ws = None
    nws = 0
    if param_grads:
        dw, db = torch.empty(d, dtype=pd, device=dev), torch.empty(d, dtype=pd, device=dev)
        nws = _norm_ws(n, d, dev.index)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
    _lib.check(_lib.lib().fg_layer_norm_backward(dy.data_ptr(), lddy, x.data_ptr(), DTYPES[t], n, d, ld, w, DTYPES[pd],
                                                 m, r, dx.data_ptr(), 0, _ptr(dw), _ptr(db), _ptr(ws), nws,
                                                 _stream(x)), "fg_layer_norm_backward")
    return dx, dw, db


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {name!r}")
    return ACTIVATIONS[name]


@_on
def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
           residual: torch.Tensor | None = None, return_pre: bool = False):
    """activation(x w^T + bias) + residual for x [rows][in], w [out][in]; with
    return_pre also x w^T + bias, which :func:`linear_backward` takes.
    activation: "none", "relu", "gelu" (erf) or "silu"."""
    act = _activation(activation)
    x, ldx = _matrix(x, "x")
    n, i = x.shape
    w, ldw = _matrix(w, "w", x, -1, i)
    o = w.shape[0]
    t, dev = DTYPES[x.dtype], x.device
    b = _vector(bias, "bias", o, x.dtype, dev)
    ldr = 0
    if residual is not None:
        residual, ldr = _matrix(residual, "residual", x, n, o)
    y = _rows(x, n, o)
    pre = _rows(x, n, o) if return_pre else None
    px, pw = x.data_ptr(), w.data_ptr()
    off = _off16(px, pw)
    p = _lib.LinearParams(n, i, o, t, act, ldx, ldw, ldr, 0, 0, off)
    nws = _linear_ws("fg_linear_workspace_size", n, i, o, t, act, ldx, ldw, 0, off, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.check(_lib.lib().fg_linear(C.byref(p), px, pw, b, _ptr(residual), _ptr(pre),
                                    y.data_ptr(), _ptr(ws), nws, _stream(x)), "fg_linear")
    return (y, pre) if return_pre else y


@_on
def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, pre: torch.Tensor | None = None,
                    activation: str = "none", input_grad: bool = True, param_grads: bool = True):
    """Gradients (dx, dw, dbias) of :func:`linear`, of x's type; `pre` from the
    forward pass unless the activation is "none".  The residual's gradient is
    dy.  What input_grad and param_grads leave out is None."""
    act = _activation(activation)
    x, ldx = _matrix(x, "x")
    n, i = x.shape
    w, ldw = _matrix(w, "w", x, -1, i)
    o = w.shape[0]
    t, dev = DTYPES[x.dtype], x.device
    dy, lddy = _matrix(dy, "dy", x, n, o)
    ldp = 0
    if not act:
        pre = None
    elif pre is None:
        raise ValueError("the activation's gradient needs pre")
    else:
        pre, ldp = _matrix(pre, "pre", x, n, o)
    dx = _rows(x, n, i) if input_grad else None
    dw, db = (_rows(x, o, i), torch.empty(o, dtype=x.dtype, device=dev)) if param_grads else (None, None)
    px, pw, pdy = x.data_ptr(), w.data_ptr(), dy.data_ptr()
    off = _off16(px, pw, pdy)
    p = _lib.LinearParams(n, i, o, t, act, ldx, ldw, 0, ldp, lddy, off)
    nws = _linear_ws("fg_linear_backward_workspace_size", n, i, o, t, act, ldx, ldw, lddy, off, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.check(_lib.lib().fg_linear_backward(C.byref(p), pdy, px, pw, _ptr(pre),
                                             _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nws, _stream(x)),
               "fg_linear_backward")
    return dx, dw, db


@_on
def gated_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "silu",
                 return_pre: bool = False):
    """activation(z) * p for [z p] = x w^T + bias, x [rows][in], w [2 out][in] (the
    gates' rows, then their partners'), bias [2 out]; with return_pre also [z p]
    [rows][2 out], which :func:`gated_linear_backward` takes."""
    act = _activation(activation)
    x, ldx = _matrix(x, "x")
    n, i = x.shape
    w, ldw = _matrix(w, "w", x, -1, i)
    if w.shape[0] % 2:
        raise ValueError(f"w must have an even number of rows, not {w.shape[0]}")
    o = w.shape[0] // 2
    t, dev = DTYPES[x.dtype], x.device
    b = _vector(bias, "bias", 2 * o, x.dtype, dev)
    y = _rows(x, n, o)
    pre = _rows(x, n, 2 * o) if return_pre else None
    px, pw = x.data_ptr(), w.data_ptr()
    off = _off16(px, pw)
    p = _lib.LinearParams(n, i, o, t, act, ldx, ldw, 0, 0, 0, off)
    nws = _linear_ws("fg_gated_linear_workspace_size", n, i, o, t, act, ldx, ldw, 0, off, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.check(_lib.lib().fg_gated_linear(C.byref(p), px, pw, b, _ptr(pre), y.data_ptr(), _ptr(ws), nws, _stream(x)),
               "fg_gated_linear")
    return (y, pre) if return_pre else y


@_on
def gated_linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, pre: torch.Tensor,
                          activation: str = "silu", input_grad: bool = True, param_grads: bool = True):
    """Gradients (dx, dw, dbias) of :func:`gated_linear`, of x's type; `pre` from the
    forward pass.  What input_grad and param_grads leave out is None."""
    act = _activation(activation)
    x, ldx = _matrix(x, "x")
    n, i = x.shape
    w, ldw = _matrix(w, "w", x, -1, i)
    if w.shape[0] % 2:
        raise ValueError(f"w must have an even number of rows, not {w.shape[0]}")
    o = w.shape[0] // 2
    t, dev = DTYPES[x.dtype], x.device
    dy, lddy = _matrix(dy, "dy", x, n, o)
    if pre is None:
        raise ValueError("pre of the forward pass is needed")
    pre, ldp = _matrix(pre, "pre", x, n, 2 * o)
    dx = _rows(x, n, i) if input_grad else None
    dw, db = (_rows(x, 2 * o, i), torch.empty(2 * o, dtype=x.dtype, device=dev)) if param_grads else (None, None)
    px, pw = x.data_ptr(), w.data_ptr()
    off = _off16(px, pw)
    p = _lib.LinearParams(n, i, o, t, act, ldx, ldw, 0, ldp, lddy, off)
    nws = _linear_ws("fg_gated_linear_backward_workspace_size", n, i, o, t, act, ldx, ldw, lddy, off, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.check(_lib.lib().fg_gated_linear_backward(C.byref(p), dy.data_ptr(), px, pw, pre.data_ptr(), _ptr(dx), _ptr(dw),
                                                   _ptr(db), _ptr(ws), nws, _stream(x)), "fg_gated_linear_backward")
    return dx, dw, db


def _codes(t: torch.Tensor, name: str, device=None, cols: int = -1):
    """The same as _matrix for codes of 8 bits."""
    if not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if t.dtype != torch.int8 or (device is not None and t.device != device):
        raise TypeError(f"{name} must be int8{'' if device is None else f' on {device}'}, not {t.dtype} on {t.device}")
    n, d = t.shape
    if cols >= 0 and d != cols:
        raise ValueError(f"{name} has {d} columns, not {cols}")
    s0, s1 = t.stride()
    if (s1 != 1 and d > 1) or (s0 < d and n > 1):
        t = t.contiguous()
        s0 = d
    return t, s0 if n > 1 else 0


@_on
def quantize_rows(x: torch.Tensor):
    """Codes of 8 bits and their scales for x's rows: scale = max |x| / 127 and
    q = 127 x / max |x|, rounded to nearest, ties to even.  Returns (q int8
    [rows][dim], its rows on 16-byte boundaries, so strided where dim is no multiple
    of 16; scale float32 [rows]).  A row that holds an infinity or a NaN has scale
    NaN."""
    x, ld = _matrix(x, "x")
    n, d = x.shape
    dev = x.device
    ldq = (d + 15) // 16 * 16
    q = torch.empty_strided((n, d), (ldq, 1), dtype=torch.int8, device=dev)
    scale = torch.empty(n, dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().fg_quantize_rows(x.data_ptr(), DTYPES[x.dtype], n, d, ld, q.data_ptr(), ldq, scale.data_ptr(),
                                           _stream(x)), "fg_quantize_rows")
    return q, scale


@_on
def linear_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                bias: torch.Tensor | None = None, activation: str = "none", residual: torch.Tensor | None = None,
                dtype: torch.dtype = torch.float32):
    """activation(x_scale w_scale (x w^T) + bias) + residual for codes x [rows][in]
    and w [out][in] with a float32 scale per row, as :func:`quantize_rows` gives
    them; the sums are exact.  bias, residual and the result are of `dtype`."""
    act = _activation(activation)
    if dtype not in DTYPES:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    x, ldx = _codes(x, "x")
    n, i = x.shape
    dev = x.device
    w, ldw = _codes(w, "w", dev, i)
    o = w.shape[0]
    if x_scale is None or w_scale is None:
        raise ValueError("x_scale and w_scale are needed")
    xs, wsc = _vector(x_scale, "x_scale", n, torch.float32, dev), _vector(w_scale, "w_scale", o, torch.float32, dev)
    b = _vector(bias, "bias", o, dtype, dev)
    y = torch.empty_strided((n, o), (o, 1), dtype=dtype, device=dev)
    ldr = 0
    if residual is not None:
        residual, ldr = _matrix(residual, "residual", y, n, o)
    px, pw = x.data_ptr(), w.data_ptr()
    off = _off16(px, pw)
    p = _lib.LinearParams(n, i, o, DTYPES[dtype], act, ldx, ldw, ldr, 0, 0, off)
    nws = _linear_ws("fg_linear_int8_workspace_size", n, i, o, DTYPES[dtype], act, ldx, ldw, 0, off, dev.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _lib.check(_lib.lib().fg_linear_int8(C.byref(p), px, xs, pw, wsc, b, _ptr(residual), y.data_ptr(), _ptr(ws), nws,
                                         _stream(x)), "fg_linear_int8")
    return y


@_on
def orthogonalize(g: torch.Tensor, steps: int = 5, coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7):
    """The orthogonalised update of g [rows][cols], or of each matrix of g
    [batch][rows][cols]: X = g / (|g|_F + eps), then `steps` times A = X X^T,
    X = a X + (b A + c A^2) X.  Of g's type, contiguous."""
    if not g.is_cuda or g.dim() not in (2, 3):
        raise ValueError("g must be a 2-D or 3-D CUDA tensor")
    if g.dtype not in DTYPES:
        raise TypeError(f"g must be float32, float16 or bfloat16, not {g.dtype}")
    batch = g.shape[0] if g.dim() == 3 else 1
    m, n = g.shape[-2:]
    if not m or not n:
        raise ValueError(f"g has shape {tuple(g.shape)}")
    s1, s2 = g.stride(-2), g.stride(-1)
    if (s2 != 1 and n > 1) or (s1 < n and m > 1) or (batch > 1 and g.stride(0) <= 0):
        g = g.contiguous()
        s1 = n
    ld = s1 if m > 1 else n
    out = torch.empty_strided(g.shape, (n, 1) if g.dim() == 2 else (m * n, n, 1), dtype=g.dtype, device=g.device)
    a, b, c = coefficients
    p = _lib.OrthogonalizeParams(batch, m, n, DTYPES[g.dtype], steps, a, b, c, eps, ld, g.stride(0) if batch > 1 else 0)
    nws = _orthogonalize_ws(batch, m, n, DTYPES[g.dtype], steps, g.device.index)
    ws = torch.empty(nws, dtype=torch.uint8, device=g.device) if nws else None
    _lib.check(_lib.lib().fg_orthogonalize(C.byref(p), g.data_ptr(), out.data_ptr(), _ptr(ws), nws, _stream(g)),
               "fg_orthogonalize")
    return out


@_on
def preference_loss(queries: torch.Tensor, base: torch.Tensor, offsets: torch.Tensor, pos_ids: torch.Tensor,
                    neg_ids: torch.Tensor, ref: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                    beta: float = 1.0, label_smoothing: float = 0.0, metric: str = "ip", grad: bool = True):
    """Paired preference loss of queries [nq][dim] over the documents base
    [nbase][dim] (float32, float16, bfloat16 or uint8): query i prefers document
    pos_ids[p] to neg_ids[p] for its pairs p in [offsets[i], offsets[i+1])
    (offsets int64 [nq+1], ascending, ids int32; a pair with an id outside the
    base, or that no query holds, is masked: loss and margin 0).  `ref`: the reference queries the log ratios are taken against
    (the unadapted ones).  Returns (losses [pairs], margins [pairs], dq), dq the
    gradient of sum(weights * losses), or None when grad is false."""
    q, ldq = _matrix(queries, "queries")
    nq, d = q.shape
    dev = q.device
    ldr = 0
    if ref is not None:
        ref, ldr = _matrix(ref, "ref", q, nq, d)
    if metric not in METRICS:
        raise ValueError(f"metric must be one of {sorted(METRICS)}, not {metric!r}")
    if base.dtype not in BASE_DTYPES or base.device != dev:
        raise TypeError(f"base must be one of {list(BASE_DTYPES)} on {dev}")
    if base.dim() != 2 or base.shape[1] != d or not base.is_contiguous():
        raise ValueError(f"base must be contiguous [nbase][{d}]")
    m = pos_ids.numel()
    po, ne = _vector(pos_ids, "pos_ids", m, torch.int32, dev), _vector(neg_ids, "neg_ids", m, torch.int32, dev)
    off = _vector(offsets, "offsets", nq + 1, torch.int64, dev)
    wt = _vector(weights, "weights", m, torch.float32, dev)
    losses, margins = torch.empty(m, dtype=torch.float32, device=dev), torch.empty(m, dtype=torch.float32, device=dev)
    dq = _rows(q, nq, d) if grad else None
    p = _lib.PreferenceParams(nq, d, DTYPES[q.dtype], BASE_DTYPES[base.dtype], base.shape[0], m, METRICS[metric], beta,
                              label_smoothing, ldq, ldr, 0)
    _lib.check(_lib.lib().fg_preference_loss(C.byref(p), q.data_ptr(), _ptr(ref), base.data_ptr(), off, po, ne, wt,
                                             losses.data_ptr(), margins.data_ptr(), _ptr(dq), _stream(q)),
               "fg_preference_loss")
    return losses, margins, dq


class QueryAdapter:
    """adapted = q + w2 act(w1 layer_norm(q) + b1) + b2, trained on preferences; with
    gated=True the inner layer is :func:`gated_linear`, w1 [2 hidden][dim] and b1
    [2 hidden] holding the gates' rows, then their partners'.

    `params` holds the tensors (norm_weight, norm_bias in float32, the others in
    `dtype`); w2 and b2 start at zero, so an untrained adapter returns its
    queries.  :meth:`train_step` leaves the gradients in the tensors' ``grad``,
    where a ``torch.optim`` optimizer over ``parameters()`` finds them."""

    def __init__(self, dim: int, hidden: int, activation: str = "gelu", dtype: torch.dtype = torch.float32,
                 seed: int = 0, device="cuda", gated: bool = False):
        if dtype not in DTYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
        _activation(activation)
        self.dim, self.hidden, self.activation, self.dtype, self.gated = dim, hidden, activation, dtype, gated
        g = torch.Generator().manual_seed(seed)
        inner = 2 * hidden if gated else hidden
        w1 = torch.randn(inner, dim, generator=g) / math.sqrt(dim)
        self.params = {
            "norm_weight": torch.ones(dim, device=device),
            "norm_bias": torch.zeros(dim, device=device),
            "w1": w1.to(device=device, dtype=dtype),
            "b1": torch.zeros(inner, device=device, dtype=dtype),
            "w2": torch.zeros(dim, hidden, device=device, dtype=dtype),
            "b2": torch.zeros(dim, device=device, dtype=dtype),
        }

    def parameters(self) -> list[torch.Tensor]:
        return list(self.params.values())

    def matrices(self) -> list[torch.Tensor]:
        """The parameters that :class:`Muon` takes."""
        return [p for p in self.params.values() if p.dim() == 2]

    def vectors(self) -> list[torch.Tensor]:
        """The others."""
        return [p for p in self.params.values() if p.dim() != 2]

    def __call__(self, queries: torch.Tensor, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """The adapted queries [nq][dim], of the adapter's type: what the index
        is searched with."""
        p = self.params
        with contextlib.nullcontext() if stream is None else _entered(queries.device, stream):
            q = queries.to(self.dtype)
            n = layer_norm(q, p["norm_weight"], p["norm_bias"])
            h = (gated_linear if self.gated else linear)(n, p["w1"], p["b1"], activation=self.activation)
            return linear(h, p["w2"], p["b2"], residual=q)

    def quantized(self) -> "QuantizedQueryAdapter":
        """What this adapter has learned, as it is now, for serving in 8 bits."""
        return QuantizedQueryAdapter(self)

    def train_step(self, queries: torch.Tensor, base: torch.Tensor, offsets: torch.Tensor, pos_ids: torch.Tensor,
                   neg_ids: torch.Tensor, beta: float = 1.0, label_smoothing: float = 0.0, metric: str = "l2",
                   weights: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
        """One forward and backward pass on the pairs of `queries`, against the
        unadapted queries as the reference.  Returns (losses, margins) and
        leaves the gradient of sum(weights * losses) in the parameters'
        ``grad``."""
        p = self.params
        inner, inner_backward = (gated_linear, gated_linear_backward) if self.gated else (linear, linear_backward)
        with contextlib.nullcontext() if stream is None else _entered(queries.device, stream):
            q = queries.to(self.dtype)
            n, mean, rstd = layer_norm(q, p["norm_weight"], p["norm_bias"], return_stats=True)
            h, z = inner(n, p["w1"], p["b1"], activation=self.activation, return_pre=True)
            out = linear(h, p["w2"], p["b2"], residual=q)
            losses, margins, dout = preference_loss(out, base, offsets, pos_ids, neg_ids, ref=q, weights=weights,
                                                    beta=beta, label_smoothing=label_smoothing, metric=metric)
            dh, p["w2"].grad, p["b2"].grad = linear_backward(dout, h, p["w2"])
            dn, p["w1"].grad, p["b1"].grad = inner_backward(dh, n, p["w1"], pre=z, activation=self.activation)
            _, p["norm_weight"].grad, p["norm_bias"].grad = layer_norm_backward(dn, q, mean, rstd, p["norm_weight"])
        return losses, margins


class QuantizedQueryAdapter:
    """A trained :class:`QueryAdapter` whose matrices are codes of 8 bits with a scale
    per row; the rows that meet them are quantised on the way.  Layer norm, biases,
    activations and the residual stay as they are.  Keeps copies: the adapter may be
    trained on.

    Its matrices take a quarter of float32's bytes.  float32 adapters are faster so from
    about a hundred queries on (768 wide, 10,000 queries: 153 us on the device, 343),
    those of 16 bits only where they are plain and the queries very many (1,000,000:
    4.3 ms, 4.7): the codes of the rows are passes of their own."""

    def __init__(self, adapter: QueryAdapter):
        p = adapter.params
        self.dim, self.hidden, self.activation, self.dtype = adapter.dim, adapter.hidden, adapter.activation, adapter.dtype
        self.gated = adapter.gated
        self.params = {k: p[k].detach().clone() for k in ("norm_weight", "norm_bias", "b1", "b2")}
        for k in ("w1", "w2"):
            self.params[k], self.params[k + "_scale"] = quantize_rows(p[k].detach())

    def _inner(self, x: torch.Tensor, x_scale: torch.Tensor, rows: slice, activation: str) -> torch.Tensor:
        p = self.params
        return linear_int8(x, x_scale, p["w1"][rows], p["w1_scale"][rows], p["b1"][rows], activation=activation,
                           dtype=self.dtype)

    def __call__(self, queries: torch.Tensor, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """The adapted queries [nq][dim], of the adapter's type."""
        p, hid = self.params, self.hidden
        with contextlib.nullcontext() if stream is None else _entered(queries.device, stream):
            q = queries.to(self.dtype)
            x, x_scale = quantize_rows(layer_norm(q, p["norm_weight"], p["norm_bias"]))
            h = self._inner(x, x_scale, slice(0, hid), self.activation)
            # both factors and their product are of the adapter's type: the update is off by 2.67 % in
            # bfloat16, with 32 bits there 2.66 %, since the codes make the error (768 -> 1024)
            if self.gated:
                h *= self._inner(x, x_scale, slice(hid, 2 * hid), "none")
            h, h_scale = quantize_rows(h)
            return linear_int8(h, h_scale, p["w2"], p["w2_scale"], p["b2"], residual=q, dtype=self.dtype)


class Muon(torch.optim.Optimizer):
    """Momentum whose update of a matrix is orthogonalised (:func:`orthogonalize`):

        m = momentum m + grad,   u = grad + momentum m (nesterov) or m
        p = (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    for matrices on the GPU; vectors go to another optimizer.  Matrices of one shape
    and type are orthogonalised together.  (K. Jordan and others, "Muon: An optimizer
    for hidden layers in neural networks", 2024.)

    m is of the parameter's type, as torch's optimizers keep their states: rounded twice
    a step, it is off by 0.7 % of its norm in bfloat16 and 0.1 % in float16 (momentum
    0.95).  Parameters of float32 keep all of it in 32 bits.

    A decay smaller than the type resolves (lr weight_decay below 2^-7 in bfloat16,
    2^-10 in float16) would be rounded away step by step, so it is held back, in the
    state's "decay", until four times as much is due; such a step cannot be captured
    into a CUDA graph."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> None:
        """Refuses what a step could not finish."""
        if not group["lr"] >= 0 or not 0 <= group["momentum"] < 1 or not group["weight_decay"] >= 0:
            raise ValueError("lr and weight_decay must not be negative, momentum must be in [0, 1)")
        for p in group["params"]:
            if p.dim() != 2 or p.dtype not in DTYPES:
                raise ValueError(f"Muon takes matrices of float32, float16 or bfloat16, not {tuple(p.shape)} {p.dtype}")
            _orthogonalize_check(*p.shape, DTYPES[p.dtype], group["steps"], *group["coefficients"], group["eps"])

    def _check_step(self) -> None:
        """The same of the whole step, before anything moves."""
        for group in self.param_groups:
            self._check(group)
            d = group["lr"] * group["weight_decay"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda or p.grad.layout != torch.strided:
                    raise ValueError(f"Muon takes matrices on the GPU with dense gradients, not on {p.device} with {p.grad.layout}")
                if 0 < d < torch.finfo(p.dtype).eps and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(f"a decay of {d:g} a step, which {p.dtype} does not resolve, cannot be captured into a CUDA graph")

    def _decay(self, p: torch.Tensor, d: float) -> None:
        """p = (1 - d) p, or held back.  A factor of 1 - d is off by half a step, eps / 2 of
        p, when it is rounded: half of what is due where d is eps, an eighth of 4 eps."""
        eps, state = torch.finfo(p.dtype).eps, self.state[p]
        keep = state.pop("decay", 1.0) * (1 - d)
        if d >= eps or 1 - keep >= 4 * eps:
            p.mul_(keep)
        else:
            state["decay"] = keep

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_step()
        for group in self.param_groups:
            alike: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                m = state["momentum"].mul_(group["momentum"]).add_(p.grad)
                u = p.grad.add(m, alpha=group["momentum"]) if group["nesterov"] else m
                alike.setdefault((p.shape, p.dtype, p.device), []).append((p, u))
            for (shape, _, _), pairs in alike.items():
                u = pairs[0][1] if len(pairs) == 1 else torch.stack([u for _, u in pairs])
                o = orthogonalize(u, steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
                scale = math.sqrt(max(1.0, shape[0] / shape[1]))
                for (p, _), x in zip(pairs, [o] if len(pairs) == 1 else o):
                    if group["weight_decay"]:
                        self._decay(p, group["lr"] * group["weight_decay"])
                    p.add_(x, alpha=-group["lr"] * scale)
        return loss
