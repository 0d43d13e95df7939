"""Query adapter: a small model between an embedding model and the search, and
its training on preferences over the index's documents.

The reference searches the queries as they are given (search_pipeline.cu:594);
this is what a user of an index puts before that call to fit it to other
queries without re-embedding and re-building it.  :class:`QueryAdapter` is the
residual block

    adapted = q + w2 act(w1 layer_norm(q) + b1) + b2

whose operators (:func:`layer_norm`, :func:`linear`, :func:`preference_loss`
and the gradients) are the package's own sm_100a kernels behind the C ABI
(fg_layer_norm, fg_linear, fg_preference_loss in ``include/fusiongpu.h``).
Tensors are CUDA tensors of float32, float16 or bfloat16; the documents may be
uint8.  Rows may be strided; a tensor whose last dimension is not contiguous
is copied.  Every call runs on ``stream`` (default: the current stream), does
not synchronise, and allocates its results and workspace there.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import torch

from . import _lib
from .graph import METRICS

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
BASE_DTYPES = {**DTYPES, torch.uint8: 3}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _matrix(t: torch.Tensor, name: str, like: torch.Tensor | None = None, shape=None) -> torch.Tensor:
    """A CUDA matrix with unit column stride, checked against `like`'s type and device."""
    if not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if like is None:
        if t.dtype not in DTYPES:
            raise TypeError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    elif t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, not {t.dtype} on {t.device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    rows, cols = t.shape
    s0, s1 = t.stride()
    if (s1 != 1 and cols > 1) or (s0 < cols and rows > 1):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else 0


def _vector(t: torch.Tensor | None, name: str, n: int, dtypes, device) -> int | None:
    if t is None:
        return None
    if t.dtype not in dtypes or t.device != device:
        raise TypeError(f"{name} must be one of {dtypes} on {device}, not {t.dtype} on {t.device}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n}")
    return t.data_ptr()


@contextlib.contextmanager
def _entered(device, stream):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield stream.cuda_stream


def _on(t: torch.Tensor, stream):
    """The stream to launch on, current while results are allocated."""
    if stream is None and t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext(torch.cuda.current_stream().cuda_stream)
    return _entered(t.device, stream if stream is not None else torch.cuda.current_stream(t.device))


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, return_stats: bool = False, stream: torch.cuda.Stream | None = None):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension
    of x [rows][dim]; weight and bias of x's type or both float32.  With
    return_stats also the rows' mean and 1 / sqrt(variance + eps), which
    :func:`layer_norm_backward` takes."""
    x = _matrix(x, "x")
    n, d = x.shape
    p = weight if weight is not None else bias
    pd = x.dtype if p is None else p.dtype
    allowed = (pd,) if pd in (x.dtype, torch.float32) else (x.dtype, torch.float32)
    w, b = _vector(weight, "weight", d, allowed, x.device), _vector(bias, "bias", d, allowed, x.device)
    with _on(x, stream) as s:
        y = torch.empty((n, d), dtype=x.dtype, device=x.device)
        mean = rstd = None
        if return_stats:
            mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x.device).unbind(0)
        _lib.call("fg_layer_norm", x.data_ptr(), DTYPES[x.dtype], n, d, _ld(x), w, b, DTYPES[pd], eps, y.data_ptr(),
                  0, None if mean is None else mean.data_ptr(), None if rstd is None else rstd.data_ptr(), s)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None, param_grads: bool = True,
                        stream: torch.cuda.Stream | None = None):
    """Gradients (dx, dweight, dbias) of :func:`layer_norm`; the parameters'
    are of weight's type (x's without one), None when param_grads is false."""
    x = _matrix(x, "x")
    dy = _matrix(dy, "dy", x, x.shape)
    n, d = x.shape
    m, r = (_vector(t, k, n, (torch.float32,), x.device) for t, k in ((mean, "mean"), (rstd, "rstd")))
    if m is None or r is None:
        raise ValueError("mean and rstd of the forward pass are needed")
    w = _vector(weight, "weight", d, (x.dtype, torch.float32), x.device)
    pd = x.dtype if weight is None else weight.dtype
    with _on(x, stream) as s:
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device)
        dw = db = ws = None
        if param_grads:
            dw = torch.empty(d, dtype=pd, device=x.device)
            db = torch.empty(d, dtype=pd, device=x.device)
            ws = torch.empty(_lib.size_query("fg_layer_norm_backward_workspace_size", n, d), dtype=torch.uint8,
                             device=x.device)
        _lib.call("fg_layer_norm_backward", dy.data_ptr(), _ld(dy), x.data_ptr(), DTYPES[x.dtype], n, d, _ld(x), w,
                  DTYPES[pd], m, r, dx.data_ptr(), 0, None if dw is None else dw.data_ptr(),
                  None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(),
                  0 if ws is None else ws.numel(), s)
    return dx, dw, db


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {name!r}")
    return ACTIVATIONS[name]


def _workspace(query: str, p, device) -> torch.Tensor | None:
    n = _lib.size_query(query, C.byref(p))
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
           residual: torch.Tensor | None = None, return_pre: bool = False,
           stream: torch.cuda.Stream | None = None):
    """activation(x w^T + bias) + residual for x [rows][in], w [out][in]; with
    return_pre also x w^T + bias, which :func:`linear_backward` takes.
    activation: "none", "relu", "gelu" (erf) or "silu"."""
    act = _activation(activation)
    x = _matrix(x, "x")
    n, i = x.shape
    w = _matrix(w, "w", x)
    o = w.shape[0]
    if w.shape[1] != i:
        raise ValueError(f"w has {w.shape[1]} columns, x {i}")
    b = _vector(bias, "bias", o, (x.dtype,), x.device)
    if residual is not None:
        residual = _matrix(residual, "residual", x, (n, o))
    with _on(x, stream) as s:
        y = torch.empty((n, o), dtype=x.dtype, device=x.device)
        pre = torch.empty((n, o), dtype=x.dtype, device=x.device) if return_pre else None
        p = _lib.LinearParams(n, i, o, DTYPES[x.dtype], act, _ld(x), _ld(w),
                              0 if residual is None else _ld(residual), 0, 0)
        ws = _workspace("fg_linear_workspace_size", p, x.device)
        _lib.call("fg_linear", C.byref(p), x.data_ptr(), w.data_ptr(), b,
                  None if residual is None else residual.data_ptr(), None if pre is None else pre.data_ptr(),
                  y.data_ptr(), None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), s)
    return (y, pre) if return_pre else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, pre: torch.Tensor | None = None,
                    activation: str = "none", input_grad: bool = True, param_grads: bool = True,
                    stream: torch.cuda.Stream | None = None):
    """Gradients (dx, dw, dbias) of :func:`linear`, of x's type; `pre` from the
    forward pass unless the activation is "none".  The residual's gradient is
    dy.  What input_grad and param_grads leave out is None."""
    act = _activation(activation)
    x = _matrix(x, "x")
    n, i = x.shape
    w = _matrix(w, "w", x)
    o = w.shape[0]
    if w.shape[1] != i:
        raise ValueError(f"w has {w.shape[1]} columns, x {i}")
    dy = _matrix(dy, "dy", x, (n, o))
    if act:
        if pre is None:
            raise ValueError("the activation's gradient needs pre")
        pre = _matrix(pre, "pre", x, (n, o))
    else:
        pre = None
    with _on(x, stream) as s:
        dx = torch.empty((n, i), dtype=x.dtype, device=x.device) if input_grad else None
        dw = torch.empty((o, i), dtype=x.dtype, device=x.device) if param_grads else None
        db = torch.empty(o, dtype=x.dtype, device=x.device) if param_grads else None
        p = _lib.LinearParams(n, i, o, DTYPES[x.dtype], act, _ld(x), _ld(w), 0, 0 if pre is None else _ld(pre),
                              _ld(dy))
        ws = _workspace("fg_linear_backward_workspace_size", p, x.device)
        _lib.call("fg_linear_backward", C.byref(p), dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                  None if pre is None else pre.data_ptr(), None if dx is None else dx.data_ptr(),
                  None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                  None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), s)
    return dx, dw, db


def preference_loss(queries: torch.Tensor, base: torch.Tensor, offsets: torch.Tensor, pos_ids: torch.Tensor,
                    neg_ids: torch.Tensor, ref: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                    beta: float = 1.0, label_smoothing: float = 0.0, metric: str = "ip", grad: bool = True,
                    stream: torch.cuda.Stream | None = None):
    """Paired preference loss of queries [nq][dim] over the documents base
    [nbase][dim] (float32, float16, bfloat16 or uint8): query i prefers document
    pos_ids[p] to neg_ids[p] for its pairs p in [offsets[i], offsets[i+1])
    (offsets int64 [nq+1], ids int32; a pair with an id outside the base is
    masked).  `ref`: the reference queries the log ratios are taken against
    (the unadapted ones).  Returns (losses [pairs], margins [pairs], dq), dq the
    gradient of sum(weights * losses), or None when grad is false."""
    q = _matrix(queries, "queries")
    nq, d = q.shape
    if ref is not None:
        ref = _matrix(ref, "ref", q, q.shape)
    if metric not in METRICS:
        raise ValueError(f"metric must be one of {sorted(METRICS)}, not {metric!r}")
    if base.dtype not in BASE_DTYPES or base.device != q.device:
        raise TypeError(f"base must be one of {list(BASE_DTYPES)} on {q.device}")
    if base.dim() != 2 or base.shape[1] != d or not base.is_contiguous():
        raise ValueError(f"base must be contiguous [nbase][{d}]")
    m = pos_ids.numel()
    po = _vector(pos_ids, "pos_ids", m, (torch.int32,), q.device)
    ne = _vector(neg_ids, "neg_ids", m, (torch.int32,), q.device)
    off = _vector(offsets, "offsets", nq + 1, (torch.int64,), q.device)
    wt = _vector(weights, "weights", m, (torch.float32,), q.device)
    with _on(q, stream) as s:
        losses, margins = torch.empty((2, m), dtype=torch.float32, device=q.device).unbind(0)
        dq = torch.empty((nq, d), dtype=q.dtype, device=q.device) if grad else None
        p = _lib.PreferenceParams(nq, d, DTYPES[q.dtype], BASE_DTYPES[base.dtype], base.shape[0], m, METRICS[metric],
                                  beta, label_smoothing, _ld(q), 0 if ref is None else _ld(ref), 0)
        _lib.call("fg_preference_loss", C.byref(p), q.data_ptr(), None if ref is None else ref.data_ptr(),
                  base.data_ptr(), off, po, ne, wt, losses.data_ptr(), margins.data_ptr(),
                  None if dq is None else dq.data_ptr(), s)
    return losses, margins, dq


class QueryAdapter:
    """adapted = q + w2 act(w1 layer_norm(q) + b1) + b2, trained on preferences.

    `params` holds the tensors (norm_weight, norm_bias in float32, the others in
    `dtype`); w2 and b2 start at zero, so an untrained adapter returns its
    queries.  :meth:`train_step` leaves the gradients in the tensors' ``grad``,
    where a ``torch.optim`` optimizer over ``parameters()`` finds them."""

    def __init__(self, dim: int, hidden: int, activation: str = "gelu", dtype: torch.dtype = torch.float32,
                 seed: int = 0, device="cuda"):
        if dtype not in DTYPES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
        _activation(activation)
        self.dim, self.hidden, self.activation, self.dtype = dim, hidden, activation, dtype
        g = torch.Generator().manual_seed(seed)
        w1 = torch.randn(hidden, dim, generator=g) / math.sqrt(dim)
        self.params = {
            "norm_weight": torch.ones(dim, device=device),
            "norm_bias": torch.zeros(dim, device=device),
            "w1": w1.to(device=device, dtype=dtype),
            "b1": torch.zeros(hidden, device=device, dtype=dtype),
            "w2": torch.zeros(dim, hidden, device=device, dtype=dtype),
            "b2": torch.zeros(dim, device=device, dtype=dtype),
        }

    def parameters(self) -> list[torch.Tensor]:
        return list(self.params.values())

    def __call__(self, queries: torch.Tensor, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """The adapted queries [nq][dim], of the adapter's type: what the index
        is searched with."""
        p = self.params
        q = queries.to(self.dtype)
        n = layer_norm(q, p["norm_weight"], p["norm_bias"], stream=stream)
        h = linear(n, p["w1"], p["b1"], activation=self.activation, stream=stream)
        return linear(h, p["w2"], p["b2"], residual=q, stream=stream)

    def train_step(self, queries: torch.Tensor, base: torch.Tensor, offsets: torch.Tensor, pos_ids: torch.Tensor,
                   neg_ids: torch.Tensor, beta: float = 1.0, label_smoothing: float = 0.0, metric: str = "l2",
                   weights: torch.Tensor | None = None):
        """One forward and backward pass on the pairs of `queries`, against the
        unadapted queries as the reference.  Returns (losses, margins) and
        leaves the gradient of sum(weights * losses) in the parameters'
        ``grad``."""
        p = self.params
        q = queries.to(self.dtype)
        n, mean, rstd = layer_norm(q, p["norm_weight"], p["norm_bias"], return_stats=True)
        h, z = linear(n, p["w1"], p["b1"], activation=self.activation, return_pre=True)
        out = linear(h, p["w2"], p["b2"], residual=q)
        losses, margins, dout = preference_loss(out, base, offsets, pos_ids, neg_ids, ref=q, weights=weights,
                                                beta=beta, label_smoothing=label_smoothing, metric=metric)
        dh, p["w2"].grad, p["b2"].grad = linear_backward(dout, h, p["w2"])
        dn, p["w1"].grad, p["b1"].grad = linear_backward(dh, n, p["w1"], pre=z, activation=self.activation)
        _, p["norm_weight"].grad, p["norm_bias"].grad = layer_norm_backward(dn, q, mean, rstd, p["norm_weight"])
        return losses, margins
