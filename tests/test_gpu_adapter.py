"""GPU tests of the query adapter's operators against plain implementations in
64 bits.

Tolerances follow from the arithmetic, element by element.  U[t] is the unit
roundoff of a result's type (one rounding when it is written), E32 = 2^-24 that
of the 32-bit sums; a sum of n products in 32 bits, in any order and with
truncating additions, is within (n + 8) * 2 * E32 of the sum of the products'
magnitudes.  The kernels' activation functions are held to ACT (an absolute
error per unit of max(|z|, 1)): a few ulp of 32 bits for float32, 2^-18 where
the result is rounded to 16 bits.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
ACT = {"f32": 2.0 ** -20, "f16": 2.0 ** -18, "bf16": 2.0 ** -18}
E32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ad():
    from fusiongpu_b200 import adapter
    return adapter


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, t="f32", scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(T[t])


def _within(got, want, tol, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} x tolerance"


# ---- layer norm ---------------------------------------------------------------------

DIMS = [1, 2, 31, 64, 96, 100, 128, 200, 256, 257, 500, 768, 1001, 1024, 1025, 1536, 2000, 4096, 4100, 5001, 8192, 16384]


def _norm_ref(x, w, b, eps):
    x = x.double()
    m = x.mean(1, keepdim=True)
    r = 1 / (((x - m) ** 2).mean(1, keepdim=True) + eps).sqrt()
    h = (x - m) * r
    y = h
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, m, r, h


def _norm_tol(x, m, r, h, w, eps):
    """Error of h: the mean and the variance are sums of dim terms (taken by at
    least 8 threads, dim / 8 + 16 additions deep), scaled by r."""
    n = x.shape[1]
    depth = (n / 8 + 16) * 2 * E32
    ax = x.double().abs().mean(1, keepdim=True)
    return depth * (ax * r + h.abs()) + 8 * E32 * (1 + h.abs())


@pytest.mark.parametrize("t,p", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("dim", DIMS)
def test_layer_norm(ad, dim, t, p):
    g = _gen(dim)
    for rows in (1, 3, 37, 130):
        x = _randn(g, rows, dim, t=t, scale=0.7, mean=0.4)
        w, b = _randn(g, dim, t=p, mean=1.0, scale=0.3), _randn(g, dim, t=p, scale=0.3)
        y, mean, rstd = ad.layer_norm(x, w, b, return_stats=True)
        ry, m, r, h = _norm_ref(x, w, b, 1e-5)
        th = _norm_tol(x, m, r, h, w, 1e-5)
        assert y.dtype == x.dtype
        _within(y, ry, th * w.double().abs() + 2 * E32 * b.double().abs() + U[t] * ry.abs() + TINY[t] + E32, "y")
        _within(mean, m[:, 0], (dim / 8 + 16) * 2 * E32 * x.double().abs().mean(1) + TINY["f32"], "mean")
        _within(rstd, r[:, 0], ((dim / 8 + 24) * 4 * E32 * (1 + (x.double().abs().mean(1, keepdim=True) * r)[:, 0]))
                * r[:, 0], "rstd")
        assert torch.equal(y, ad.layer_norm(x, w, b))  # serving form, same values


@pytest.mark.parametrize("t,p", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("dim", DIMS)
def test_layer_norm_backward(ad, dim, t, p):
    g = _gen(dim + 1)
    for rows in (1, 5, 300):
        x, dy = _randn(g, rows, dim, t=t, scale=0.7, mean=0.2), _randn(g, rows, dim, t=t, scale=0.3)
        w = _randn(g, dim, t=p, mean=1.0, scale=0.3)
        _, mean, rstd = ad.layer_norm(x, w, None, return_stats=True)
        dx, dw, db = ad.layer_norm_backward(dy, x, mean, rstd, w)
        m, r = mean.double()[:, None], rstd.double()[:, None]
        h = (x.double() - m) * r
        a = dy.double() * w.double()
        ma, mah = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
        want = r * (a - ma - h * mah)
        depth = (dim / 8 + 24) * 2 * E32
        scale = r * (a.abs() + a.abs().mean(1, keepdim=True) + h.abs() * (a * h).abs().mean(1, keepdim=True))
        # h itself: x - m rounds once, by the larger of the two
        he = 4 * E32 * ((x.double().abs() + m.abs()) * r + h.abs())
        extra = r * (he * (a * h).abs().mean(1, keepdim=True) + h.abs() * (a.abs() * he).mean(1, keepdim=True))
        _within(dx, want, depth * scale + 2 * extra + U[t] * want.abs() + TINY[t], "dx")
        deep = (rows + 16) * 2 * E32
        rdw, rdb = (dy.double() * h).sum(0), dy.double().sum(0)
        _within(dw, rdw, deep * (dy.double() * h).abs().sum(0) + (dy.double().abs() * he).sum(0) + U[p] * rdw.abs()
                + TINY[p], "dweight")
        _within(db, rdb, deep * dy.double().abs().sum(0) + U[p] * rdb.abs() + TINY[p], "dbias")
        assert dw.dtype == T[p] and dx.dtype == T[t]
        again = ad.layer_norm_backward(dy, x, mean, rstd, w)
        for u, v in zip((dx, dw, db), again):
            assert torch.equal(u, v)  # no order of additions that changes


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("dim", [96, 768, 1001])
def test_layer_norm_strides_and_absent_parameters(ad, t, dim):
    g = _gen(9)
    big = _randn(g, 65, dim + 37, t=t)
    for x in (big[:, 1:1 + dim], big[::2, 16:16 + dim], big[:, :dim]):
        c = x.contiguous()
        assert torch.equal(ad.layer_norm(x), ad.layer_norm(c))
        w = _randn(g, dim, t=t)
        _, mean, rstd = ad.layer_norm(x, w, return_stats=True)
        dy = big[:c.shape[0], 3:3 + dim]
        for u, v in zip(ad.layer_norm_backward(dy, x, mean, rstd, w),
                        ad.layer_norm_backward(dy.contiguous(), c, mean, rstd, w)):
            _within(u, v.double(), U[t] * 2 * v.double().abs() + 1e-4 * U[t] ** 0.5 + 64 * E32 * v.double().abs().max(), "strided")
        ones = torch.ones(dim, device="cuda", dtype=T[t])
        for u, v in zip(ad.layer_norm_backward(c, c, mean, rstd, None), ad.layer_norm_backward(c, c, mean, rstd, ones)):
            assert torch.equal(u, v)
        assert torch.equal(ad.layer_norm(c, bias=w), ad.layer_norm(c, ones, w))
        assert ad.layer_norm_backward(c, c, mean, rstd, w, param_grads=False)[1:] == (None, None)


@pytest.mark.parametrize("t,p", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,rows", [(40, 40001), (128, 21000), (100, 21000), (301, 6000), (512, 6007), (768, 6001),
                                      (1000, 5003), (1001, 3001), (1536, 3001), (4096, 1501), (5000, 701)])
def test_layer_norm_more_rows_than_groups(ad, dim, rows, t, p):
    """Groups that take several rows in turn: every row comes out as it does alone,
    on 16-byte boundaries and off them, and the weight's gradients hold all rows."""
    g = _gen(rows)
    x, dy = _randn(g, rows, dim, t=t, scale=0.7, mean=0.2), _randn(g, rows, dim, t=t, scale=0.3)
    w, b = _randn(g, dim, t=p, mean=1.0, scale=0.3), _randn(g, dim, t=p, scale=0.3)
    y, mean, rstd = ad.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = ad.layer_norm_backward(dy, x, mean, rstd, w)
    for i in (0, rows // 2 - 11, rows - 23):
        k = slice(i, i + 23)
        y1, m1, r1 = ad.layer_norm(x[k], w, b, return_stats=True)
        assert torch.equal(y1, y[k]) and torch.equal(m1, mean[k]) and torch.equal(r1, rstd[k])
        assert torch.equal(ad.layer_norm_backward(dy[k], x[k], m1, r1, w, param_grads=False)[0], dx[k])
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    he = 4 * E32 * ((x.double().abs() + mean.double().abs()[:, None]) * rstd.double()[:, None] + h.abs())
    deep, d = (rows + 16) * 2 * E32, dy.double()
    rdw, rdb = (d * h).sum(0), d.sum(0)
    _within(dw, rdw, deep * (d * h).abs().sum(0) + (d.abs() * he).sum(0) + U[p] * rdw.abs() + TINY[p], "dweight")
    _within(db, rdb, deep * d.abs().sum(0) + U[p] * rdb.abs() + TINY[p], "dbias")
    xo = torch.empty(rows, dim + 3, device="cuda", dtype=T[t])[:, 1:1 + dim]
    xo.copy_(x)
    assert torch.equal(ad.layer_norm(xo, w, b), y)
    for u, v in zip(ad.layer_norm_backward(dy, xo, mean, rstd, w), (dx, dw, db)):
        assert torch.equal(u, v)


def test_layer_norm_empty_constant_and_nonfinite_rows(ad):
    x = torch.zeros(0, 64, device="cuda")
    y, mean, rstd = ad.layer_norm(x, return_stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = ad.layer_norm_backward(x, x, mean, rstd, torch.ones(64, device="cuda"))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    for dim in (64, 768, 1030, 5000):
        g = _gen(dim)
        x = _randn(g, 9, dim)
        x[2] = 3.5          # no variance: rstd = 1 / sqrt(eps), y = bias
        x[4, 7] = math.nan  # poison stays in its row
        x[6, 1] = math.inf
        b = _randn(g, dim)
        y = ad.layer_norm(x, None, b)
        assert torch.equal(y[2], b)
        assert y[4].isnan().all() and y[6].isnan().all()
        assert y[[0, 1, 2, 3, 5, 7, 8]].isfinite().all()


def test_layer_norm_large_mean(ad):
    """Rows whose spread is a thousandth of their mean: the second pass over the
    centred values keeps the variance."""
    g = _gen(3)
    x = _randn(g, 64, 768, scale=0.01, mean=10.0)
    y, mean, rstd = ad.layer_norm(x, return_stats=True)
    ry, m, r, h = _norm_ref(x, None, None, 1e-5)
    # the mean is off by a few ulp of 10, which is 2^-21 / 0.01 of a deviation
    _within(y, ry, torch.full_like(ry, 16 * 10 * 2 * E32 / 0.01), "y")
    _within(rstd, r[:, 0], 1e-4 * r[:, 0], "rstd")


def test_layer_norm_beyond_32_bit_offsets(ad):
    rows, dim = 2_800_000, 768  # 2.15e9 elements
    x = torch.empty(rows, dim, device="cuda", dtype=torch.float16)
    x[:8] = _randn(_gen(1), 8, dim, t="f16")
    x[8:-8].fill_(1.0)
    x[-8:] = x[:8]
    y, mean, rstd = ad.layer_norm(x, return_stats=True)
    assert torch.equal(y[:8], y[-8:]) and torch.equal(mean[:8], mean[-8:])
    assert torch.equal(y[:8], ad.layer_norm(x[:8].clone()))
    dx, dw, _ = ad.layer_norm_backward(x, x, mean, rstd, torch.ones(dim, device="cuda"))
    assert torch.equal(dx[:8], dx[-8:])


# ---- linear -------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 768, 1536), (2, 96, 96), (3, 33, 17), (7, 100, 257), (16, 128, 64), (17, 768, 130), (33, 64, 1),
          (64, 1, 64), (100, 1536, 768), (127, 72, 129), (128, 64, 256), (129, 65, 255), (200, 2000, 31),
          (257, 264, 520), (1000, 40, 300), (1500, 512, 384)]


def _act(z, act):
    return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v),
            "silu": lambda v: v * torch.sigmoid(v)}[act](z)


def _act_grad(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).to(z.dtype),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            "silu": lambda: s * (1 + z * (1 - s))}[act]()


def _linear_ref(x, w, b, res, act):
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z = z + b.double()
        mag = mag + b.double().abs()
    y = _act(z, act)
    if res is not None:
        y = y + res.double()
    return y, z, mag


def _check_linear(ad, x, w, b, res, act, t):
    y, pre = ad.linear(x, w, b, activation=act, residual=res, return_pre=True)
    ry, rz, mag = _linear_ref(x, w, b, res, act)
    ez = (x.shape[1] + 8) * 2 * E32 * mag
    _within(pre, rz, ez + U[t] * rz.abs() + TINY[t], "pre")
    add = 0.0 if res is None else 2 * E32 * res.double().abs()
    _within(y, ry, 1.2 * ez + ACT[t] * rz.abs().clamp(min=1) * (act not in ("none", "relu")) + 4 * E32 * ry.abs() + add
            + U[t] * ry.abs() + TINY[t], "y")
    return y, pre


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n * 7 + i)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    b, res = _randn(g, o, t=t, scale=0.3), _randn(g, n, o, t=t)
    y, _ = _check_linear(ad, x, w, b, res, act, t)
    assert torch.equal(y, ad.linear(x, w, b, activation=act, residual=res))
    _check_linear(ad, x, w, None, None, act, t)


def _check_backward(ad, dy, x, w, pre, act, t):
    dx, dw, db = ad.linear_backward(dy, x, w, pre=pre, activation=act)
    d = dy.double()
    f = torch.ones_like(d) if act == "none" else _act_grad(pre.double(), act)
    dz = d * f
    # dz is an operand of the products: rounded to the type where that is 16 bits
    soft = act in ("gelu", "silu")
    edz = (ACT[t] * d.abs() if soft else 0) + (0 if act == "none" else 2 * U[t] * dz.abs()) + TINY[t]
    edz = edz + torch.zeros_like(d)
    n, o = d.shape
    rdx, rdw, rdb = dz @ w.double(), dz.t() @ x.double(), dz.sum(0)
    mag = dz.abs() @ w.double().abs()
    _within(dx, rdx, edz @ w.double().abs() + (o + 8) * 2 * E32 * mag + U[t] * rdx.abs() + TINY[t], "dx")
    mag = dz.abs().t() @ x.double().abs()
    _within(dw, rdw, edz.t() @ x.double().abs() + (n + 8) * 2 * E32 * mag + U[t] * rdw.abs() + TINY[t], "dw")
    _within(db, rdb, (ACT[t] * d.abs().sum(0) if soft else 0) + (n + 8) * 2 * E32 * dz.abs().sum(0)
            + U[t] * rdb.abs() + TINY[t], "dbias")
    return dx, dw, db


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_backward(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n * 5 + o)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, o, t=t, scale=1.5)
    got = _check_backward(ad, dy, x, w, pre, act, t)
    again = ad.linear_backward(dy, x, w, pre=pre, activation=act)
    for u, v in zip(got, again):
        assert torch.equal(u, v)
    dx, dw, db = ad.linear_backward(dy, x, w, pre=pre, activation=act, param_grads=False)
    assert dw is None and db is None and torch.equal(dx, got[0])
    assert ad.linear_backward(dy, x, w, pre=pre, activation=act, input_grad=False)[0] is None


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", [(1, 56, 107), (1, 65, 1), (2, 1, 600), (3, 130, 1030), (4, 64, 512), (8, 300, 513), (5, 768, 1536)])
def test_linear_backward_of_few_rows(ad, shape, act, t):
    """dz is not rounded before its products: every gradient has one rounding."""
    n, i, o = shape
    g = _gen(i + o)
    x, w = _randn(g, n, i + 3, t=t)[:, 2:2 + i], _randn(g, o, i + 1, t=t, scale=i ** -0.5)[:, 1:]
    dy, pre = _randn(g, n, o + 5, t=t, scale=0.1)[:, 1:1 + o], _randn(g, n, o, t=t, scale=1.5)
    dx, dw, db = ad.linear_backward(dy, x, w, pre=None if act == "none" else pre, activation=act)
    f = torch.ones_like(pre.double()) if act == "none" else _act_grad(pre.double(), act)
    dz, mag = dy.double() * f, dy.double().abs() * (1 + f.abs())
    for got, want, m, k in ((dx, dz @ w.double(), mag @ w.double().abs(), o), (db, dz.sum(0), mag.sum(0), n),
                            (dw, dz.t() @ x.double(), mag.t() @ x.double().abs(), n)):
        _within(got, want, (k + 32) * 2 * E32 * m + U[t] * want.abs() + TINY[t], "gradient")
    again = ad.linear_backward(dy, x, w, pre=pre, activation=act, param_grads=False)
    assert torch.equal(again[0], dx) and again[1] is None
    only = ad.linear_backward(dy, x, w, pre=pre, activation=act, input_grad=False)
    assert only[0] is None and torch.equal(only[1], dw) and torch.equal(only[2], db)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", [(40000, 64, 128), (20000, 136, 264), (9000, 520, 1000), (30001, 72, 72),
                                   (2500, 40, 8200), (19000, 200, 100)])
@pytest.mark.parametrize("extras", ["", "bias", "pre", "residual", "bias pre residual"])
def test_linear_many_rows(ad, shape, t, extras):
    """Sizes of many tiles, with every combination the epilogue treats apart."""
    n, i, o = shape
    g = _gen(n)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    b = _randn(g, o, t=t) if "bias" in extras else None
    res = _randn(g, n, o, t=t) if "residual" in extras else None
    if "pre" in extras:
        _check_linear(ad, x, w, b, res, "gelu", t)
        _check_backward(ad, res if res is not None else _randn(g, n, o, t=t), x, w, _randn(g, n, o, t=t), "silu", t)
        return
    y = ad.linear(x, w, b, activation="silu", residual=res)
    ry, rz, mag = _linear_ref(x, w, b, res, "silu")
    _within(y, ry, 1.2 * (i + 8) * 2 * E32 * mag + ACT[t] * rz.abs().clamp(min=1) + 8 * E32 * (ry.abs() + rz.abs())
            + U[t] * ry.abs() + TINY[t], "y")


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lead", [0, 1, 4, 8])
def test_linear_strides_and_alignment(ad, t, lead):
    """Row strides beyond the row length, odd ones, and bases off 16 bytes."""
    g = _gen(lead)
    n, i, o = 150, 136, 200
    xs, ws = _randn(g, n, i + 8 + lead, t=t), _randn(g, o, i + 24 + lead, t=t, scale=i ** -0.5)
    rs = _randn(g, 2 * n, o + lead, t=t)
    x, w, res = xs[:, lead:lead + i], ws[:, lead:lead + i], rs[::2, lead:]
    b = _randn(g, o, t=t)
    _check_linear(ad, x, w, b, res, "gelu", t)
    _check_linear(ad, x[:1], w, b, res[:1], "gelu", t)
    _check_linear(ad, x[:40], w[3:], b[3:].clone(), None, "silu", t)
    _check_backward(ad, res, x, w, rs[1::2, lead:], "gelu", t)
    _check_backward(ad, res[5:], x[5:], w, None, "none", t)
    col = _randn(g, i, n, t=t).t()  # column-major: copied
    _check_linear(ad, col, w, None, None, "none", t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(300, 8192, 520), (1, 512, 264), (40, 512, 264), (700, 72, 264), (3000, 264, 333)])
def test_linear_vectors_off_their_alignment(ad, shape, t):
    """A bias one element off any boundary, residuals of an odd width, few rows to
    many, sums that are split over k and that are not."""
    n, i, o = shape
    g = _gen(n + o)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    b, res = _randn(g, o + 1, t=t)[1:], _randn(g, n, o + 3, t=t)[:, 1:1 + o]
    _check_linear(ad, x, w, b, res, "gelu", t)
    _check_linear(ad, x, w, b, None, "none", t)
    y = ad.linear(x, w, b, activation="silu", residual=res)
    assert torch.equal(y, ad.linear(x, w, b.clone(), activation="silu", residual=res.contiguous()))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 40, 2500), (2, 40, 2500), (3, 64, 2401), (4, 520, 2999), (5, 7, 2999), (8, 136, 4000)])
def test_linear_few_rows_many_columns(ad, shape, t):
    n, i, o = shape
    g = _gen(o + n)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    b, res = _randn(g, o, t=t, scale=0.3), _randn(g, n, o, t=t)
    _check_linear(ad, x, w, b, res, "gelu", t)
    _check_linear(ad, x, w, None, None, "none", t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_linear_nonfinite_stays_in_its_rows(ad, t, n):
    g = _gen(n)
    x, w = _randn(g, n, 256, t=t), _randn(g, 140, 256, t=t)
    x[n // 2, 3] = math.nan
    y = ad.linear(x, w, activation="relu")
    keep = torch.arange(n, device="cuda") != n // 2
    assert y[n // 2].isnan().all() and y[keep].isfinite().all()
    x[n // 2, 3] = math.inf
    y = ad.linear(x, w)
    want = torch.where(w[:, 3] > 0, math.inf, -math.inf).to(y.dtype)
    assert torch.equal(y[n // 2], want) and y[keep].isfinite().all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_activations_at_their_ends(ad, t):
    """w = 1: the activations at chosen points, their limits at infinity, NaN."""
    z = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 3.0, -3.0, 5.5, -5.5, 9.0, -9.0, 40.0, -40.0, 95.0, -95.0, 3e4, -3e4,
                      math.inf, -math.inf, math.nan], device="cuda", dtype=T[t])[:, None]
    one = torch.ones(1, 1, device="cuda", dtype=T[t])
    zd = z.double()
    for act, at_inf in (("none", (math.inf, -math.inf)), ("relu", (math.inf, 0)), ("gelu", (math.inf, 0)),
                        ("silu", (math.inf, 0))):
        y = ad.linear(z, one, activation=act)[:, 0].double()
        want = _act(zd, act)[:, 0]
        tol = (ACT[t] if act in ("gelu", "silu") else 0) * zd[:, 0].abs().clamp(min=1) + U[t] * want.abs() + TINY[t]
        _within(y[:16], want[:16], tol[:16], act)
        assert (y[16], y[17]) == at_inf and y[18].isnan()
        d = ad.linear_backward(torch.ones_like(z), z, one, pre=z, activation=act, param_grads=False)[0][:, 0].double()
        want = _act_grad(zd, act)[:, 0]
        _within(d[:16], want[:16], ACT[t] * 2 + 3 * U[t] * want[:16].abs() + TINY[t], act + "'")
        assert d[16] == 1 and d[17] == (act == "none")
        if act in ("gelu", "silu"):
            assert d[18].isnan()


def test_linear_overflow_and_empty(ad):
    x = torch.full((40, 64), 300.0, device="cuda", dtype=torch.float16)
    y = ad.linear(x, x[:8].contiguous())
    assert torch.isinf(y).all() and (y > 0).all()  # 64 * 300^2 is past float16's largest
    e = torch.empty(0, 64, device="cuda")
    w = torch.ones(32, 64, device="cuda")
    y, pre = ad.linear(e, w, return_pre=True)
    assert y.shape == (0, 32) and pre.shape == (0, 32)
    dx, dw, db = ad.linear_backward(y, e, w, pre=pre, activation="gelu")
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_linear_beyond_32_bit_offsets(ad):
    rows, i, o = 2_800_000, 768, 64
    x = torch.empty(rows, i, device="cuda", dtype=torch.bfloat16)
    x[:200] = _randn(_gen(1), 200, i, t="bf16")
    x[200:-200].fill_(0.5)
    x[-200:] = x[:200]
    w = _randn(_gen(2), o, i, t="bf16", scale=0.04)
    y = ad.linear(x, w, activation="silu")
    assert torch.equal(y[:200], y[-200:]) and y[:200].float().std() > 0.1
    w2 = w.t().contiguous()  # 2.15e9 outputs
    z = ad.linear(y, w2)
    assert torch.equal(z[:200], z[-200:])
    _check_linear(ad, x[-200:], w, None, None, "silu", "bf16")


# ---- preference loss ----------------------------------------------------------------

def _pairs(g, nq, nb, counts, holes=True):
    off = torch.zeros(nq + 1, dtype=torch.int64, device="cuda")
    off[1:] = torch.as_tensor(counts, device="cuda").cumsum(0)
    m = int(off[-1])
    pos = torch.randint(0, nb, (m,), generator=g, device="cuda", dtype=torch.int32)
    neg = torch.randint(0, nb, (m,), generator=g, device="cuda", dtype=torch.int32)
    if holes and m > 4:
        neg[1::7] = -1
        pos[3::11] = nb
    return off, pos, neg


def _pref_ref(q, base, off, pos, neg, ref, w, beta, e, metric):
    nq, nb = q.shape[0], base.shape[0]
    m = pos.numel()
    i = torch.repeat_interleave(torch.arange(nq, device="cuda"), off[1:] - off[:-1])
    fine = (pos >= 0) & (pos < nb) & (neg >= 0) & (neg < nb)
    b = base.double()
    up, dn = b[torch.where(fine, pos, 0).long()], b[torch.where(fine, neg, 0).long()]
    q, r = q.double(), None if ref is None else ref.double()

    def s(v, d):
        return (v[i] * d).sum(1) if metric == "ip" else -((v[i] - d) ** 2).sum(1)

    z = s(q, up) - s(q, dn)
    if r is not None:
        z = z - (s(r, up) - s(r, dn))
    z = beta * z * fine
    w = torch.ones(m, dtype=torch.float64, device="cuda") if w is None else w.double()
    sp = torch.nn.functional.softplus
    loss = ((1 - e) * sp(-z) + e * sp(z)) * fine
    k = (2 if metric == "l2" else 1) * beta
    coef = (e - torch.sigmoid(-z)) * fine * w * k
    dq = torch.zeros_like(q).index_add_(0, i, coef[:, None] * (up - dn))
    # magnitudes for the bounds
    u = q[i] if r is None else (q - r)[i]
    um = u.abs() + (0.5 * (up + dn).abs() if r is None and metric == "l2" else 0)
    zm = k * (um * (up - dn).abs()).sum(1) * fine
    return loss, z, dq, i, fine, w, k, coef, (up - dn), zm


def _check_pref(ad, q, base, off, pos, neg, t, ref=None, w=None, beta=1.0, e=0.0, metric="ip"):
    losses, margins, dq = ad.preference_loss(q, base, off, pos, neg, ref=ref, weights=w, beta=beta, label_smoothing=e,
                                             metric=metric)
    loss, z, rdq, i, fine, wd, k, coef, diff, zm = _pref_ref(q, base, off, pos, neg, ref, w, beta, e, metric)
    d = q.shape[1]
    ez = (d + 16) * 2 * E32 * zm + 2 * E32
    _within(margins, z, ez * fine, "margins")
    _within(losses, loss, (ez + 8 * E32 * (1 + loss)) * fine, "losses")
    n = torch.bincount(i, minlength=q.shape[0])[:, None].double()
    mag = torch.zeros_like(rdq).index_add_(0, i, (coef.abs()[:, None] * diff.abs()))
    ec = torch.zeros_like(rdq).index_add_(0, i, ((ez / 4 + 8 * E32) * wd * k * fine)[:, None] * diff.abs())
    _within(dq, rdq, ec + (n + 8) * 2 * E32 * mag + U[t] * rdq.abs() + TINY[t], "dq")
    assert not losses[~fine].any() and not margins[~fine].any()
    l2, m2, none = ad.preference_loss(q, base, off, pos, neg, ref=ref, weights=w, beta=beta, label_smoothing=e,
                                      metric=metric, grad=False)
    assert none is None and torch.equal(l2, losses) and torch.equal(m2, margins)
    again = ad.preference_loss(q, base, off, pos, neg, ref=ref, weights=w, beta=beta, label_smoothing=e, metric=metric)
    assert torch.equal(again[2], dq)
    return losses, margins, dq


def _base(g, nb, d, bt):
    if bt == "u8":
        return torch.randint(0, 256, (nb, d), generator=g, device="cuda", dtype=torch.uint8)
    return _randn(g, nb, d, t=bt, scale=d ** -0.5)


@pytest.mark.parametrize("metric", ["ip", "l2"])
@pytest.mark.parametrize("t,bt", [("f32", "f32"), ("f32", "u8"), ("f16", "f16"), ("bf16", "f16"), ("f32", "bf16"),
                                  ("f16", "u8")])
@pytest.mark.parametrize("dim", [1, 7, 32, 96, 100, 128, 250, 256, 257, 512, 768, 1000, 1024, 1100, 1536, 4096, 5000])
def test_preference(ad, dim, t, bt, metric):
    g = _gen(dim)
    nq, nb = 21, 50
    counts = [0, 1, 2, 3, 5, 8, 13, 40, 0, 1] + [4] * 11
    base = _base(g, nb, dim, bt)
    s = 30.0 if bt == "u8" else dim ** -0.5
    q, ref = _randn(g, nq, dim, t=t, scale=s), _randn(g, nq, dim, t=t, scale=s)
    off, pos, neg = _pairs(g, nq, nb, counts)
    w = torch.rand(int(off[-1]), generator=g, device="cuda")
    beta = 1e-3 / dim ** 0.5 if bt == "u8" else 2.0
    for r in (ref, None):
        _, _, dq = _check_pref(ad, q, base, off, pos, neg, t, ref=r, w=w, beta=beta, e=0.1, metric=metric)
        assert not dq[0].any() and not dq[8].any()  # queries without pairs
        _check_pref(ad, q, base, off, pos, neg, t, ref=r, beta=beta * 30, metric=metric)


def test_preference_many_and_few_pairs(ad):
    g = _gen(5)
    base = _base(g, 3000, 768, "f16")
    for counts in ([700], [0], [1], [3, 999, 0, 2], [0, 0, 0], list(range(60))):
        q = _randn(g, len(counts), 768, t="f16", scale=0.04)
        off, pos, neg = _pairs(g, len(counts), 3000, counts)
        _check_pref(ad, q, base, off, pos, neg, "f16", ref=_randn(g, len(counts), 768, t="f16", scale=0.04), beta=3.0)


def test_preference_extreme_margins_and_masks(ad):
    d = 64
    base = torch.zeros(3, d, device="cuda")
    base[1] = 1e3
    base[2, 0] = math.nan
    q = torch.ones(5, d, device="cuda")
    off = torch.tensor([0, 1, 2, 3, 4, 5], device="cuda")
    pos = torch.tensor([1, 0, -1, 0, 0], dtype=torch.int32, device="cuda")
    neg = torch.tensor([0, 1, 2, 3, 0], dtype=torch.int32, device="cuda")
    losses, margins, dq = ad.preference_loss(q, base, off, pos, neg, beta=100.0)
    assert losses[0] == 0 and margins[0] == 6.4e6 and not dq[0].any()  # certain: no loss, no gradient
    assert losses[1] == 6.4e6 and margins[1] == -6.4e6 and torch.equal(dq[1], torch.full((d,), 1e5, device="cuda"))
    assert not losses[2:4].any() and not dq[2:4].any()  # masked: the NaN document is not read into them
    assert abs(float(losses[4]) - math.log(2)) < 1e-6 and not dq[4].any()  # equal documents


def test_preference_strides_empty_and_bad_offsets(ad):
    g = _gen(8)
    base = _base(g, 40, 96, "f32")
    big = _randn(g, 12, 120)
    off, pos, neg = _pairs(g, 6, 40, [2, 0, 5, 1, 3, 4])
    q, r = big[::2, 5:101], big[1::2, 8:104]
    _check_pref(ad, q, base, off, pos, neg, "f32", ref=r)
    out = ad.preference_loss(q[:0], base, off[:1] * 0, pos[:0], neg[:0])
    assert out[0].shape == (0,) and out[2].shape == (0, 96)
    # offsets past the pairs are clamped, descending ones leave a query empty
    bad = torch.tensor([0, 2, -5, 9, 1 << 40, 3, 15], device="cuda")
    losses, _, dq = ad.preference_loss(q, base, bad, pos, neg)
    assert dq.isfinite().all() and losses.shape == (15,)


def test_preference_beyond_32_bit_offsets(ad):
    nb, d = 4_400_000, 512  # 2.25e9 bytes
    base = torch.randint(0, 256, (nb, d), device="cuda", dtype=torch.uint8, generator=_gen(1))
    q, ref = _randn(_gen(2), 4, d, scale=20.0), _randn(_gen(3), 4, d, scale=20.0)
    off = torch.arange(5, device="cuda") * 2
    pos = torch.tensor([nb - 1, nb - 2, nb - 3, 5, 4_250_000, 1, nb - 9, 0], dtype=torch.int32, device="cuda")
    neg = torch.tensor([3, nb - 7, 4_200_001, nb - 1, 9, nb - 2, nb - 1, nb - 5], dtype=torch.int32, device="cuda")
    sub = torch.cat([pos, neg]).unique()
    to = {int(v): k for k, v in enumerate(sub)}
    small = base[sub.long()].contiguous()
    mp = [torch.tensor([to[int(v)] for v in x], dtype=torch.int32, device="cuda") for x in (pos, neg)]
    a = ad.preference_loss(q, base, off, pos, neg, ref=ref, beta=1e-5, metric="l2")
    b = ad.preference_loss(q, small, off, *mp, ref=ref, beta=1e-5, metric="l2")
    for u, v in zip(a, b):
        assert torch.equal(u, v)


# ---- gradients against differences ----------------------------------------------------

def _plain_loss(p, q, base, off, pos, neg, beta, metric, act):
    """The adapter's loss in 64 bits."""
    q = q.double()
    h = _norm_ref(q, p["norm_weight"], p["norm_bias"], 1e-5)[0]
    h = _act(h @ p["w1"].double().t() + p["b1"].double(), act)
    out = q + h @ p["w2"].double().t() + p["b2"].double()
    return _pref_ref(out, base, off, pos, neg, q, None, beta, 0.0, metric)[0].sum()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("metric", ["ip", "l2"])
def test_train_step_against_differences(ad, metric, act):
    """Each parameter's gradient along a random direction against the central
    difference of the 64-bit loss.  The gradients are float32 through a few
    hundred operations: 2^-24 * 2000 of their magnitude; the difference's
    step of 1e-5 leaves 1e-9."""
    g = _gen(11)
    d, hid, nq, nb = 40, 72, 50, 60
    base = _randn(g, nb, d, scale=0.3)
    q = _randn(g, nq, d, scale=0.3)
    off, pos, neg = _pairs(g, nq, nb, [k % 5 for k in range(nq)])
    m = ad.QueryAdapter(d, hid, act, seed=1)
    for k in m.params:
        m.params[k] += _randn(g, *m.params[k].shape, scale=0.2)
    losses, margins = m.train_step(q, base, off, pos, neg, beta=1.5, metric=metric)
    want = _plain_loss(m.params, q, base, off, pos, neg, 1.5, metric, act)
    assert abs(float(losses.double().sum() - want)) <= 2000 * E32 * float(want)
    for k, v in m.params.items():
        for _ in range(3):
            u = _randn(g, *v.shape).double()
            step = 1e-5 / float(u.norm())
            vals = []
            for sgn in (1, -1):
                p = {n: t.double() for n, t in m.params.items()}
                p[k] = p[k] + sgn * step * u
                vals.append(float(_plain_loss(p, q, base, off, pos, neg, 1.5, metric, act)))
            diff = (vals[0] - vals[1]) / (2 * step)
            got = float((v.grad.double() * u).sum())
            scale = float(v.grad.double().norm() * u.norm())
            assert abs(got - diff) <= 2000 * E32 * scale + 1e-7 * float(u.norm()), k


# ---- streams, refusals, the whole -----------------------------------------------------

def test_query_adapter_converts_on_its_stream(ad):
    """Queries of another type are converted on the stream of the call, not on the
    current one, which is busy here."""
    from fusiongpu_b200 import QueryAdapter
    a = QueryAdapter(96, 160, dtype=torch.float16)
    a.params["w2"].normal_(generator=_gen(1))
    q = _randn(_gen(2), 300, 96)
    want = a(q)
    torch.empty(300, 96, device="cuda", dtype=torch.float16).fill_(math.nan)  # what an unfinished conversion leaves
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    got = a(q, stream=s)
    s.synchronize()
    assert torch.equal(got, want)


def test_operators_on_another_stream(ad):
    g = _gen(4)
    x, w = _randn(g, 3000, 512, t="bf16"), _randn(g, 256, 512, t="bf16", scale=0.05)
    dy, pre = _randn(g, 3000, 256, t="bf16"), _randn(g, 3000, 256, t="bf16")
    here = ad.linear_backward(dy, x, w, pre=pre, activation="gelu")
    ln = ad.layer_norm(x, return_stats=True)
    lb = ad.layer_norm_backward(x, x, ln[1], ln[2])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        there = ad.linear_backward(dy, x, w, pre=pre, activation="gelu", stream=s)
        ln2 = ad.layer_norm(x, return_stats=True, stream=s)
        lb2 = ad.layer_norm_backward(x, x, ln2[1], ln2[2], stream=s)
        torch.empty(1 << 22, device="cuda").fill_(7)  # the default stream's allocations stay off that workspace
    s.synchronize()
    for u, v in zip(here + ln + lb, there + ln2 + lb2):
        assert torch.equal(u, v)


def test_operators_in_a_cuda_graph(ad):
    """The serving path for one query, captured and replayed on new queries."""
    m = ad.QueryAdapter(256, 512, dtype=torch.float16)
    m.params["w2"].normal_(std=0.05)
    q = _randn(_gen(1), 1, 256, t="f16")
    m(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(q)
    for seed in range(3):
        q.copy_(_randn(_gen(seed), 1, 256, t="f16"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m(q))


def test_refusals(ad):
    x = torch.zeros(4, 32, device="cuda")
    w = torch.zeros(8, 32, device="cuda")
    off = torch.zeros(5, dtype=torch.int64, device="cuda")
    ids = torch.zeros(0, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        ad.layer_norm(x.cpu())
    with pytest.raises(TypeError):
        ad.layer_norm(x.double())
    with pytest.raises(TypeError):
        ad.layer_norm(x, x[0].half())
    with pytest.raises(ValueError):
        ad.layer_norm(x, torch.ones(31, device="cuda"))
    with pytest.raises(ValueError):
        ad.layer_norm_backward(x[:3], x, x[:, 0].contiguous(), x[:, 0].contiguous())
    with pytest.raises(TypeError):
        ad.linear(x, w.half())
    with pytest.raises(ValueError):
        ad.linear(x, w[:, :31])
    with pytest.raises(ValueError):
        ad.linear(x, w, activation="tanh")
    with pytest.raises(ValueError):
        ad.linear(x, w, residual=x)
    with pytest.raises(ValueError):
        ad.linear_backward(x[:, :8], x, w, activation="gelu")
    with pytest.raises(TypeError):
        ad.preference_loss(x, x, off, ids.long(), ids)
    with pytest.raises(TypeError):
        ad.preference_loss(x, x, off.int(), ids, ids)
    with pytest.raises(ValueError):
        ad.preference_loss(x, x, off[:4], ids, ids)
    with pytest.raises(ValueError):
        ad.preference_loss(x, x[:, :16], off, ids, ids)
    with pytest.raises(ValueError):
        ad.preference_loss(x, x, off, ids, ids, metric="cosine")
    from fusiongpu_b200 import _lib
    for kw in (dict(beta=0.0), dict(beta=math.nan), dict(label_smoothing=0.6), dict(label_smoothing=-0.1)):
        with pytest.raises(_lib.FgError):
            ad.preference_loss(x, x, off, ids, ids, **kw)
    with pytest.raises(_lib.FgError):
        ad.layer_norm(x, eps=-1.0)
    with pytest.raises(_lib.FgError):
        ad.layer_norm(torch.zeros(2, 20000, device="cuda"))


def test_adapter_trains_and_serves_an_index(ad):
    """Queries from a shifted embedding: the adapter learns from labelled pairs
    to find what the index holds, through the index's own search."""
    import examples.train_query_adapter as ex
    before, after = ex.run(nbase=4000, dim=64, nq=512, nlist=32, pq_m=16, hidden=128, steps=60, verbose=False)
    assert after > before + 0.1
