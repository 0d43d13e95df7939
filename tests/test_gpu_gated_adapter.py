"""GPU tests of the gated layer, the quantisation of rows and the 8-bit linear layer
against plain implementations in 64 bits.

Tolerances follow from the arithmetic, element by element.  U[t] is the unit
roundoff of a result's type, E32 = 2^-24 that of the 32-bit sums; a sum of n
products in 32 bits, in any order and with truncating additions, is within
(n + 8) * 2 * E32 of the sum of the products' magnitudes.  The kernels' activation
functions are held to ACT (an absolute error per unit of max(|z|, 1)).  A product
of factors in 32 bits adds 4 * E32 of itself.  An operand in parts (the gradients
of the pre-activations) is within PART[t] of its value, plus LOW[t].
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
ACT = {"f32": 2.0 ** -20, "f16": 2.0 ** -18, "bf16": 2.0 ** -18}
PART = {"f32": 2.0 ** -23, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}
LOW = {"f32": 2.0 ** -130, "f16": 2.0 ** -36, "bf16": 2.0 ** -130}
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


def _act(z, act):
    return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v),
            "silu": lambda v: v * torch.sigmoid(v)}[act](z)


def _act_grad(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).to(z.dtype),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            "silu": lambda: s * (1 + z * (1 - s))}[act]()


# ---- gated layer --------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 768, 1024), (2, 96, 96), (3, 33, 17), (7, 100, 257), (9, 40, 8), (16, 128, 64), (17, 768, 130),
          (33, 64, 1), (64, 1, 64), (100, 768, 1024), (127, 72, 129), (128, 64, 256), (129, 65, 255), (200, 2000, 31),
          (257, 264, 520), (1000, 40, 300), (1500, 512, 384)]


def _check_gated(ad, x, w, b, act, t):
    h = w.shape[0] // 2
    y, pre = ad.gated_linear(x, w, b, activation=act, return_pre=True)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = (x.shape[1] + 8) * 2 * E32 * mag
    _within(pre, z, ez + U[t] * z.abs() + TINY[t], "pre")
    a, p = _act(z[:, :h], act), z[:, h:]
    ea = 1.2 * ez[:, :h] + (ACT[t] * z[:, :h].abs().clamp(min=1) if act in ("gelu", "silu") else 0)
    ry = a * p
    _within(y, ry, ea * (p.abs() + ez[:, h:]) + a.abs() * ez[:, h:] + 4 * E32 * ry.abs() + U[t] * ry.abs() + TINY[t], "y")
    assert torch.equal(y, ad.gated_linear(x, w, b, activation=act))
    return y, pre


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gated(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n * 7 + i)
    x, w = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=i ** -0.5)
    _check_gated(ad, x, w, _randn(g, 2 * o, t=t, scale=0.3), act, t)
    _check_gated(ad, x, w, None, act, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(40000, 64, 64), (20000, 136, 136), (9000, 520, 520), (30001, 72, 40), (6001, 264, 1000),
                                   (8000, 101, 333)])
def test_gated_many_rows(ad, shape, t):
    n, i, o = shape
    g = _gen(n + o)
    x, w = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=i ** -0.5)
    _check_gated(ad, x, w, _randn(g, 2 * o, t=t, scale=0.3), "silu", t)
    _check_gated(ad, x, w, None, "gelu", t)


def _check_gated_backward(ad, dy, x, w, pre, act, t):
    h = dy.shape[1]
    dx, dw, db = ad.gated_linear_backward(dy, x, w, pre, activation=act)
    d, z, p = dy.double(), pre[:, :h].double(), pre[:, h:].double()
    f, a = _act_grad(z, act), _act(z, act)
    dz = torch.cat([d * p * f, d * a], 1)
    soft = ACT[t] if act in ("gelu", "silu") else 0.0
    edz = torch.cat([soft * (d * p).abs(), soft * d.abs() * z.abs().clamp(min=1)], 1) + 4 * E32 * dz.abs()
    part = edz + PART[t] * dz.abs() + LOW[t]  # as an operand
    n, k = d.shape[0], 2 * h
    rdx, rdw, rdb = dz @ w.double(), dz.t() @ x.double(), dz.sum(0)
    _within(dx, rdx, part @ w.double().abs() + (k + 8) * 2 * E32 * (dz.abs() @ w.double().abs()) + U[t] * rdx.abs() + TINY[t], "dx")
    _within(dw, rdw, part.t() @ x.double().abs() + (n + 8) * 2 * E32 * (dz.abs().t() @ x.double().abs()) + U[t] * rdw.abs()
            + TINY[t], "dw")
    _within(db, rdb, edz.sum(0) + (n + 8) * 2 * E32 * dz.abs().sum(0) + U[t] * rdb.abs() + TINY[t], "dbias")
    return dx, dw, db


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", SHAPES + [(5000, 72, 104), (3, 64, 2000), (8, 264, 700)])
def test_gated_backward(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n * 5 + o)
    x, w = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, 2 * o, t=t, scale=1.5)
    got = _check_gated_backward(ad, dy, x, w, pre, act, t)
    for u, v in zip(got, ad.gated_linear_backward(dy, x, w, pre, activation=act)):
        assert torch.equal(u, v)
    dx, dw, db = ad.gated_linear_backward(dy, x, w, pre, activation=act, param_grads=False)
    assert dw is None and db is None and torch.equal(dx, got[0])
    dx, dw, db = ad.gated_linear_backward(dy, x, w, pre, activation=act, input_grad=False)
    assert dx is None and torch.equal(dw, got[1]) and torch.equal(db, got[2])


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(30000, 24, 1), (20001, 16, 9), (30000, 40, 32), (12345, 33, 40), (9999, 17, 64), (20000, 24, 65),
                                   (5001, 65, 128), (4000, 40, 129), (10000, 8, 333)])
def test_gated_backward_narrow(ad, shape, t):
    """Layers as narrow as a part of a warp, on rows that more than fill the GPU."""
    n, i, o = shape
    g = _gen(n + o)
    x, w = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, 2 * o, t=t, scale=1.5)
    got = _check_gated_backward(ad, dy, x, w, pre, "silu", t)
    wide = _randn(g, n, o + 11, t=t)  # the same from rows that start anywhere
    wide[:, 3:3 + o] = dy
    for u, v in zip(got, ad.gated_linear_backward(wide[:, 3:3 + o], x, w, pre, activation="silu")):
        assert torch.equal(u, v)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(10000, 768, 1024), (3000, 256, 256), (5000, 700, 450), (2500, 520, 300), (20000, 256, 640)])
def test_gated_backward_in_parts(ad, shape, t):
    """Sums over rows in three, five, ... parts, whichever fill the GPU."""
    n, i, o = shape
    g = _gen(n + i)
    x, w = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, 2 * o, t=t, scale=1.5)
    got = _check_gated_backward(ad, dy, x, w, pre, "gelu", t)
    for u, v in zip(got, ad.gated_linear_backward(dy, x, w, pre, activation="gelu")):
        assert torch.equal(u, v)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("n", [5, 200])
def test_gated_backward_against_differences(ad, act, n):
    """The gradients against central differences of the definition in 64 bits, along
    random directions: off by step^2 / 6 times a third derivative, which for sums of
    this size stays below 10, and by the gradients' own error."""
    g = _gen(n)
    x, w, b = _randn(g, n, 24), _randn(g, 40, 24, scale=0.2), _randn(g, 40, scale=0.3)
    dy = _randn(g, n, 20, scale=0.1)
    _, pre = ad.gated_linear(x, w, b, activation=act, return_pre=True)
    grads = ad.gated_linear_backward(dy, x, w, pre, activation=act)

    def value(v):
        z = v[0] @ v[1].t() + v[2]
        return float((dy.double() * _act(z[:, :20], act) * z[:, 20:]).sum())

    at, step = [x.double(), w.double(), b.double()], 1e-4
    for k in range(3):
        u = torch.randn(at[k].shape, generator=g, device="cuda", dtype=torch.float64)
        up, down = list(at), list(at)
        up[k], down[k] = at[k] + step * u, at[k] - step * u
        want = (value(up) - value(down)) / (2 * step)
        got = float((grads[k].double() * u).sum())
        mag = float((grads[k].double() * u).abs().sum())
        assert abs(got - want) <= 1e-5 * mag + 100 * step ** 2, (k, got, want)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lead", [0, 1, 4, 8])
@pytest.mark.parametrize("n", [3, 300, 5000])
def test_gated_strides_and_alignment(ad, t, lead, n):
    """Rows that start anywhere: the same values as from contiguous rows."""
    g = _gen(lead + n)
    x, w = _randn(g, n, 200, t=t)[:, lead:lead + 72], _randn(g, 144, 200, t=t, scale=0.1)[:, lead:lead + 72]
    dy, b = _randn(g, n, 90, t=t)[:, lead:lead + 72], _randn(g, 144, t=t)
    y, pre = ad.gated_linear(x, w, b, return_pre=True)
    wide = torch.empty(n, 160, device="cuda", dtype=T[t])
    wide[:, lead:lead + 144] = pre
    grads = ad.gated_linear_backward(dy, x, w, wide[:, lead:lead + 144])
    _check_gated(ad, x, w, b, "silu", t)
    if n > 8:  # of up to eight rows, rows off 16 bytes are added in another order
        xc, wc = x.contiguous(), w.contiguous()
        assert torch.equal(y, ad.gated_linear(xc, wc, b))
        for u, v in zip(grads, ad.gated_linear_backward(dy.contiguous(), xc, wc, pre)):
            assert torch.equal(u, v)
    _check_gated_backward(ad, dy, x, w, wide[:, lead:lead + 144], "silu", t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 40, 300, 20000])
def test_gated_nonfinite_stays_in_its_rows(ad, t, n):
    g = _gen(n)
    x, w = _randn(g, n, 64, t=t), _randn(g, 96, 64, t=t, scale=0.1)
    clean = ad.gated_linear(x, w)
    bad = x.clone()
    bad[n // 2, 5] = math.nan
    y, pre = ad.gated_linear(bad, w, return_pre=True)
    keep = torch.arange(n, device="cuda") != n // 2
    assert y[n // 2].isnan().all() and pre[n // 2].isnan().all() and torch.equal(y[keep], clean[keep])
    bad[n // 2, 5] = math.inf
    y, pre = ad.gated_linear(bad, w, activation="none", return_pre=True)
    z = bad[n // 2].double() @ w.double().t()
    assert torch.equal(pre[n // 2].double(), z)
    assert torch.equal(y[n // 2].double(), z[:48] * z[48:])
    assert torch.equal(y[keep], ad.gated_linear(x, w, activation="none")[keep])


def test_gated_empty(ad):
    for t in T:
        x, w = torch.empty(0, 40, device="cuda", dtype=T[t]), torch.ones(60, 40, device="cuda", dtype=T[t])
        y, pre = ad.gated_linear(x, w, return_pre=True)
        assert y.shape == (0, 30) and pre.shape == (0, 60)
        dx, dw, db = ad.gated_linear_backward(y, x, w, pre)
        assert dx.shape == (0, 40) and dw.shape == (60, 40) and not dw.any() and not db.any()


def test_gated_beyond_32_bit_offsets(ad):
    n, i, o = 1_100_000, 24, 1000  # pre holds 2.2e9 elements
    g = _gen(2)
    x = torch.ones(n, i, device="cuda", dtype=torch.float16)
    x[:300] = _randn(g, 300, i, t="f16")
    x[-300:] = x[:300]
    w, b = _randn(g, 2 * o, i, t="f16", scale=0.2), _randn(g, 2 * o, t="f16")
    y, pre = ad.gated_linear(x, w, b, return_pre=True)
    small, spre = ad.gated_linear(x[:300], w, b, return_pre=True)
    for k in (slice(0, 300), slice(n - 300, n)):
        # another kernel may take 300 rows: the same sums to 32 bits
        _within(y[k], small.double(), 2 ** -9 * small.double().abs() + 2 ** -10, "y")
        _within(pre[k], spre.double(), 2 ** -9 * spre.double().abs() + 2 ** -10, "pre")
    assert torch.equal(y[:300], y[-300:]) and torch.equal(pre[:300], pre[-300:])
    dy = torch.zeros(n, o, device="cuda", dtype=torch.float16)
    dy[:300] = _randn(g, 300, o, t="f16")
    dy[-300:] = dy[:300]
    dx, _, _ = ad.gated_linear_backward(dy, x, w, pre, param_grads=False)
    assert torch.equal(dx[:300], dx[-300:]) and not dx[300:-300].any()


# ---- codes of rows ------------------------------------------------------------------

DIMS = [1, 2, 7, 16, 31, 64, 100, 128, 255, 256, 333, 512, 768, 1000, 1024, 1025, 1536, 2048, 2049, 4096, 4100, 8192, 8200, 20000]


def _quantised(x):
    """Scales and codes by the definition."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True) if x.shape[0] else x.new_zeros(0, 1)
    q = torch.where(top > 0, 127 * x / top.clamp(min=5e-324), torch.zeros_like(x)).round()
    return q.to(torch.int8), (top[:, 0] / 127).float()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
def test_quantize_rows(ad, dim, t):
    g = _gen(dim)
    for rows in (0, 1, 5, 300):
        x = _randn(g, rows, dim, t=t, scale=0.7)
        for view in (x, _randn(g, rows, dim + 3, t=t)[:, 1:1 + dim]):
            q, s = ad.quantize_rows(view)
            rq, rs = _quantised(view)
            assert q.dtype == torch.int8 and torch.equal(q, rq) and torch.equal(s, rs)
            assert q.data_ptr() % 16 == 0 and (rows < 2 or q.stride(0) % 16 == 0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,dim", [(100_001, 1), (60_000, 9), (50_001, 40), (40_000, 100), (20_001, 129), (20_000, 333),
                                      (9_001, 600), (3_001, 1025), (2_501, 3001)])
def test_quantize_more_rows_than_groups(ad, rows, dim, t):
    x = _randn(_gen(rows), rows, dim, t=t)
    x[rows // 2] = math.nan
    q, s = ad.quantize_rows(x)
    good = torch.arange(rows, device="cuda") != rows // 2
    rq, rs = _quantised(x[good])
    assert torch.equal(q[good], rq) and torch.equal(s[good], rs)
    assert s[rows // 2].isnan() and not q[rows // 2].any()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [40, 700, 1500, 9000])
def test_quantize_rows_at_its_ends(ad, t, dim):
    f = torch.finfo(T[t])
    x = torch.zeros(12, dim, device="cuda", dtype=T[t])
    x[1] = 0
    x[2, 3], x[2, 4] = f.max, -f.max
    x[3, 5], x[3, 6] = f.smallest_normal, -f.smallest_normal / 2  # a row of the smallest numbers
    x[4] = f.smallest_normal / 4
    x[5] = (torch.arange(dim, device="cuda") % 128 + 0.5).to(T[t]) / 2  # halves between codes where the largest is 63.5
    x[5, 0] = 63.5
    x[6] = -1
    x[7, dim - 1] = math.nan
    x[8, 0] = math.inf
    x[9, dim // 2] = -math.inf
    x[10] = torch.arange(dim, device="cuda").to(T[t])
    q, s = ad.quantize_rows(x)
    rq, rs = _quantised(x)
    good = [0, 1, 2, 3, 4, 5, 6, 10, 11]
    assert torch.equal(q[good], rq[good]) and torch.equal(s[good], rs[good])
    assert s[7:10].isnan().all() and not q[7:10].any()
    assert s[0] == 0 and not q[0].any() and (q[6] == -127).all()


def test_quantize_rows_near_halves(ad):
    """float32 values within a few units in the last place of a half between codes."""
    for top in (1.0, 0.7, 3.3e-38, 1e30, 127.0):
        half = ((torch.arange(126, device="cuda", dtype=torch.float64) + 0.5) * torch.tensor(top, dtype=torch.float32).double() / 127)
        rows = []
        for step in range(-3, 4):
            v = half.float()
            for _ in range(abs(step)):
                v = torch.nextafter(v, torch.full_like(v, math.inf if step > 0 else -math.inf))
            rows.append(torch.cat([torch.tensor([top], device="cuda"), v, -v]))
        x = torch.stack(rows)
        q, s = ad.quantize_rows(x)
        rq, rs = _quantised(x)
        assert torch.equal(q, rq) and torch.equal(s, rs)


def test_quantize_rows_beyond_32_bit_offsets(ad):
    x = torch.empty(2_200_000, 1000, device="cuda", dtype=torch.float16).fill_(0.5)
    x[:8] = _randn(_gen(1), 8, 1000, t="f16")
    x[-8:] = x[:8]
    q, s = ad.quantize_rows(x)
    rq, rs = _quantised(x[:8])
    for k in (slice(0, 8), slice(-8, None)):
        assert torch.equal(q[k], rq) and torch.equal(s[k], rs)


# ---- 8-bit linear layer -------------------------------------------------------------

def _code(g, n, d, pad=16):
    ld = (d + pad - 1) // pad * pad
    q = torch.randint(-128, 128, (n, ld), generator=g, device="cuda", dtype=torch.int8)
    return q[:, :d]


def _check_int8(ad, x, xs, w, ws, b, res, act, t):
    y = ad.linear_int8(x, xs, w, ws, b, activation=act, residual=res, dtype=T[t])
    s = x.double() @ w.double().t()  # exact
    z = s * (xs.double()[:, None] * ws.double())
    ez = 3 * E32 * z.abs()  # the sum in 32 bits, the scales' product, theirs
    if b is not None:
        z = z + b.double()
        ez = ez + E32 * z.abs()
    ry = _act(z, act)
    ey = 1.2 * ez + (ACT[t] * z.abs().clamp(min=1) if act in ("gelu", "silu") else 0) + 4 * E32 * ry.abs()
    if res is not None:
        ry = ry + res.double()
        ey = ey + 2 * E32 * (res.double().abs() + ry.abs())
    _within(y, ry, ey + U[t] * ry.abs() + TINY[t], "y")
    assert torch.equal(y, ad.linear_int8(x, xs, w, ws, b, activation=act, residual=res, dtype=T[t]))
    return y


INT8_SHAPES = [(1, 1, 1), (1, 768, 1536), (2, 96, 96), (3, 33, 17), (4, 16, 40), (7, 100, 257), (8, 1000, 64), (9, 40, 8),
               (16, 128, 64), (17, 768, 130), (33, 64, 1), (64, 1, 64), (100, 1536, 768), (127, 72, 129), (128, 128, 256),
               (129, 65, 255), (200, 4000, 31), (257, 264, 520), (1000, 40, 300), (1500, 512, 384)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("shape", INT8_SHAPES)
def test_linear_int8(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n * 3 + i)
    x, w = _code(g, n, i), _code(g, o, i)
    xs, ws = torch.rand(n, generator=g, device="cuda") / 64, torch.rand(o, generator=g, device="cuda") / 64 * i ** -0.5
    b, res = _randn(g, o, t=t, scale=0.3), _randn(g, n, o, t=t)
    _check_int8(ad, x, xs, w, ws, b, res, act, t)
    _check_int8(ad, x.contiguous(), xs, w.contiguous(), ws, None, None, act, t)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(40000, 64, 128), (20000, 136, 264), (9000, 520, 1000), (30001, 72, 72), (8000, 101, 333)])
def test_linear_int8_many_rows(ad, shape, t):
    n, i, o = shape
    g = _gen(n + o)
    x, w = _code(g, n, i), _code(g, o, i)
    xs, ws = torch.rand(n, generator=g, device="cuda") / 64, torch.rand(o, generator=g, device="cuda") / 64 * i ** -0.5
    b, res = _randn(g, o, t=t, scale=0.3), _randn(g, n, o, t=t)
    _check_int8(ad, x, xs, w, ws, b, res, "silu", t)
    _check_int8(ad, x, xs, w, ws, None, None, "none", t)
    _check_int8(ad, x, xs, w, ws, b, None, "gelu", t)


@pytest.mark.parametrize("shape", [(1, 2000, 50), (5, 2000, 50), (100, 1000, 100), (3000, 1040, 264)])
def test_linear_int8_sums_are_exact(ad, shape):
    """With scales of one, sums below 2^24 are the result."""
    n, i, o = shape
    g = _gen(i)
    x = torch.randint(-90, 91, (n, i), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-90, 91, (o, i), generator=g, device="cuda", dtype=torch.int8)
    y = ad.linear_int8(x, torch.ones(n, device="cuda"), w, torch.ones(o, device="cuda"))
    assert torch.equal(y.double(), x.double() @ w.double().t())


@pytest.mark.parametrize("n", [1, 8, 40, 300])
def test_linear_int8_longest_sums(ad, n):
    """The largest sums of the longest rows stay within 32 bits."""
    i, o = 131071, 24
    x, w = torch.full((n, i), -128, device="cuda", dtype=torch.int8), torch.full((o, i), -128, device="cuda", dtype=torch.int8)
    w[1] = 127
    y = ad.linear_int8(x, torch.ones(n, device="cuda"), w, torch.ones(o, device="cuda"))
    assert (y[:, 0] == float(torch.tensor(128 * 128 * i).float())).all()
    assert (y[:, 1] == float(torch.tensor(-128 * 127 * i).float())).all()


@pytest.mark.parametrize("n", [2, 50, 5000])
def test_linear_int8_strides_and_alignment(ad, n):
    g = _gen(n)
    x, w = _code(g, n, 300), _code(g, 90, 300)
    xs, ws = torch.rand(n, generator=g, device="cuda"), torch.rand(90, generator=g, device="cuda")
    for lead in (0, 1, 16, 37):
        a, b = x[:, lead:lead + 200], w[:, lead:lead + 200]
        y = ad.linear_int8(a, xs, b, ws)
        assert torch.equal(y, ad.linear_int8(a.contiguous(), xs, b.contiguous(), ws))
    res = _randn(g, n, 100)[:, 3:93]
    assert torch.equal(ad.linear_int8(x, xs, w, ws, residual=res), ad.linear_int8(x, xs, w, ws, residual=res.contiguous()))
    off = torch.cat([ws[:1], ws])[1:]  # scales off 16 bytes
    assert torch.equal(ad.linear_int8(x, xs, w, off), ad.linear_int8(x, xs, w, ws))


@pytest.mark.parametrize("n", [3, 60, 6000])
def test_linear_int8_of_quantised_rows(ad, n):
    """A row that held a NaN is NaN, a row of zeros is the bias; the others within what
    half a code of either operand makes."""
    g = _gen(n)
    x, w = _randn(g, n, 100, t="bf16"), _randn(g, 48, 100, scale=0.1)
    x[0, 7] = math.nan
    x[1] = 0
    b = _randn(g, 48, t="bf16")
    (xq, xs), (wq, ws) = ad.quantize_rows(x), ad.quantize_rows(w)
    y = ad.linear_int8(xq, xs, wq, ws, b, dtype=torch.bfloat16)
    assert y[0].isnan().all() and torch.equal(y[1], b)
    x, xs = x[2:].double(), xs[2:].double()[:, None]
    ref = x @ w.double().t() + b.double()
    tol = (0.5 * xs) * (w.double().abs().sum(1)) + (x.abs() + 0.5 * xs).sum(1, keepdim=True) * (0.5 * ws.double())
    _within(y[2:], ref, 1.001 * tol + U["bf16"] * (ref.abs() + tol) + 1e-6, "y")


def test_linear_int8_beyond_32_bit_offsets(ad):
    n, i, o = 2_200_000, 32, 1000
    g = _gen(4)
    x = torch.ones(n, i, device="cuda", dtype=torch.int8)
    x[:300] = _code(g, 300, i)
    x[-300:] = x[:300]
    xs, w, ws = torch.ones(n, device="cuda"), _code(g, o, i), torch.rand(o, generator=g, device="cuda")
    y = ad.linear_int8(x, xs, w, ws, dtype=torch.float16)
    small = ad.linear_int8(x[:300], xs[:300], w, ws, dtype=torch.float16)
    assert torch.equal(y[:300], small) and torch.equal(y[-300:], small)


def _framed(rows, cols, t, lead=3, tail=5, above=2):
    """A matrix within a larger one of a value that no result takes, and the larger one."""
    frame = torch.full((rows + 2 * above, lead + cols + tail), 77.0, device="cuda").to(t)
    return frame[above:above + rows, lead:lead + cols], frame


def _frame_stayed(frame, view):
    clean = frame.clone()
    off = (view.data_ptr() - frame.data_ptr()) // frame.element_size()
    r, c = off // frame.shape[1], off % frame.shape[1]
    clean[r:r + view.shape[0], c:c + view.shape[1]] = 77
    return bool((clean == 77).all())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 9, 130, 700, 20000])
@pytest.mark.parametrize("i,o", [(33, 17), (40, 1), (64, 130), (72, 200), (16, 66)])
def test_results_stay_within_their_matrices(ad, n, i, o, t):
    """Through the C ABI, into the middle of larger matrices: what lies around the results
    is left as it was, and they are the values of the Python call."""
    import ctypes as C

    from fusiongpu_b200 import _lib
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    ws = torch.empty(1 << 27, dtype=torch.uint8, device="cuda")
    g = _gen(n + o)
    x, w, b = _randn(g, n, i, t=t), _randn(g, 2 * o, i, t=t, scale=0.2), _randn(g, 2 * o, t=t)
    for lead in (3, 8):
        y, fy = _framed(n, o, T[t], lead)
        pre, fp = _framed(n, 2 * o, T[t], lead)
        p = _lib.LinearParams(n, i, o, ad.DTYPES[T[t]], 3, 0, 0, 0, pre.stride(0), y.stride(0), 0)
        _lib.check(L.fg_gated_linear(C.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), pre.data_ptr(), y.data_ptr(),
                                     ws.data_ptr(), ws.numel(), s), "fg_gated_linear")
        ry, rp = ad.gated_linear(x, w, b, return_pre=True)
        assert torch.equal(y, ry) and torch.equal(pre, rp)
        assert _frame_stayed(fy, y) and _frame_stayed(fp, pre)
        q, xs = ad.quantize_rows(x)
        wq, wsc = ad.quantize_rows(w)
        y, fy = _framed(n, 2 * o, T[t], lead)
        p = _lib.LinearParams(n, i, 2 * o, ad.DTYPES[T[t]], 2, q.stride(0), wq.stride(0), 0, 0, y.stride(0), 0)
        _lib.check(L.fg_linear_int8(C.byref(p), q.data_ptr(), xs.data_ptr(), wq.data_ptr(), wsc.data_ptr(), b.data_ptr(), None,
                                    y.data_ptr(), ws.data_ptr(), ws.numel(), s), "fg_linear_int8")
        assert torch.equal(y, ad.linear_int8(q, xs, wq, wsc, b, activation="gelu", dtype=T[t])) and _frame_stayed(fy, y)
        codes, fc = _framed(n, i, torch.int8, lead)
        scale, fs = _framed(1, n, torch.float32, lead)
        _lib.check(L.fg_quantize_rows(x.data_ptr(), ad.DTYPES[T[t]], n, i, 0, codes.data_ptr(), codes.stride(0),
                                      scale.data_ptr(), s), "fg_quantize_rows")
        assert torch.equal(codes, q) and torch.equal(scale[0], xs) and _frame_stayed(fc, codes) and _frame_stayed(fs, scale)
    dy = _randn(g, n, o, t=t)
    want = ad.gated_linear_backward(dy, x, w, rp)
    frames = [_framed(1, v.numel(), T[t]) for v in want]
    p = _lib.LinearParams(n, i, o, ad.DTYPES[T[t]], 3, 0, 0, 0, 0, 0, 7)
    off = [v.data_ptr() for v, _ in frames]
    _lib.check(L.fg_gated_linear_backward(C.byref(p), dy.data_ptr(), x.data_ptr(), w.data_ptr(), rp.data_ptr(), *off,
                                          ws.data_ptr(), ws.numel(), s), "fg_gated_linear_backward")
    for (v, f), r in zip(frames, want):
        assert torch.equal(v.view(r.shape), r) and _frame_stayed(f, v)


def test_refusals(ad):
    x, w = torch.zeros(4, 32, device="cuda"), torch.zeros(20, 32, device="cuda")
    with pytest.raises(ValueError):
        ad.gated_linear(x, w[:19])  # an odd number of rows
    with pytest.raises(ValueError):
        ad.gated_linear(x, w[:, :31])
    with pytest.raises(ValueError):
        ad.gated_linear(x, w, torch.zeros(10, device="cuda"))
    with pytest.raises(ValueError):
        ad.gated_linear(x, w, activation="tanh")
    with pytest.raises(TypeError):
        ad.gated_linear(x, w.half())
    with pytest.raises(ValueError):
        ad.gated_linear_backward(torch.zeros(4, 10, device="cuda"), x, w, None)
    with pytest.raises(ValueError):
        ad.gated_linear_backward(torch.zeros(4, 10, device="cuda"), x, w, torch.zeros(4, 10, device="cuda"))
    q, s = ad.quantize_rows(x)
    wq, wsc = ad.quantize_rows(w)
    with pytest.raises(TypeError):
        ad.quantize_rows(q)
    with pytest.raises(TypeError):
        ad.linear_int8(x, s, wq, wsc)
    with pytest.raises(ValueError):
        ad.linear_int8(q[:, :31], s, wq, wsc)
    with pytest.raises(ValueError):
        ad.linear_int8(q, s[:3], wq, wsc)
    with pytest.raises(TypeError):
        ad.linear_int8(q, s.double(), wq, wsc)
    with pytest.raises(ValueError):
        ad.linear_int8(q, None, wq, wsc)
    with pytest.raises(TypeError):
        ad.linear_int8(q, s, wq, wsc, dtype=torch.int8)
    with pytest.raises(TypeError):
        ad.linear_int8(q, s, wq, wsc, torch.zeros(20, device="cuda"), dtype=torch.float16)
    from fusiongpu_b200._lib import FgError
    long = torch.zeros(1, 131072, device="cuda", dtype=torch.int8)
    with pytest.raises(FgError):
        ad.linear_int8(long, s[:1], long, s[:1])
    with pytest.raises(FgError):
        ad.gated_linear(torch.zeros(1, 32769, device="cuda"), torch.zeros(2, 32769, device="cuda"))
