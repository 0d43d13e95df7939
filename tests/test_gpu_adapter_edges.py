"""GPU tests of the query adapter's operators where they can lose what the
definition keeps: gradients of 16-bit layers, the activations' tails, values that
are not finite, operands off 16-byte boundaries, pairs that no query holds.

Tolerances follow from the arithmetic as in test_gpu_adapter.py, whose helpers
are used: U[t] is the unit roundoff of a result's type, E32 that of 32-bit sums.
"""
import math

import pytest
import torch

from tests.test_gpu_adapter import E32, T, TINY, U, _act, _act_grad, _check_backward, _check_linear, _gen, _randn, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ad():
    from fusiongpu_b200 import adapter
    return adapter


# ---- dz of 16-bit layers of more than eight rows ---------------------------------------
#
# dz = dy act'(pre) goes to the tensor cores in two parts of the type: together they are
# off by the product of two unit roundoffs (2^-18 bf16, 2^-24 f16), doubled here, and in
# float16 by half the lower part's last place, 2^-36.  The derivative's own error is
# SLOPE: 2^-22 of the fit and a few operations in 32 bits, or of __expf.

PARTS = {"f16": 2.0 ** -23, "bf16": 2.0 ** -17}
FLOOR = {"f16": 2.0 ** -36, "bf16": 0.0}
SLOPE = 2.0 ** -19


def _check_dz(ad, dy, x, w, pre, act, t):
    dx, dw, db = ad.linear_backward(dy, x, w, pre=pre, activation=act)
    d = dy.double()
    dz = d * _act_grad(pre.double(), act)
    edz = SLOPE * d.abs() + PARTS[t] * dz.abs() + FLOOR[t]
    n, o = d.shape
    for got, want, err, k, mag in (
            (dx, dz @ w.double(), edz @ w.double().abs(), o, dz.abs() @ w.double().abs()),
            (dw, dz.t() @ x.double(), edz.t() @ x.double().abs(), n, dz.abs().t() @ x.double().abs()),
            (db, dz.sum(0), SLOPE * d.abs().sum(0), n, dz.abs().sum(0))):
        _within(got, want, err + (k + 8) * 2 * E32 * mag + U[t] * want.abs() + TINY[t], f"{tuple(got.shape)}")
    return dx, dw, db


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("shape", [(9, 56, 107), (40, 264, 520), (300, 768, 1536), (3000, 136, 264), (10000, 768, 1536),
                                   (20001, 72, 1000), (40000, 520, 72)])
def test_gradients_have_one_rounding(ad, shape, act, t):
    n, i, o = shape
    g = _gen(n + i)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, o, t=t, scale=1.5)
    got = _check_dz(ad, dy, x, w, pre, act, t)
    for u, v in zip(got, ad.linear_backward(dy, x, w, pre=pre, activation=act)):
        assert torch.equal(u, v)
    k = slice(0, 8)  # eight rows have a kernel of their own: the same values to 32 bits
    _check_dz(ad, dy[k], x[k], w, pre[k], act, t)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("shape", [(16, 40, 72), (4000, 136, 264)])
def test_float16_gradients_below_and_above_its_range(ad, shape, act):
    """Terms of dz too small for float16 whose sum is not, and terms past its largest."""
    n, i, o = shape
    g = _gen(n)
    x, w = _randn(g, n, i, t="f16").abs() + 0.5, _randn(g, o, i, t="f16").abs() + 0.5
    dy = (torch.rand(n, o, generator=g, device="cuda") + 0.5).mul(1e-6).half()
    pre = (-3.5 - torch.rand(n, o, generator=g, device="cuda")).half()
    d, p = dy.double(), pre.double()
    dx, dw, _ = ad.linear_backward(dy, x, w, pre=pre, activation=act)
    dz = d * _act_grad(p, act)
    edz = 2.0 ** -15 * dz.abs() + FLOOR["f16"]  # this far out the derivative is right to 2^-16 of itself
    assert dz.abs().mean() < 2.0 ** -23 and dz.abs().max() > 2.0 ** -34
    for got, want, err in ((dx, dz @ w.double(), edz @ w.double()), (dw, dz.t() @ x.double(), edz.t() @ x.double())):
        _within(got, want, err + U["f16"] * want.abs() + TINY["f16"], "small")
    if n > 1000:
        assert (dw != 0).all()
    dy = torch.full((n, o), 62000.0, device="cuda", dtype=torch.float16)
    pre = torch.full((n, o), 1.40625 if act == "gelu" else 2.40625, device="cuda", dtype=torch.float16)
    dz = dy.double() * _act_grad(pre.double(), act)
    assert (dz > 65520).all()
    x, w = torch.full_like(x, 2.0 ** -7 / n), torch.full_like(w, 2.0 ** -10)
    dx, dw, _ = ad.linear_backward(dy, x, w, pre=pre, activation=act)
    edz = 2.0 ** -18 * dz
    for got, want, err in ((dx, dz @ w.double(), edz @ w.double()), (dw, dz.t() @ x.double(), edz.t() @ x.double())):
        _within(got, want, err + (n + o) * 2 * E32 * want + U["f16"] * want, "large")


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(30, 72, 40), (3000, 264, 520), (30000, 136, 264)])
def test_gradients_with_infinite_operands(ad, shape, t):
    """An infinite weight or input times any dz but 0 is infinite, whatever parts dz has."""
    n, i, o = shape
    g = _gen(i)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t)
    dy, pre = _randn(g, n, o, t=t), _randn(g, n, o, t=t)
    dy[:, o // 2] = torch.where(dy[:, o // 2] == 0, 1.0, dy[:, o // 2])
    w[o // 2, 5] = math.inf
    x[n // 2, 3] = -math.inf
    dy[n // 2] = 0.5
    pre[n // 2] = 1.0
    dz = dy.double() * _act_grad(pre.double(), "gelu")
    dx, dw, db = ad.linear_backward(dy, x, w, pre=pre, activation="gelu")
    assert torch.equal(dx[:, 5].double(), torch.sign(dz[:, o // 2]) * math.inf)
    assert torch.equal(dw[:, 3].double(), torch.full_like(dz[0], -math.inf))
    dx[:, 5] = dw[:, 3] = 0
    assert dx.isfinite().all() and dw.isfinite().all() and db.isfinite().all()
    dy[1, 2] = math.nan  # poison reaches what depends on it
    dx, dw, db = ad.linear_backward(dy, x, w, pre=pre, activation="gelu")
    assert dx[1].isnan().all() and dw[2].isnan().all() and db[2].isnan()
    keep = torch.arange(n, device="cuda") != 1
    assert not dx[keep].isnan().any() and not dw[torch.arange(o, device="cuda") != 2].isnan().any()


# ---- buffers handed from ordinary accesses to copies ---------------------------------------

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(40000, 64, 128), (20000, 136, 264), (9000, 520, 1000)])
def test_residual_with_and_without_the_pre_activation(ad, shape, t):
    """The residual comes through the buffer that held the sums: the same result whether
    or not the pre-activation left through it in between."""
    n, i, o = shape
    g = _gen(o)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    b, res = _randn(g, o, t=t), _randn(g, n, o, t=t)
    for act in ("none", "silu"):
        want = ad.linear(x, w, b, activation=act, residual=res, return_pre=True)[0]
        for _ in range(5):
            assert torch.equal(ad.linear(x, w, b, activation=act, residual=res), want)


# ---- float32 sums that are not finite -------------------------------------------------------

@pytest.mark.parametrize("shape,lead", [((9, 40, 72), 0), ((5000, 520, 264), 0), ((5000, 520, 264), 1), ((20000, 72, 1000), 0),
                                        ((300, 20000, 520), 0)])
def test_float32_sums_past_its_largest(ad, shape, lead):
    """Every sum of whole tiles overflows: infinities of the right sign where all products
    have one, the other rows and columns as without them."""
    n, i, o = shape
    g = _gen(i)
    x, w = _randn(g, n, i), _randn(g, o, i, scale=i ** -0.5)
    b, res = _randn(g, o), _randn(g, n, o + 4)[:, lead:lead + o]
    rows, cols = torch.arange(n, device="cuda") % 3 == 0, torch.arange(o, device="cuda") % 5 == 0
    xl, wl = x.clone(), w.clone()
    xl[rows], wl[cols] = -2e20, 3e20
    y, pre = ad.linear(xl, wl, b, activation="silu", residual=res, return_pre=True)
    big = rows[:, None] & cols
    assert (pre[big] == -math.inf).all() and torch.equal(y[big], res.expand(n, o)[big])  # silu(-inf) = 0
    want, wpre = ad.linear(x, w, b, activation="silu", residual=res, return_pre=True)
    small = ~rows[:, None] & ~cols
    assert torch.equal(pre[small], wpre[small]) and torch.equal(y[small], want[small])
    plain = ad.linear(xl, wl)
    assert (plain[big] == -math.inf).all()
    assert torch.equal(plain[small], ad.linear(x, w)[small])
    xl[1::3, 0] = math.nan  # rows that are not all one sign
    y = ad.linear(xl, wl, residual=res)
    assert (y[big] == -math.inf).all() and y[1::3].isnan().all() and not y[rows].isnan().any()


def test_float32_gradients_past_its_largest(ad):
    """The same where the sums run over many rows, split and not."""
    for n, i, o in ((3000, 264, 520), (60000, 136, 264), (30000, 2000, 2100)):
        g = _gen(n)
        x, w = _randn(g, n, i).abs() + 0.5, _randn(g, o, i)
        dy = _randn(g, n, o)
        x[:, 3], dy[:, 5] = 1e25, -1e25
        dx, dw, db = ad.linear_backward(dy, x, w, param_grads=True)
        assert dw[5, 3] == -math.inf
        assert dw[5, 4:].isfinite().all() and dx.isfinite().all() and db.isfinite().all()
        dy[n // 2, 7] = math.inf
        dx, dw, db = ad.linear_backward(dy, x, w)
        assert (dw[7] == math.inf).all() and db[7] == math.inf
        assert torch.equal(dx[n // 2], torch.sign(w[7]) * math.inf)
        keep = torch.arange(o, device="cuda") != 7
        assert not dw[keep].isnan().any() and dw[keep][:, 8:].isfinite().all()


# ---- the tails of the activations ---------------------------------------------------------

@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_tails_keep_their_relative_accuracy(ad, act, t):
    """Results of 16 bits: within their own rounding and 2^-15 of the value (2^-11 below
    -6, where only bfloat16 has anything to show), not of one."""
    z = torch.cat([torch.linspace(-13, -2, 4001), torch.linspace(-2, 6, 2001)]).cuda().to(T[t])[:, None]
    one = torch.ones(1, 1, device="cuda", dtype=T[t])
    zd = z.double()
    phi = 0.5 * torch.special.erfc(-zd * math.sqrt(0.5))  # torch's ndtr is (1 + erf) / 2: 0 below -8.3
    want = zd * phi if act == "gelu" else zd * torch.sigmoid(zd)
    rel = torch.where(zd < -6, 2.0 ** -11, 2.0 ** -15)
    tol = (U[t] + rel) * want.abs() + TINY[t]
    _within(ad.linear(z, one, activation=act), want, tol, "y")
    _within(ad.linear(z[1000:1003], one, activation=act), want[1000:1003], tol[1000:1003], "y of three rows")
    d = ad.linear_backward(torch.ones_like(z), z, one, pre=z, activation=act, param_grads=False)[0]
    want = phi + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi) if act == "gelu" else _act_grad(zd, act)
    near = 2.0 ** -19 * (zd > -2.5)  # the derivative passes through 0 there
    _within(d, want, (U[t] + 2.0 ** -15) * want.abs() + near + TINY[t], "derivative")


# ---- sums over very many rows ---------------------------------------------------------------

def _ms(f, n=5):
    f()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(n):
        f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / n


def test_weight_gradient_of_very_many_rows(ad):
    """262,200 rows, just past a count whose sums fit one number of parts: still cut into
    parts, right to 64 bits and no slower than its share."""
    n, i, o = 262200, 768, 1536
    g = _gen(1)
    x, dy = _randn(g, n, i, t="bf16"), _randn(g, n, o, t="bf16")
    w = _randn(g, o, i, t="bf16")
    _, dw, db = ad.linear_backward(dy, x, w, input_grad=False)
    want = torch.zeros(o, i, dtype=torch.float64, device="cuda")
    for a, b in zip(dy.split(32768), x.split(32768)):
        want += a.double().t() @ b.double()
    # 4,097 blocks of 64 k in parts of 512 at most: 2^-24 of the running value (about the
    # sum's size) for each of 2,048 additions of 16 products, all cut to one side at worst
    _within(dw, want, 2048 * 2 * E32 * want.abs().max() + U["bf16"] * want.abs(), "dw")
    _within(db, dy.double().sum(0), (n + 16) * 2 * E32 * dy.double().abs().sum(0), "dbias")
    k = slice(0, 262144)
    here, there = (_ms(lambda s=s: ad.linear_backward(dy[s], x[s], w, input_grad=False)) for s in (slice(0, n), k))
    assert here < 2.5 * there, (here, there)  # unsplit it was 4.3 times


# ---- operands that do not start on 16-byte boundaries -------------------------------------

def _off(m, lead):
    """The same matrix, rows a multiple of 16 bytes apart, `lead` elements off a boundary."""
    n, d = m.shape
    big = torch.zeros(n, (d + lead + 15) // 8 * 8, device="cuda", dtype=m.dtype)
    v = big[:, lead:lead + d]
    v.copy_(m)
    assert v.stride(0) % 8 == 0 and v.data_ptr() % 16 == lead * m.element_size()
    return v


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(9, 40, 24), (100, 264, 136), (3000, 136, 520), (5001, 768, 264)])
def test_operands_off_16_bytes(ad, shape, t):
    n, i, o = shape
    g = _gen(n + o)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t), _randn(g, n, o, t=t)
    for lead in (1, 4):
        for xo, wo, do in ((_off(x, lead), w, dy), (x, _off(w, lead), dy), (_off(x, lead), _off(w, lead), _off(dy, lead))):
            _check_linear(ad, xo, wo, None, pre, "silu", t)
            for act in ("none", "gelu"):
                want = ad.linear_backward(dy, x, w, pre=pre, activation=act)
                for u, v in zip(ad.linear_backward(do, xo, wo, pre=_off(pre, lead), activation=act), want):
                    assert torch.equal(u, v)
                _check_backward(ad, do, xo, wo, _off(pre, lead), act, t)
            assert torch.equal(ad.linear(xo, wo, activation="gelu"), ad.linear(x, w, activation="gelu"))


def test_operands_off_16_bytes_stay_on_the_tensor_cores(ad):
    """Packing costs a pass over memory, not the FP32 units' twenty to forty times."""
    g = _gen(1)
    x, w, dy = _randn(g, 10000, 768, t="f16"), _randn(g, 1536, 768, t="f16"), _randn(g, 10000, 1536, t="f16")
    xo, wo, do = _off(x, 4), _off(w, 1), _off(dy, 1)
    here, there = _ms(lambda: ad.linear(x, w)), _ms(lambda: ad.linear(xo, wo))
    assert there < 5 * here, (here, there)
    here, there = _ms(lambda: ad.linear_backward(dy, x, w)), _ms(lambda: ad.linear_backward(do, xo, wo))
    assert there < 5 * here, (here, there)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_operands_off_16_bytes_that_are_not_named(ad, t):
    """Through the C ABI without the `unaligned` bits: the same values to their rounding,
    from the CUDA cores."""
    import ctypes as C

    from fusiongpu_b200 import _lib
    n, i, o = 150, 136, 72
    g = _gen(6)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, o, t=t)
    xo, wo = _off(x, 1), _off(w, 1)
    s = torch.cuda.current_stream().cuda_stream

    def call(name, off, *args):
        p = _lib.LinearParams(n, i, o, ad.DTYPES[T[t]], 2, xo.stride(0), wo.stride(0), 0, 0, 0, off)
        ws = torch.empty(_lib.size_query(name + "_workspace_size", C.byref(p)), dtype=torch.uint8, device="cuda")
        _lib.check(getattr(_lib.lib(), name)(C.byref(p), *args, ws.data_ptr(), ws.numel(), s), name)

    ys, dxs, dws = [], [], []
    for off in (0, 3):
        y, dx, dw = torch.full_like(dy, math.nan), torch.full_like(x, math.nan), torch.full_like(w, math.nan)
        call("fg_linear", off, xo.data_ptr(), wo.data_ptr(), None, None, None, y.data_ptr())
        call("fg_linear_backward", off, dy.data_ptr(), xo.data_ptr(), wo.data_ptr(), pre.data_ptr(), dx.data_ptr(),
             dw.data_ptr(), None)
        ys.append(y), dxs.append(dx), dws.append(dw)
    z = x.double() @ w.double().t()
    zm = x.double().abs() @ w.double().abs().t()
    dz = dy.double() * _act_grad(pre.double(), "gelu")
    for got, want, mag, k in ((ys, _act(z, "gelu"), 1.2 * zm, i), (dxs, dz @ w.double(), dy.double().abs() @ w.double().abs(), o),
                              (dws, dz.t() @ x.double(), dy.double().abs().t() @ x.double().abs(), n)):
        for v in got:  # 2^-15: the activation and its derivative
            _within(v, want, ((k + 8) * 2 * E32 + 2.0 ** -15) * mag + U[t] * want.abs() + TINY[t], str(tuple(v.shape)))


# ---- preference loss ------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 256])
def test_preference_infinite_margins(ad, dim):
    """A margin of either infinity under label smoothing: the loss is infinite, not NaN."""
    base = torch.zeros(2, dim, device="cuda")
    base[1] = 1e38
    q = torch.full((2, dim), 1e38, device="cuda")
    off = torch.tensor([0, 1, 2], device="cuda")
    pos = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    neg = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for e, first in ((0.0, 0.0), (0.1, math.inf)):
        losses, margins, _ = ad.preference_loss(q, base, off, pos, neg, label_smoothing=e)
        assert margins.tolist() == [math.inf, -math.inf]
        assert losses.tolist() == [first, math.inf]


def _poison(*sizes):
    """Leaves NaN in the memory that the next allocations of these sizes get."""
    for t in [torch.full((n,), math.nan, device="cuda") for n in sizes]:
        del t


@pytest.mark.parametrize("dim", [96, 512])
def test_preference_pairs_outside_the_offsets(ad, dim):
    """Pairs that no query holds: loss and margin 0, as for masked ones."""
    g = _gen(dim)
    base, q = _randn(g, 50, dim), _randn(g, 3, dim)
    pos = torch.randint(0, 50, (1000,), generator=g, device="cuda", dtype=torch.int32)
    neg = torch.randint(0, 50, (1000,), generator=g, device="cuda", dtype=torch.int32)
    for off in ([300, 310, 310, 700], [0, 0, 5, 5], [990, 1000, 1000, 1000], [1000] * 4):
        _poison(1000, 1000)
        o = torch.tensor(off, device="cuda")
        losses, margins, dq = ad.preference_loss(q, base, o, pos, neg, beta=0.1)
        a, b = off[0], off[-1]
        assert not losses[:a].any() and not losses[b:].any() and not margins[:a].any() and not margins[b:].any()
        held = ad.preference_loss(q, base, o - a, pos[a:b], neg[a:b], beta=0.1)
        assert torch.equal(losses[a:b], held[0]) and torch.equal(margins[a:b], held[1]) and torch.equal(dq, held[2])
    _poison(1000, 1000)
    losses, margins, dq = ad.preference_loss(q[:0], base, torch.zeros(1, dtype=torch.int64, device="cuda"), pos, neg)
    assert dq.shape == (0, dim) and not losses.any() and not margins.any()


def test_operators_by_keyword(ad):
    g = _gen(2)
    x, w, dy = _randn(g, 40, 64), _randn(g, 24, 64), _randn(g, 40, 24)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y, mean, rstd = ad.layer_norm(x, return_stats=True)
    for kw in ({}, {"stream": s}):
        for got, want in ((ad.layer_norm(x=x, **kw), y), (ad.linear(x=x, w=w, **kw), ad.linear(x, w)),
                          (ad.linear_backward(dy=dy, x=x, w=w, **kw), ad.linear_backward(dy, x, w)),
                          (ad.layer_norm_backward(dy=x, x=x, mean=mean, rstd=rstd, **kw), ad.layer_norm_backward(x, x, mean, rstd))):
            s.synchronize()
            for u, v in zip(got, want):
                assert torch.equal(u, v)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 40, 2560), (4, 72, 2561), (4, 33, 5121), (8, 40, 1537), (5, 136, 3200), (8, 4000, 1100)])
def test_gradients_of_few_rows_of_wide_layers(ad, shape, t):
    """On both sides of the widths from which the products of more rows take them."""
    n, i, o = shape
    g = _gen(o)
    x, w = _randn(g, n, i, t=t), _randn(g, o, i, t=t, scale=i ** -0.5)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, o, t=t, scale=1.5)
    for act in ("gelu", "silu"):
        if t != "f32":
            _check_dz(ad, dy, x, w, pre, act, t)
        _check_backward(ad, dy, x, w, pre, act, t)


# ---- layer norm: the parameters' gradients alone ----------------------------------------------

@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("dim", [40, 301, 768, 1536, 5000])
def test_layer_norm_parameter_gradients_alone(ad, t, dim):
    """Through the C ABI without dx, and without one of the two sums: the same bits."""
    from fusiongpu_b200 import _lib
    g = _gen(dim)
    x, dy, w = _randn(g, 700, dim, t=t), _randn(g, 700, dim, t=t), _randn(g, dim)
    _, mean, rstd = ad.layer_norm(x, w, return_stats=True)
    _, dw, db = ad.layer_norm_backward(dy, x, mean, rstd, w)
    ws = torch.empty(_lib.size_query("fg_layer_norm_backward_workspace_size", 700, dim), dtype=torch.uint8, device="cuda")
    for want_w, want_b in ((1, 1), (1, 0), (0, 1)):
        gw, gb = torch.full_like(dw, math.nan), torch.full_like(db, math.nan)
        _lib.check(_lib.lib().fg_layer_norm_backward(
            dy.data_ptr(), 0, x.data_ptr(), ad.DTYPES[T[t]], 700, dim, 0, w.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(),
            None, 0, gw.data_ptr() if want_w else None, gb.data_ptr() if want_b else None, ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream().cuda_stream), "fg_layer_norm_backward")
        assert torch.equal(gw, dw) if want_w else gw.isnan().all()
        assert torch.equal(gb, db) if want_b else gb.isnan().all()
