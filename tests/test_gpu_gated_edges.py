"""GPU tests of the gated adapter's operators at the ends of their ranges, against plain
implementations in 64 bits.

Tolerances are those of the operators' own tests: U[t] the unit roundoff of a result's
type, E32 = 2^-24 that of 32-bit sums, (n + 8) * 2 * E32 of the magnitudes for a sum of n
products, ACT for the activation functions.  A gradient of a pre-activation that passes
float16's range enters the products with 2^-21 of it (20 bits behind the leading one,
rounded), any other with PART of it.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
ACT = {"f32": 2.0 ** -20, "f16": 2.0 ** -18, "bf16": 2.0 ** -18}
PART = {"f32": 2.0 ** -23, "f16": 2.0 ** -21, "bf16": 2.0 ** -16}
LOW = {"f32": 2.0 ** -130, "f16": 2.0 ** -36, "bf16": 2.0 ** -130}
E32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ad():
    from fusiongpu_b200 import adapter
    return adapter


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, t="f32", scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(T[t])


def _within(got, want, tol, t, what):
    """A value past the type's range is infinite in it, as its rounding is."""
    round_ = want.to(T[t]).double()
    past = round_.isinf()
    assert torch.equal(got.double()[past], round_[past]), what
    bad = ~((got.double() - want).abs() <= tol) & ~past
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float(((got.double() - want).abs() / tol)[bad].max()):.3g} x tolerance"


def _backward(dy, x, w, pre, act):
    """The gradients and what their operands' and sums' errors make of them at most, but
    for the results' rounding."""
    h = dy.shape[1]
    d, z, p = dy.double(), pre[:, :h].double(), pre[:, h:].double()
    s = torch.sigmoid(z)
    f, a = {"none": lambda: (torch.ones_like(z), z), "silu": lambda: (s * (1 + z * (1 - s)), z * s),
            "gelu": lambda: (torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), z * torch.special.ndtr(z))}[act]()
    return torch.cat([d * p * f, d * a], 1), torch.cat([(d * p).abs(), d.abs() * z.abs().clamp(min=1)], 1)


def _check_backward(ad, dy, x, w, pre, act, t):
    dx, dw, db = ad.gated_linear_backward(dy, x, w, pre, activation=act)
    dz, mag = _backward(dy, x, w, pre, act)
    edz = (ACT[t] * mag if act != "none" else 0) + 4 * E32 * dz.abs()
    part = edz + PART[t] * dz.abs() + LOW[t]
    n, k = dz.shape
    rdx, rdw, rdb = dz @ w.double(), dz.t() @ x.double(), dz.sum(0)
    _within(dx, rdx, part @ w.double().abs() + (k + 8) * 2 * E32 * (dz.abs() @ w.double().abs()) + U[t] * rdx.abs() + TINY[t], t, "dx")
    _within(dw, rdw, part.t() @ x.double().abs() + (n + 8) * 2 * E32 * (dz.abs().t() @ x.double().abs()) + U[t] * rdw.abs()
            + TINY[t], t, "dw")
    _within(db, rdb, edz.sum(0) + (n + 8) * 2 * E32 * dz.abs().sum(0) + U[t] * rdb.abs() + TINY[t], t, "dbias")
    return dx, dw, db


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("n,i,o", [(2, 40, 24), (8, 64, 900), (40, 72, 48), (300, 64, 130), (3000, 264, 333), (20000, 128, 256)])
def test_gated_backward_past_the_range_of_its_type(ad, n, i, o, t, act):
    """dz = dy p act'(z) and dp = dy act(z) of values that float16 holds may lie past its
    range while the gradients do not."""
    g = _gen(n + o)
    x, w = _randn(g, n, i, t=t, scale=2.0 ** -8), _randn(g, 2 * o, i, t=t, scale=2.0 ** -9)
    dy, pre = _randn(g, n, o, t=t, scale=0.1), _randn(g, n, 2 * o, t=t, scale=1.5)
    rows = torch.randint(0, n, (6,), generator=g, device="cuda")
    cols = torch.randint(0, o, (6,), generator=g, device="cuda")
    dy[rows, cols] = torch.tensor([3000, -3000, 50000, 1312, -400, 1310], device="cuda").to(T[t])
    pre[rows, cols] = torch.tensor([2, 1.5, 300, 30, 1000, 100], device="cuda").to(T[t])
    pre[rows, o + cols] = torch.tensor([100, 200, -80, 100, 1000, -100], device="cuda").to(T[t])
    _check_backward(ad, dy, x, w, pre, act, t)  # the largest, of 50000 * 300 * 2^-9 and more, may round to an infinity


@pytest.mark.parametrize("n", [5, 60, 5000])
def test_gated_backward_of_the_largest_values(ad, n):
    """float16's largest dy and p: dz of 2^32."""
    top = 65504.0
    x = torch.zeros(n, 40, device="cuda", dtype=torch.float16)
    w = torch.zeros(64, 40, device="cuda", dtype=torch.float16)
    dy, pre = torch.zeros(n, 32, device="cuda", dtype=torch.float16), torch.zeros(n, 64, device="cuda", dtype=torch.float16)
    dy[n // 2, 3], pre[n // 2, 3], pre[n // 2, 35] = -top, top, top
    x[n // 2, 7], w[3, 5], w[35, 6] = 2.0 ** -20, 2.0 ** -24, 3 * 2.0 ** -24
    dx, dw, _ = _check_backward(ad, dy, x, w, pre, "silu", "f16")
    assert abs(float(dx[n // 2, 5]) + top * top * 2.0 ** -24) <= 1 and abs(float(dx[n // 2, 6]) + 3 * top * top * 2.0 ** -24) <= 2
    assert int((dx != 0).sum()) == 2 and int((dw != 0).sum()) == 2


@pytest.mark.parametrize("n", [60, 5000])
def test_gated_backward_keeps_infinities_and_nan(ad, n):
    """A dy that is infinite or NaN, beside one whose dz passes the range."""
    g = _gen(n)
    x, w = _randn(g, n, 64, t="f16", scale=2.0 ** -8), _randn(g, 96, 64, t="f16", scale=2.0 ** -9)
    dy, pre = _randn(g, n, 48, t="f16"), _randn(g, n, 96, t="f16")
    pre[1, 48 + 4], dy[1, 4], pre[1, 4] = 1000, 1000, 3
    clean = ad.gated_linear_backward(dy, x, w, pre, activation="none", param_grads=False)[0]
    dy[2, 5], dy[3, 6] = math.nan, math.inf
    dx = ad.gated_linear_backward(dy, x, w, pre, activation="none", param_grads=False)[0]
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[2:4] = False
    assert dx[2].isnan().all() and torch.equal(dx[keep], clean[keep]) and clean.isfinite().all()
    dz, _ = _backward(dy[3:4], x, w, pre[3:4], "none")
    torch.testing.assert_close(dx[3].double(), dz[0, [6, 54]] @ w[[6, 54]].double(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_muon_keeps_a_small_decay(ad, dtype, monkeypatch):
    """The usual lr and a weight decay of 0.05 over a thousand steps without a gradient:
    each factor off by half a step, eps / 2, where at least 4 eps (or the step's decay, if
    that is eps or more) is taken at a time, and less than 4 eps held back."""
    eps, d, n = torch.finfo(dtype).eps, 0.02 * 0.05, 1000
    p = (torch.rand(50, 70, generator=_gen(3), device="cuda") + 0.5).to(dtype)
    start = p.double()
    p.grad = torch.zeros_like(p)
    opt = ad.Muon([p], lr=0.02, weight_decay=0.05)
    for _ in range(n):
        opt.step()
    want, due = n * math.log1p(-d), d if d >= eps else 4 * eps
    assert float((torch.log(p.double() / start) - want).abs().max()) <= 1.02 * eps / 2 / due * abs(want) + 4 * eps + d
    if d < eps:
        while 1 - opt.state[p].get("decay", 1.0) + d >= 4 * eps:  # off the step that takes it
            opt.step()
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()


def test_muon_refused_step_moves_nothing(ad):
    """What one parameter is refused for is found before another one moves."""
    here, there = torch.ones(4, 8, device="cuda"), torch.ones(4, 8)
    here.grad, there.grad = torch.ones_like(here), torch.ones_like(there)
    opt = ad.Muon([dict(params=[here]), dict(params=[there])], weight_decay=0.1)
    with pytest.raises(ValueError, match="GPU"):
        opt.step()
    assert (here == 1).all() and not opt.state[here]
    there.grad = None
    opt.step()
    assert (here != 1).all()


@pytest.mark.parametrize("n,o", [(2500, 2001), (2500, 2000), (700, 33)])
def test_linear_int8_of_long_rows(ad, n, o):
    """Sums past 65,536 codes are integers like any other: exact, and of the same tiles as
    shorter ones.  2^-22 of the result: the sum's rounding to 32 bits, those of the two
    products with the scales, and the result's."""
    i = 65552
    g = _gen(o)
    x, w = (torch.randint(-128, 128, (k, i), generator=g, device="cuda", dtype=torch.int8) for k in (n, o))
    xs, ws = (torch.rand(k, generator=g, device="cuda") + 0.5 for k in (n, o))
    y = ad.linear_int8(x, xs, w, ws)
    rows = torch.randint(0, n, (64,), generator=g, device="cuda")
    want = (x[rows].double() @ w.double().t()) * xs[rows].double()[:, None] * ws.double()
    assert bool(((y[rows].double() - want).abs() <= 2.0 ** -22 * want.abs()).all())


def _kernels(f):
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        f()
        torch.cuda.synchronize()
    return [e.key for e in prof.key_averages()]


@pytest.mark.parametrize("o", [2000, 2001])
def test_linear_int8_of_long_rows_takes_pairs(ad, o):
    """The kernel that takes rows of 65,536 codes takes longer ones too."""
    xs, ws = torch.ones(2500, device="cuda"), torch.ones(o, device="cuda")
    names = []
    for i in (65536, 65552):
        x, w = (torch.ones(k, i, device="cuda", dtype=torch.int8) for k in (2500, o))
        names.append([k.split("<")[0] for k in _kernels(lambda: ad.linear_int8(x, xs, w, ws)) if "gemm_" in k])
    if not names[0]:
        pytest.skip("no kernels recorded")
    assert names[0] == names[1]


def _us(f, n=20):
    for _ in range(3):
        f()
    best = math.inf
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / n)
    return best


@pytest.mark.parametrize("n,i,o", [(390, 5113, 620), (1882, 5504, 207), (6606, 5479, 54)])
def test_gated_deep_sums_take_no_longer_than_plain_ones(ad, n, i, o):
    """float32 layers of few tiles and long sums: the gated layer against the plain one of
    as many columns, the same products (1.0 to 1.1 times as long; 1.8 is allowed)."""
    g = _gen(n)
    x, w = _randn(g, n, i), _randn(g, 2 * o, i, scale=i ** -0.5)
    assert _us(lambda: ad.gated_linear(x, w)) <= 1.8 * _us(lambda: ad.linear(x, w))


@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (True, 0.1), (False, 0.01)])
@pytest.mark.parametrize("shape", [(60, 40), (30, 100), (300, 200)])
def test_muon_against_its_formula_in_64_bits(ad, shape, nesterov, decay):
    """Three float32 steps.  u is off by eight roundings at most of three times its own
    magnitude (three gradients, as large each), and the iteration multiplies what X is off
    by 3.4445, its largest slope, a step; the operator adds its own error (three standard
    deviations).  p is rounded twice a step."""
    from tests.test_gpu_orthogonalize import _iterate
    g = _gen(shape[0])
    p = _randn(g, *shape)
    want, m, off = p.double(), torch.zeros_like(p).double(), 0.0
    opt = ad.Muon([p], lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    scale = 0.05 * math.sqrt(max(1.0, shape[0] / shape[1]))
    for _ in range(3):
        p.grad = _randn(g, *shape)
        opt.step()
        m = 0.9 * m + p.grad.double()
        o, err = _iterate(p.grad.double() + 0.9 * m if nesterov else m)
        want = (1 - 0.05 * decay) * want - scale * o
        off += scale * (3 * err + 3.4445 ** 5 * 24 * E32) + 2 * E32 * float(want.norm())
        assert float((p.double() - want).norm()) <= off
