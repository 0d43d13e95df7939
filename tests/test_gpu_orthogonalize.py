"""GPU tests of the orthogonalised update against the iteration in 64 bits.

Tolerances are on the Frobenius norm of the error and follow the iteration.  A
product of P and Q is off by ROUND for each of its terms, independently (two
operands' roundings to 22 bits and the product of their low planes, which is left
out), so by ROUND * sqrt(sum of the terms' squares), and by what 32-bit sums lose: 16 * 2^-24 of
the result for the cuts within runs of at most 128 k (twice what their eight additions make)
and 8 * 2^-24 for the runs' additions; a matrix kept between products adds 2^-22 of its norm.  An error of X grows in a step by
the largest slope of a s + b s^3 + c s^5 over the singular values, chords through
the origin among them.  Three times the sum of these is allowed, the terms being
standard deviations, and the rounding of the result to its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
COEF = (3.4445, -4.7750, 2.0315)
ROUND = 3 * 2.0 ** -22
KEPT = 2.0 ** -22


@pytest.fixture(scope="module")
def ad():
    from fusiongpu_b200 import adapter
    return adapter


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _iterate(g, steps=5, coef=COEF, eps=1e-7):
    """The result in 64 bits and the bound on a result's error (Frobenius)."""
    a, b, c = coef
    x = g.double()
    x = x / (x.square().sum().sqrt() + eps)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    err = KEPT * float(x.norm())

    def product(p, q):
        rms = float((p.square() @ q.square()).sum().sqrt())
        return ROUND * rms + 24 * 2.0 ** -24 * float((p @ q).norm())

    for _ in range(steps):
        gram = x @ x.t()
        poly = b * gram + c * gram @ gram
        top = float(torch.linalg.matrix_norm(x, ord=2))
        dg = product(x, x.t()) + KEPT * float(gram.norm())
        dp = abs(b) * dg + abs(c) * (2 * top ** 2 * dg + product(gram, gram)) + KEPT * float(poly.norm())
        new = a * x + poly @ x
        dx = top * dp + product(poly, x) + 2 * KEPT * float(new.norm())
        s = torch.linspace(0, top, 200, dtype=torch.float64)
        slope = float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max())
        err = max(slope, float((a + b * s ** 2 + c * s ** 4).abs().max())) * err + dx
        x = new
    return (x.t() if tall else x), err


def _check(ad, g, t, steps=5, coef=COEF, eps=1e-7):
    got = ad.orthogonalize(g, steps=steps, coefficients=coef, eps=eps)
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    for x, y in zip(g if g.dim() == 3 else [g], got if g.dim() == 3 else [got]):
        want, err = _iterate(x, steps, coef, eps)
        off = float((y.double() - want).norm())
        tol = 3 * err + U[t] * float(want.norm()) + 2.0 ** -25 * math.sqrt(want.numel()) * (t == "f16")
        assert off <= tol, (tuple(g.shape), off, tol)
    assert torch.equal(got, ad.orthogonalize(g, steps=steps, coefficients=coef, eps=eps))
    return got


SHAPES = [(128, 257), (600, 100), (40, 511), (128, 512), (513, 128), (70, 1000), (1024, 128), (3, 1025), (128, 2000), (2048, 65),
          (100, 2049), (1, 2048), (1, 1), (1, 50), (50, 1), (7, 5), (5, 7), (64, 64), (100, 257), (128, 256), (256, 128), (129, 127), (333, 101),
          (101, 333), (768, 300), (1000, 1000), (64, 3000), (3000, 60), (2000, 520), (768, 1536)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(ad, shape, t):
    g = _gen(shape[0] + shape[1])
    _check(ad, (torch.randn(*shape, generator=g, device="cuda") * 0.02).to(T[t]), t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 5000), (5000, 3), (1, 32768), (32768, 2), (17, 4001), (9001, 130)])
def test_orthogonalize_long_and_thin(ad, shape, t):
    _check(ad, torch.randn(*shape, generator=_gen(shape[0]), device="cuda").to(T[t]), t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("batch,m,n", [(2, 40, 24), (3, 100, 257), (8, 256, 128), (5, 128, 700), (4, 1024, 600),
                                       (30, 64, 1500), (29, 700, 120), (200, 30, 300)])
def test_orthogonalize_batches(ad, batch, m, n, t):
    x = (torch.randn(batch, m, n, generator=_gen(m), device="cuda") * torch.logspace(-6, 3, batch, device="cuda")[:, None, None]).to(T[t])
    got = _check(ad, x, t)
    for k in range(batch):  # each on its own; another split of k may serve another batch
        assert float((got[k].double() - ad.orthogonalize(x[k]).double()).norm()) <= (
            6 * _iterate(x[k])[1] + 2 * U[t] * float(got[k].double().norm()))


@pytest.mark.parametrize("steps", [0, 1, 2, 8])
@pytest.mark.parametrize("coef", [COEF, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.5, -0.6, 0.01), (1.9, 0.0, 0.0)])
def test_orthogonalize_steps_and_coefficients(ad, steps, coef):
    for m, n in ((60, 200), (300, 70), (100, 1100), (300, 260)):
        _check(ad, torch.randn(m, n, generator=_gen(m + steps), device="cuda"), "f32", steps, coef)


@pytest.mark.parametrize("m,n", [(96, 200), (400, 130)])
def test_orthogonalize_few_directions(ad, m, n):
    """Singular values that fall by 1e5, and a matrix of rank three."""
    g = _gen(m)
    r = min(m, n)
    u, _ = torch.linalg.qr(torch.randn(m, r, generator=g, device="cuda", dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(n, r, generator=g, device="cuda", dtype=torch.float64))
    s = torch.logspace(0, -5, r, device="cuda", dtype=torch.float64)
    _check(ad, ((u * s) @ v.t()).float(), "f32")
    _check(ad, ((u[:, :3] * s[:3]) @ v[:, :3].t()).float(), "f32")


def test_orthogonalize_brings_singular_values_to_one(ad):
    x = torch.randn(200, 600, generator=_gen(9), device="cuda")
    s = torch.linalg.svdvals(ad.orthogonalize(x).double())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25
    u, _, v = torch.linalg.svd(x.double(), full_matrices=False)
    d = (u.t() @ ad.orthogonalize(x).double() @ v.t())
    assert float((d - torch.diag(d.diagonal())).norm()) < 1e-4  # the singular vectors stay


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_orthogonalize_strides(ad, t):
    g = _gen(1)
    x = torch.randn(3, 90, 140, generator=g, device="cuda").to(T[t])
    for view in (x[:, 3:70, 5:101], x[0, :, 1:], x[::2, ::3], x[1].t(), x.transpose(1, 2), x[:1].expand(3, 90, 140),
                 x[1, 4:5], x[1, :, 7:8]):
        assert torch.equal(ad.orthogonalize(view), ad.orthogonalize(view.contiguous()))


def test_orthogonalize_ends(ad):
    for m, n in ((40, 100), (100, 40), (120, 900), (600, 50), (300, 300)):
        z = torch.zeros(3, m, n, device="cuda")
        z[1] = torch.randn(m, n, generator=_gen(m), device="cuda")
        alone = ad.orthogonalize(z[1])
        y = ad.orthogonalize(z)
        assert not y[0].any() and not y[2].any()
        z[0, 3, 4], z[2, 1, 1] = math.nan, math.inf
        bad = ad.orthogonalize(z)
        assert bad[0].isnan().all() and bad[2].isnan().all() and torch.equal(bad[1], y[1])
        assert alone.isfinite().all()
        big = torch.full((m, n), 3e38, device="cuda")  # squares past 32 bits
        _check(ad, big, "f32")
        tiny = torch.full((m, n), 1e-30, device="cuda")
        _check(ad, tiny, "f32", eps=0.0)
    assert ad.orthogonalize(torch.zeros(0, 5, 4, device="cuda")).shape == (0, 5, 4)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("batch,m,n", [(1, 5, 7), (2, 100, 33), (3, 33, 257), (1, 300, 129), (2, 131, 515), (2, 1111, 97)])
def test_orthogonalize_stays_within_its_matrices(ad, batch, m, n, t):
    """Through the C ABI: what lies around the result and the workspace is left as it was."""
    import ctypes as C

    from fusiongpu_b200 import _lib
    g = torch.randn(batch, m, n, generator=_gen(n), device="cuda").to(T[t])
    for steps in (0, 1, 5):
        p = _lib.OrthogonalizeParams(batch, m, n, ad.DTYPES[T[t]], steps, *COEF, 1e-7, 0, 0)
        need = _lib.size_query("fg_orthogonalize_workspace_size", C.byref(p))
        ws = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
        frame = torch.full((batch * m * n + 14,), 77.0, device="cuda").to(T[t])
        _lib.check(_lib.lib().fg_orthogonalize(C.byref(p), g.data_ptr(), frame[7:].data_ptr(), ws[256:].data_ptr(), need,
                                               torch.cuda.current_stream().cuda_stream), "fg_orthogonalize")
        got = frame[7:-7].view(batch, m, n)
        want = ad.orthogonalize(g, steps=steps)
        assert torch.equal(got, want)
        assert (frame[:7] == 77).all() and (frame[-7:] == 77).all()
        assert (ws[:256] == 77).all() and (ws[256 + need:] == 77).all()


@pytest.mark.parametrize("m,n", [(90, 200), (100, 900), (300, 260)])
def test_orthogonalize_at_once_and_captured(ad, m, n):
    """Calls on several streams at once, and two captured graphs beside them, each with its
    workspace."""
    xs = [torch.randn(m, n, generator=_gen(k), device="cuda") for k in range(4)]
    want = [ad.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    graphs = []
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ad.orthogonalize(x)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                if k < 2:
                    graphs[k][0].replay()
                got.append(graphs[k][1] if k < 2 else ad.orthogonalize(xs[k]))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_orthogonalize_refusals(ad):
    from fusiongpu_b200._lib import FgError
    x = torch.ones(4, 6, device="cuda")
    for bad in (x[0], x[None, None], x[:0], x.cpu()):
        with pytest.raises(ValueError):
            ad.orthogonalize(bad)
    with pytest.raises(TypeError):
        ad.orthogonalize(x.double())
    for kw in (dict(steps=-1), dict(steps=101), dict(eps=-1.0), dict(eps=math.inf), dict(eps=math.nan),
               dict(coefficients=(17.0, 0.0, 0.0)), dict(coefficients=(1.0, math.nan, 0.0))):
        with pytest.raises(FgError):
            ad.orthogonalize(x, **kw)
    with pytest.raises(FgError):
        ad.orthogonalize(torch.zeros(1, 32769, device="cuda"))
