"""GPU tests of the gated adapter as it is used: trained by orthogonalised updates,
served in 8 bits, on other streams and in CUDA graphs.

Tolerances as in the operators' own tests; where results pass through several
operators they say how they were derived."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ad():
    from fusiongpu_b200 import adapter
    return adapter


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _act(z, act):
    return {"gelu": lambda v: v * torch.special.ndtr(v), "silu": lambda v: v * torch.sigmoid(v)}[act](z)


def _plain_out(p, q, act):
    """The gated adapter in 64 bits."""
    p, q = {k: v.double() for k, v in p.items()}, q.double()
    c = q - q.mean(1, keepdim=True)
    n = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * p["norm_weight"] + p["norm_bias"]
    z = n @ p["w1"].t() + p["b1"]
    h = z.shape[1] // 2
    return q + (_act(z[:, :h], act) * z[:, h:]) @ p["w2"].t() + p["b2"]


def _plain_loss(p, q, base, off, pos, neg, beta, act):
    of = torch.repeat_interleave(torch.arange(q.shape[0], device="cuda"), off[1:] - off[:-1])
    up, down = base.double()[pos.long()], base.double()[neg.long()]
    u = _plain_out(p, q, act) - q.double()
    z = beta * 2 * (u[of] * (up - down)).sum(1)
    return -torch.nn.functional.logsigmoid(z).sum()


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gated_train_step_against_differences(ad, act):
    """Each parameter's gradient along a random direction against the central
    difference of the 64-bit loss.  The gradients are float32 through a few
    hundred operations: 2^-24 * 2000 of their magnitude; the difference's step of
    1e-5 leaves 1e-9 of a third derivative, the loss's 1e-15 over the step 1e-8."""
    g = _gen(11)
    d, hid, nq, nb = 40, 56, 50, 60
    base, q = _randn(g, nb, d, scale=0.3), _randn(g, nq, d, scale=0.3)
    off = torch.cumsum(torch.tensor([0] + [k % 5 for k in range(nq)], device="cuda"), 0)
    pos, neg = (torch.randint(0, nb, (int(off[-1]),), generator=g, device="cuda", dtype=torch.int32) for _ in range(2))
    m = ad.QueryAdapter(d, hid, act, seed=1, gated=True)
    assert m.params["w1"].shape == (2 * hid, d) and torch.equal(m(q), q)
    for k in m.params:
        m.params[k] += _randn(g, *m.params[k].shape, scale=0.2)
    losses, _ = m.train_step(q, base, off, pos, neg, beta=1.5, metric="l2")
    want = _plain_loss(m.params, q, base, off, pos, neg, 1.5, act)
    assert abs(float(losses.double().sum() - want)) <= 2000 * E32 * float(want)
    for k, v in m.params.items():
        for _ in range(3):
            u = _randn(g, *v.shape).double()
            step = 1e-5 / float(u.norm())
            vals = []
            for sgn in (1, -1):
                p = {n: t.double() for n, t in m.params.items()}
                p[k] = p[k] + sgn * step * u
                vals.append(float(_plain_loss(p, q, base, off, pos, neg, 1.5, act)))
            diff = (vals[0] - vals[1]) / (2 * step)
            got = float((v.grad.double() * u).sum())
            scale = float(v.grad.double().norm() * u.norm())
            assert abs(got - diff) <= 2000 * E32 * scale + 1e-7 * float(u.norm()), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_follows_its_formula(ad, dtype, nesterov, decay):
    """Three steps against the formula with the operator's own update: the same torch
    operations, so the same bits."""
    g = _gen(5)
    shapes = [(60, 40), (60, 40), (30, 100), (40, 60)]
    params = [_randn(g, *s, dtype=dtype) for s in shapes]
    mine = [p.clone() for p in params]
    opt = ad.Muon(params, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    moments = [torch.zeros_like(p) for p in params]
    for _ in range(3):
        grads = [_randn(g, *s, dtype=dtype) for s in shapes]
        for p, d in zip(params, grads):
            p.grad = d
        opt.step()
        us = []
        for k, d in enumerate(grads):
            moments[k].mul_(0.9).add_(d)
            us.append(d.add(moments[k], alpha=0.9) if nesterov else moments[k].clone())
        both = ad.orthogonalize(torch.stack(us[:2]))
        for k, o in enumerate([both[0], both[1], ad.orthogonalize(us[2]), ad.orthogonalize(us[3])]):
            if decay:
                mine[k].mul_(1 - 0.1 * decay)
            mine[k].add_(o, alpha=-0.1 * math.sqrt(max(1.0, shapes[k][0] / shapes[k][1])))
        for p, q in zip(params, mine):
            assert torch.equal(p, q)
    for p in params:
        p.grad = None
    opt.step()
    for p, q in zip(params, mine):
        assert torch.equal(p, q)


def test_muon_refusals(ad):
    v = torch.zeros(8, device="cuda")
    with pytest.raises(ValueError):
        ad.Muon([v])
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            ad.Muon([v.view(2, 4)], **kw)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nq", [1, 7, 200])
def test_quantized_adapter(ad, nq, dtype, gated):
    """In 8 bits against the adapter itself.  An operand's code is off by up to 1 / 254 of
    its row's largest value, evenly: 1 / 440 of it in standard deviation, so 0.7 to 1.4 %
    of values whose largest is 3 to 6 deviations.  Four operands in two layers make 2 to
    3 % of the update's norm; 5 % is allowed, and the results' rounding."""
    g = _gen(nq)
    m = ad.QueryAdapter(96, 160, "silu", dtype=dtype, gated=gated)
    for k in ("w2", "b1", "b2"):
        m.params[k].copy_(_randn(g, *m.params[k].shape, dtype=dtype, scale=0.1))
    q = _randn(g, nq, 96, dtype=dtype)
    eight = m.quantized()
    got, full = eight(q), m(q)
    assert got.dtype == dtype and got.shape == full.shape
    update = (full.double() - q.double()).norm()
    assert float((got.double() - full.double()).norm()) <= 0.05 * float(update) + torch.finfo(dtype).eps * float(full.double().norm())
    m.params["w1"].zero_()  # a copy was taken
    assert torch.equal(eight(q), got)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    there = eight(q, stream=s)
    s.synchronize()
    assert torch.equal(there, got)


def test_new_operators_on_another_stream(ad):
    g = _gen(4)
    x, w = _randn(g, 3000, 500, dtype=torch.bfloat16), _randn(g, 512, 500, dtype=torch.bfloat16, scale=0.05)
    dy = _randn(g, 3000, 256, dtype=torch.bfloat16)
    xq, xs = ad.quantize_rows(x)
    wq, ws = ad.quantize_rows(w)
    odd = xq[:, 1:]  # off 16 bytes: packed in the workspace

    def all_of(**kw):
        y, pre = ad.gated_linear(x, w, return_pre=True, **kw)
        return (y, pre, *ad.gated_linear_backward(dy, x, w, pre, **kw), *ad.quantize_rows(x, **kw),
                ad.linear_int8(odd, xs, wq[:, 1:], ws, **kw), ad.orthogonalize(w, **kw), ad.orthogonalize(x[:1200], **kw))

    here = all_of()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        there = all_of(stream=s)
        torch.empty(1 << 22, device="cuda").fill_(7)  # the default stream's allocations stay off that workspace
    s.synchronize()
    for u, v in zip(here, there):
        assert torch.equal(u, v)


@pytest.mark.parametrize("nq", [1, 40, 3000])
def test_gated_adapters_in_cuda_graphs(ad, nq):
    """Both serving paths, captured and replayed on new queries; two graphs and an
    eager call in flight do not share workspaces."""
    m = ad.QueryAdapter(250, 130, dtype=torch.float16, gated=True)
    m.params["w2"].normal_(std=0.05, generator=_gen(1))
    e = m.quantized()
    q = _randn(_gen(1), nq, 250, dtype=torch.float16)
    m(q), e(q)
    torch.cuda.synchronize()
    graphs = []
    for f in (m, e):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(q)
        graphs.append((graph, out))
    for seed in range(3):
        q.copy_(_randn(_gen(seed), nq, 250, dtype=torch.float16))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        want = m(q), e(q)
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert torch.equal(out, w)


def test_training_step_in_a_cuda_graph(ad):
    """Gradients and the orthogonalised update captured once and replayed on new data."""
    g = _gen(3)
    x, w = _randn(g, 700, 96), _randn(g, 144, 96, scale=0.1)
    dy = _randn(g, 700, 72)

    def step():
        y, pre = ad.gated_linear(x, w, return_pre=True)
        dx, dw, db = ad.gated_linear_backward(dy, x, w, pre)
        return y, dx, db, ad.orthogonalize(dw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        x.copy_(_randn(_gen(seed), 700, 96))
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, step()):
            assert torch.equal(u, v)


@pytest.mark.parametrize("flags", [dict(gated=True, muon=True, int8=True), dict(muon=True), dict(gated=True)])
def test_example_runs(flags):
    import examples.train_query_adapter as ex
    before, after = ex.run(nbase=2000, dim=64, nq=256, nlist=32, pq_m=16, hidden=96, steps=3, verbose=False, **flags)
    assert 0 <= before <= 1 and 0 <= after <= 1
