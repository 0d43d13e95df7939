"""The query adapter's operators, as cases to measure: layer norm, the linear
layer with its fused epilogue, and the preference loss over indexed documents.

A query adapter sits before the search call: it maps an embedding model's
query vectors into the space of an index that is already built, and is trained
on (preferred, rejected) document pairs against the index's raw vectors.  Each
case is one pass of one operator in one direction.  `own` selects the
framework's kernels; otherwise the plain form runs: elementary torch
operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}
_B = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1}
EPS = 1e-5


def listed():
    return [
        # one query on the serving path, embedding width 768
        dict(name="ln_fwd_one_query", op="ln_fwd", rows=1, dim=768, type="f16", param="f16", stats=False),
        # a training batch of 10,000 queries, 32-bit parameters beside 16-bit activations
        dict(name="ln_bwd_batch", op="ln_bwd", rows=10000, dim=768, type="f16", param="f32"),
        # normalising a whole 1M x 128 float base
        dict(name="ln_fwd_base", op="ln_fwd", rows=1000000, dim=128, type="f32", param="f32", stats=True),
        # odd width: no row but the first starts on a 16-byte boundary
        dict(name="ln_bwd_odd", op="ln_bwd", rows=3001, dim=1001, type="f32", param="f32"),
        # one query through the adapter's first layer
        dict(name="linear_one_query", op="lin_fwd", rows=1, n_in=768, n_out=1536, type="f16", act="gelu", bias=True,
             residual=False, pre=False),
        # a batch of 100 queries through the second layer, with the residual
        dict(name="linear_100_queries", op="lin_fwd", rows=100, n_in=1536, n_out=768, type="bf16", act="none",
             bias=True, residual=True, pre=False),
        # a training batch, the pre-activation kept for the backward pass
        dict(name="linear_train", op="lin_fwd", rows=10000, n_in=768, n_out=1536, type="bf16", act="gelu", bias=True,
             residual=False, pre=True),
        # its backward pass
        dict(name="linear_bwd_train", op="lin_bwd", rows=10000, n_in=768, n_out=1536, type="bf16", act="gelu"),
        # float vectors of an odd width, on the width of a PQ-coded index
        dict(name="linear_odd_f32", op="lin_fwd", rows=1777, n_in=101, n_out=333, type="f32", act="silu", bias=True,
             residual=True, pre=True),
        # re-projecting a whole 1M x 768 half-precision base
        dict(name="linear_base", op="lin_fwd", rows=1000000, n_in=768, n_out=768, type="f16", act="none", bias=True,
             residual=True, pre=False),
        # a small feedback batch against byte vectors, ten pairs a query
        dict(name="preference_small", op="pref", queries=32, pairs=10, dim=128, type="f32", base="u8", nbase=100000,
             metric="l2", ref=True, smooth=0.0, ragged=False),
        # a training batch of 10,000 queries with 16 pairs each on average, on the 1M x 768 half-precision base
        dict(name="preference_train", op="pref", queries=10000, pairs=32, dim=768, type="f16", base="f16",
             nbase=1000000, metric="ip", ref=True, smooth=0.1, ragged=True),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    v = v if rng.random() < 0.4 else max(8, v // 8 * 8)  # most widths are multiples of 8, the others any
    return v + 8 if v == 3072 else v


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "lin_fwd", "lin_fwd", "lin_bwd", "pref"])
    t = rng.choice(["f32", "f16", "bf16"])
    if op in ("ln_fwd", "ln_bwd"):
        dim = _width(rng, 32, 4096)
        rows = _log(rng, 1, max(2, min(1000000, 200000000 // dim)))
        c = dict(op=op, rows=rows, dim=dim, type=t, param=rng.choice([t, "f32"]))
        if op == "ln_fwd":
            c["stats"] = rng.random() < 0.5
        return c
    if op in ("lin_fwd", "lin_bwd"):
        n_in, n_out = _width(rng, 24, 2048), _width(rng, 24, 2048)
        most = 5e10 if t == "f32" else 2.5e11
        rows = _log(rng, 1, max(2, min(200000, int(most / (2 * n_in * n_out)))))
        c = dict(op=op, rows=rows, n_in=n_in, n_out=n_out, type=t, act=rng.choice(["none", "relu", "gelu", "silu"]))
        if op == "lin_fwd":
            c.update(bias=rng.random() < 0.8, residual=rng.random() < 0.5, pre=rng.random() < 0.5)
        return c
    dim = _width(rng, 32, 1024)
    pairs = _log(rng, 1, 64)
    return dict(op="pref", queries=_log(rng, 1, 200000 // pairs), pairs=pairs, dim=dim, type=t,
                base=rng.choice(["f32", "f16", "u8"]), nbase=_log(rng, 1000, 200000), metric=rng.choice(["l2", "ip"]),
                ref=rng.random() < 0.7, smooth=rng.choice([0.0, 0.1]), ragged=rng.random() < 0.5)


def _pairs(case):
    return max(1, case["queries"] * case["pairs"] // (2 if case["ragged"] else 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], _T[case["type"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    if op in ("ln_fwd", "ln_bwd"):
        n, d, p = case["rows"], case["dim"], _T[case["param"]]
        s = dict(op=op, x=normal(n, d, scale=0.6, mean=0.1), weight=normal(d, scale=0.2, mean=1.0, dtype=p),
                 bias=normal(d, scale=0.1, dtype=p))
        if op == "ln_fwd":
            s["stats"] = case["stats"]
        else:
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt(xf.var(1, unbiased=False) + EPS)
            s["dy"] = normal(n, d, scale=0.05)
        return s
    if op in ("lin_fwd", "lin_bwd"):
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        s = dict(op=op, act=case["act"], x=normal(n, i), w=normal(o, i, scale=i ** -0.5))
        if op == "lin_fwd":
            s["bias"] = normal(o, scale=0.1) if case["bias"] else None
            s["residual"] = normal(n, o, scale=0.5) if case["residual"] else None
            s["pre"] = case["pre"]
        else:
            s["pre"] = normal(n, o) if case["act"] != "none" else None
            s["dy"] = normal(n, o, scale=0.05)
        return s
    nq, d, nb = case["queries"], case["dim"], case["nbase"]
    u8 = case["base"] == "u8"
    base = (torch.randint(0, 256, (nb, d), generator=g, device="cuda", dtype=torch.uint8) if u8
            else normal(nb, d, scale=d ** -0.5, dtype=_T[case["base"]]))
    scale = 30.0 if u8 else d ** -0.5
    ref = normal(nq, d, scale=scale, mean=128.0 if u8 else 0.0)
    q = (ref.float() + torch.randn(nq, d, generator=g, device="cuda") * scale * 0.1).to(t)
    m = _pairs(case)
    offsets = torch.arange(nq + 1, device="cuda") * case["pairs"]
    if case["ragged"]:  # random cuts: some queries have no pair, some many times the mean
        offsets[1:-1] = torch.randint(0, m + 1, (nq - 1,), generator=g, device="cuda").sort().values
        offsets[-1] = m
    pos = torch.randint(0, nb, (m,), generator=g, device="cuda", dtype=torch.int32)
    neg = torch.randint(0, nb, (m,), generator=g, device="cuda", dtype=torch.int32)
    neg[torch.rand(m, generator=g, device="cuda") < 0.03] = -1  # a search's padding among the rejected documents
    spread = 30.0 * 74.0 * math.sqrt(2.0 * d) if u8 else 1.4 * d ** -0.5  # of u . (d+ - d-), u = q
    beta = 1.0 / (spread * (0.1 if case["ref"] else 1.0))
    return dict(op=op, q=q, ref=ref if case["ref"] else None, base=base, offsets=offsets, pos=pos, neg=neg,
                weights=torch.rand(m, generator=g, device="cuda") + 0.5, beta=float(beta), smooth=case["smooth"],
                metric=case["metric"])


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain(s):
    op = s["op"]
    if op == "ln_fwd":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        c = x - mean
        rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
        y = (c * rstd * s["weight"].float() + s["bias"].float()).to(s["x"].dtype)
        return (y, mean[:, 0], rstd[:, 0]) if s["stats"] else y
    if op == "ln_bwd":
        t, p = s["x"].dtype, s["weight"].dtype
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        h = (s["x"].float() - s["mean"][:, None]) * rstd
        a = dy * s["weight"].float()
        dx = (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True)) * rstd
        return dx.to(t), (dy * h).sum(0).to(p), dy.sum(0).to(p)
    if op == "lin_fwd":
        t = s["x"].dtype
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, s["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(t), z.to(t)) if s["pre"] else y.to(t)
    if op == "lin_bwd":
        t = s["x"].dtype
        dz = s["dy"].float()
        if s["act"] != "none":
            dz = dz * _act_grad(s["pre"].float(), s["act"])
        return (dz @ s["w"].float()).to(t), (dz.t() @ s["x"].float()).to(t), dz.sum(0).to(t)
    q, base = s["q"].float(), s["base"]
    nq, nb = q.shape[0], base.shape[0]
    of = torch.repeat_interleave(torch.arange(nq, device=q.device), s["offsets"][1:] - s["offsets"][:-1])
    fine = (s["pos"] >= 0) & (s["pos"] < nb) & (s["neg"] >= 0) & (s["neg"] < nb)
    dp = base[torch.where(fine, s["pos"], 0).long()].float()
    dn = base[torch.where(fine, s["neg"], 0).long()].float()
    diff = dp - dn
    k = (2.0 if s["metric"] == "l2" else 1.0) * s["beta"]
    if s["ref"] is not None:
        z = ((q - s["ref"].float())[of] * diff).sum(1) * k
    elif s["metric"] == "l2":  # |q - d-|^2 - |q - d+|^2, as one sum: 2 (q - (d+ + d-) / 2) . (d+ - d-)
        z = ((q[of] - 0.5 * (dp + dn)) * diff).sum(1) * k
    else:
        z = (q[of] * diff).sum(1) * k
    z = torch.where(fine, z, 0.0)
    tail = torch.log1p(torch.exp(-z.abs()))
    loss = torch.clamp(-z, min=0) + tail + s["smooth"] * z
    loss = torch.where(fine, loss, 0.0)
    coef = torch.where(fine, (s["smooth"] - 1 / (1 + torch.exp(z))) * s["weights"] * k, 0.0)
    dq = torch.zeros_like(q).index_add_(0, of, coef[:, None] * diff)
    return loss, z, dq.to(s["q"].dtype)


def run(state):
    if not own:
        return _plain(state)
    from fusiongpu_b200 import adapter
    s, op = state, state["op"]
    if op == "ln_fwd":
        return adapter.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, return_stats=s["stats"])
    if op == "ln_bwd":
        return adapter.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if op == "lin_fwd":
        return adapter.linear(s["x"], s["w"], s["bias"], activation=s["act"], residual=s["residual"],
                              return_pre=s["pre"])
    if op == "lin_bwd":
        return adapter.linear_backward(s["dy"], s["x"], s["w"], pre=s["pre"], activation=s["act"])
    return adapter.preference_loss(s["q"], s["base"], s["offsets"], s["pos"], s["neg"], ref=s["ref"],
                                   weights=s["weights"], beta=s["beta"], label_smoothing=s["smooth"],
                                   metric=s["metric"])


def work(case):
    op, b = case["op"], _B[case["type"]]
    if op in ("ln_fwd", "ln_bwd"):
        n, d, p = case["rows"], case["dim"], _B[case["param"]]
        if op == "ln_fwd":
            return dict(bytes=2 * n * d * b + 2 * d * p + (8 * n if case["stats"] else 0), flops=8 * n * d)
        return dict(bytes=3 * n * d * b + 8 * n + 3 * d * p, flops=14 * n * d)
    if op in ("lin_fwd", "lin_bwd"):
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        if op == "lin_fwd":
            return dict(bytes=b * (n * i + i * o + n * o * (1 + case["pre"] + case["residual"]) + o * case["bias"]),
                        flops=2 * n * i * o)
        return dict(bytes=b * (n * o * (1 + (case["act"] != "none")) + 2 * n * i + 2 * i * o + o), flops=4 * n * i * o)
    nq, d = case["queries"], case["dim"]
    m = _pairs(case)
    rows = min(2 * m, case["nbase"])  # a document read once
    return dict(bytes=rows * d * _B[case["base"]] + nq * d * b * (2 + case["ref"]) + 20 * m + 8 * (nq + 1),
                flops=7 * m * d)


def exact(case, seed):
    """The definitions in 64 bits; rows in blocks, so that the copies stay small."""
    s = prepare(case, seed)
    op, f8 = s["op"], torch.float64
    if op == "ln_fwd":
        y, mu, rs = [], [], []
        for x in s["x"].split(65536):
            v, m = torch.var_mean(x.to(f8), dim=1, correction=0, keepdim=True)
            r = (v + EPS) ** -0.5
            mu.append(m[:, 0])
            rs.append(r[:, 0])
            y.append(torch.addcmul(s["bias"].to(f8), (x.to(f8) - m) * r, s["weight"].to(f8)))
        y = torch.cat(y)
        return (y, torch.cat(mu), torch.cat(rs)) if s["stats"] else y
    if op == "ln_bwd":
        w, dx = s["weight"].to(f8), []
        dw, db = torch.zeros_like(w), torch.zeros_like(w)
        d = w.numel()
        for x, dy, m, r in zip(s["x"].split(65536), s["dy"].split(65536), s["mean"].split(65536),
                               s["rstd"].split(65536)):
            dy, r = dy.to(f8), r.to(f8)[:, None]
            xc = x.to(f8) - m.to(f8)[:, None]
            dw += torch.einsum("nd,nd,nx->d", dy, xc, r)
            db += torch.einsum("nd->d", dy)
            gw = dy * w
            # dx_j = r g_j - r/d sum(g) - r^3/d xc_j sum(g xc)
            dx.append(r * gw - r / d * gw.sum(1, keepdim=True) - r ** 3 / d * xc * (gw * xc).sum(1, keepdim=True))
        return torch.cat(dx), dw, db
    if op == "lin_fwd":
        y, zs = [], []
        w = s["w"].to(f8)
        for k, x in enumerate(s["x"].split(65536)):
            z = torch.einsum("ni,oi->no", x.to(f8), w)
            if s["bias"] is not None:
                z += s["bias"].to(f8)
            a = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0),
                 "gelu": lambda v: v * torch.special.ndtr(v), "silu": lambda v: v * torch.special.expit(v)}[s["act"]](z)
            if s["residual"] is not None:
                a = a + s["residual"][k * 65536:(k + 1) * 65536].to(f8)
            y.append(a)
            if s["pre"]:
                zs.append(z)
        return (torch.cat(y), torch.cat(zs)) if s["pre"] else torch.cat(y)
    if op == "lin_bwd":
        w = s["w"].to(f8)
        dx, dw, db = [], torch.zeros_like(w), torch.zeros(w.shape[0], dtype=f8, device=w.device)
        for k, (x, dy) in enumerate(zip(s["x"].split(65536), s["dy"].split(65536))):
            dz = dy.to(f8)
            if s["act"] != "none":
                z = s["pre"][k * 65536:(k + 1) * 65536].to(f8)
                if s["act"] == "relu":
                    dz = dz * torch.heaviside(z, torch.zeros((), dtype=f8, device=z.device))
                elif s["act"] == "gelu":
                    dz = dz * (torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) * (2 * math.pi) ** -0.5)
                else:
                    g = torch.special.expit(z)
                    dz = dz * (g + z * g * torch.special.expit(-z))
            dx.append(torch.einsum("no,oi->ni", dz, w))
            dw += torch.einsum("no,ni->oi", dz, x.to(f8))
            db += torch.einsum("no->o", dz)
        return torch.cat(dx), dw, db
    # the four scores' log ratio, pair by pair
    nq, m = s["q"].shape[0], s["pos"].numel()
    first = s["offsets"][1:].contiguous()
    losses, zs = torch.zeros(m, dtype=f8, device="cuda"), torch.zeros(m, dtype=f8, device="cuda")
    dq = torch.zeros(s["q"].shape, dtype=f8, device="cuda")
    for at in range(0, m, 65536):
        p = torch.arange(at, min(m, at + 65536), device="cuda")
        p = p[(s["neg"][p] >= 0) & (s["pos"][p] >= 0)]
        i = torch.searchsorted(first, p, right=True)
        up, down = s["base"][s["pos"][p].long()].to(f8), s["base"][s["neg"][p].long()].to(f8)

        def score(q, d):
            q = q[i].to(f8)
            return torch.einsum("pd,pd->p", q, d) if s["metric"] == "ip" else -(q - d).square().sum(1)

        ratio = score(s["q"], up) - score(s["q"], down)
        if s["ref"] is not None:
            ratio = ratio - (score(s["ref"], up) - score(s["ref"], down))
        z = s["beta"] * ratio
        e = s["smooth"]
        losses[p] = -(1 - e) * torch.nn.functional.logsigmoid(z) - e * torch.nn.functional.logsigmoid(-z)
        zs[p] = z
        dz = ((e * torch.sigmoid(z)) - (1 - e) * torch.sigmoid(-z)) * s["weights"][p].to(f8) * s["beta"]
        dq.index_add_(0, i, (dz * (2 if s["metric"] == "l2" else 1))[:, None] * (up - down))
    return losses, zs, dq
