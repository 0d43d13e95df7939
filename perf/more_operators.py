"""The gated adapter's operators, as cases to measure: the gated layer and its
gradients, the orthogonalised update its matrices are trained with, and the
8-bit linear layer it is served with, with the quantisation of rows.

A gated query adapter puts act(x w_gate^T + b_gate) * (x w_up^T + b_up) where
the plain one has act(x w1^T + b1).  Each case is one pass of one operator in
one direction.  `own` selects the framework's kernels; otherwise the plain form
runs: elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_B = {"f32": 4, "f16": 2, "bf16": 2}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed():
    return [
        # one query through a gated layer on the serving path, width 768; 1024 gated columns have the weights of
        # 1536 plain ones
        dict(name="gated_one_query", op="gated", rows=1, n_in=768, n_out=1024, type="f16", act="silu", bias=True,
             pre=False),
        # a training batch of 10,000 queries, both pre-activations kept for the backward pass
        dict(name="gated_train", op="gated", rows=10000, n_in=768, n_out=1024, type="bf16", act="silu", bias=True,
             pre=True),
        # its backward pass
        dict(name="gated_bwd_train", op="gated_bwd", rows=10000, n_in=768, n_out=1024, type="bf16", act="silu"),
        # gradients of float vectors of an odd width: no row but the first starts on a 16-byte boundary
        dict(name="gated_bwd_odd_f32", op="gated_bwd", rows=1777, n_in=101, n_out=333, type="f32", act="gelu"),
        # activations of 100 queries on their way into an 8-bit layer
        dict(name="quantize_100_queries", op="quantize", rows=100, dim=1536, type="bf16"),
        # a whole 1M x 768 half-precision base to 8 bits
        dict(name="quantize_base", op="quantize", rows=1000000, dim=768, type="f16"),
        # one query through the adapter's first layer in 8 bits
        dict(name="int8_one_query", op="int8", rows=1, n_in=768, n_out=1536, type="f16", act="gelu", bias=True,
             residual=False),
        # a batch of 100 queries through the second, with the residual
        dict(name="int8_100_queries", op="int8", rows=100, n_in=1536, n_out=768, type="bf16", act="none", bias=True,
             residual=True),
        # re-projecting a whole 1M x 768 base
        dict(name="int8_base", op="int8", rows=1000000, n_in=768, n_out=768, type="f16", act="none", bias=True,
             residual=True),
        # the update of a small adapter's first layer (128 -> 256), 32-bit weights
        dict(name="orthogonalize_small", op="orth", batch=1, rows=256, cols=128, type="f32"),
        # of an adapter's first layer (768 -> 1536)
        dict(name="orthogonalize_adapter", op="orth", batch=1, rows=1536, cols=768, type="bf16"),
        # of four adapters' layers at once (1024 -> 2048)
        dict(name="orthogonalize_four", op="orth", batch=4, rows=2048, cols=1024, type="f32"),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else max(8, v // 8 * 8)  # most widths are multiples of 8, the others any


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_bwd", "quantize", "int8", "int8", "orth", "orth"])
    t = rng.choice(["f32", "f16", "bf16"])
    if op in ("gated", "gated_bwd"):
        n_in, n_out = _width(rng, 24, 2048), _width(rng, 24, 1400)
        most = 4e10 if t == "f32" else 2e11
        rows = _log(rng, 1, max(2, min(200000, int(most / (4 * n_in * n_out)))))
        c = dict(op=op, rows=rows, n_in=n_in, n_out=n_out, type=t, act=rng.choice(["none", "relu", "gelu", "silu"]))
        if op == "gated":
            c.update(bias=rng.random() < 0.8, pre=rng.random() < 0.5)
        return c
    if op == "quantize":
        dim = _width(rng, 24, 8192)
        return dict(op=op, rows=_log(rng, 1, max(2, min(1000000, 200000000 // dim))), dim=dim, type=t)
    if op == "int8":
        n_in, n_out = _width(rng, 24, 4096), _width(rng, 24, 2048)
        rows = _log(rng, 1, max(2, min(200000, int(2.5e11 / (2 * n_in * n_out)))))
        return dict(op=op, rows=rows, n_in=n_in, n_out=n_out, type=t, act=rng.choice(["none", "relu", "gelu", "silu"]),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.5)
    while True:
        batch, rows, cols = _log(rng, 1, 8), _width(rng, 24, 2048), _width(rng, 24, 2048)
        if work(dict(op="orth", batch=batch, rows=rows, cols=cols, type=t))["flops"] <= 2e11:
            return dict(op="orth", batch=batch, rows=rows, cols=cols, type=t)


def _codes(g, n, d):
    """Rows of 8-bit codes and their scales, as the quantisation of rows hands
    them out: each row starts on a 16-byte boundary."""
    v = torch.randn(n, d, generator=g, device="cuda")
    top = v.abs().amax(1, keepdim=True).clamp_(min=1e-30)
    q = torch.zeros(n, (d + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :d]
    q.copy_((v * (127 / top)).round_().clamp_(-127, 127))
    return q, (top[:, 0] / 127)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], _T[case["type"]]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if op in ("gated", "gated_bwd"):
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        s = dict(op=op, act=case["act"], x=normal(n, i), w=normal(2 * o, i, scale=i ** -0.5))  # gate rows, then up
        if op == "gated":
            s["bias"] = normal(2 * o, scale=0.1) if case["bias"] else None
            s["pre"] = case["pre"]
        else:
            s["pre"] = normal(n, 2 * o)
            s["dy"] = normal(n, o, scale=0.05)
        return s
    if op == "quantize":
        n, d = case["rows"], case["dim"]
        return dict(op=op, x=normal(n, d, scale=0.6))
    if op == "int8":
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        x, xs = _codes(g, n, i)
        w, ws = _codes(g, o, i)
        return dict(op=op, act=case["act"], dtype=t, x=x, x_scale=xs, w=w, w_scale=ws * i ** -0.5,
                    bias=normal(o, scale=0.1) if case["bias"] else None,
                    residual=normal(n, o, scale=0.5) if case["residual"] else None)
    b, m, n = case["batch"], case["rows"], case["cols"]
    # a gradient: a few strong directions over noise, at a training step's size
    r = min(8, m, n)
    strong = normal(b, m, r, dtype=torch.float32) @ normal(b, r, n, dtype=torch.float32)
    v = 1e-3 * (normal(b, m, n, dtype=torch.float32) + 0.3 * strong)
    return dict(op=op, g=(v if b > 1 else v[0]).to(t).contiguous())


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain(s):
    op = s["op"]
    if op == "gated":
        t, h = s["x"].dtype, s["w"].shape[0] // 2
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = (_act(z[:, :h], s["act"]) * z[:, h:]).to(t)
        return (y, z.to(t)) if s["pre"] else y
    if op == "gated_bwd":
        t, h = s["x"].dtype, s["w"].shape[0] // 2
        dy, gate, up = s["dy"].float(), s["pre"][:, :h].float(), s["pre"][:, h:].float()
        dz = torch.cat([dy * up * _act_grad(gate, s["act"]), dy * _act(gate, s["act"])], dim=1)
        return (dz @ s["w"].float()).to(t), (dz.t() @ s["x"].float()).to(t), dz.sum(0).to(t)
    if op == "quantize":
        x = s["x"].double()  # 127 x / max next to a half needs more than 32 bits
        top = x.abs().amax(1, keepdim=True)
        q = torch.where(top > 0, 127 * x / top, 0.0).round().to(torch.int8)
        return q, (top[:, 0] / 127).float()
    if op == "int8":
        z = (s["x"].float() @ s["w"].float().t()) * (s["x_scale"][:, None] * s["w_scale"])
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, s["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(s["dtype"])
    a, b, c = COEFFICIENTS
    x = s["g"].float()
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    for _ in range(STEPS):
        p = x @ x.mT
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x.mT if tall else x).to(s["g"].dtype)


def run(state):
    if not own:
        return _plain(state)
    from fusiongpu_b200 import adapter
    s, op = state, state["op"]
    if op == "gated":
        return adapter.gated_linear(s["x"], s["w"], s["bias"], activation=s["act"], return_pre=s["pre"])
    if op == "gated_bwd":
        return adapter.gated_linear_backward(s["dy"], s["x"], s["w"], s["pre"], activation=s["act"])
    if op == "quantize":
        return adapter.quantize_rows(s["x"])
    if op == "int8":
        return adapter.linear_int8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["bias"], activation=s["act"],
                                   residual=s["residual"], dtype=s["dtype"])
    return adapter.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


def work(case):
    op, b = case["op"], _B[case["type"]]
    if op in ("gated", "gated_bwd"):
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        if op == "gated":
            return dict(bytes=b * (n * i + 2 * i * o + n * o * (1 + 2 * case["pre"]) + 2 * o * case["bias"]),
                        flops=4 * n * i * o)
        return dict(bytes=b * (3 * n * o + 2 * n * i + 4 * i * o + 2 * o), flops=8 * n * i * o)
    if op == "quantize":
        n, d = case["rows"], case["dim"]
        return dict(bytes=n * d * (b + 1) + 4 * n, flops=3 * n * d)
    if op == "int8":
        n, i, o = case["rows"], case["n_in"], case["n_out"]
        return dict(bytes=n * i + i * o + 4 * (n + o) + b * (n * o * (1 + case["residual"]) + o * case["bias"]),
                    flops=2 * n * i * o)
    m, n = sorted((case["rows"], case["cols"]))
    # p = x x^T and p p are symmetric: half of each; then the product with x
    return dict(bytes=2 * case["batch"] * m * n * b, flops=case["batch"] * STEPS * (m * m * n + m * m * m + 2 * m * m * n))


def exact(case, seed):
    """The definitions in 64 bits; rows in blocks, so that the copies stay small."""
    s = prepare(case, seed)
    op, f8 = s["op"], torch.float64
    act = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v),
           "silu": lambda v: v * torch.special.expit(v)}.get(case.get("act"))
    if op == "gated":
        y, zs = [], []
        gate, up = s["w"].to(f8).chunk(2)
        bias = torch.zeros(s["w"].shape[0], device="cuda", dtype=f8) if s["bias"] is None else s["bias"].to(f8)
        for x in s["x"].split(65536):
            a = torch.einsum("ni,oi->no", x.to(f8), gate) + bias[:gate.shape[0]]
            u = torch.einsum("ni,oi->no", x.to(f8), up) + bias[gate.shape[0]:]
            y.append(torch.mul(act(a), u))
            if s["pre"]:
                zs.append(torch.cat([a, u], 1))
        return (torch.cat(y), torch.cat(zs)) if s["pre"] else torch.cat(y)
    if op == "gated_bwd":
        h = s["dy"].shape[1]
        gate, up = s["w"].to(f8).chunk(2)
        dx, dwg, dwu = [], torch.zeros_like(gate), torch.zeros_like(up)
        db = torch.zeros(2 * h, dtype=f8, device="cuda")
        for x, dy, pre in zip(s["x"].split(65536), s["dy"].split(65536), s["pre"].split(65536)):
            x, dy, a, u = x.to(f8), dy.to(f8), pre[:, :h].to(f8), pre[:, h:].to(f8)
            if case["act"] == "none":
                d = 1.0
            elif case["act"] == "relu":
                d = torch.heaviside(a, torch.zeros((), dtype=f8, device="cuda"))
            elif case["act"] == "gelu":
                d = torch.special.ndtr(a) + a * torch.exp(-a.square() / 2) * (2 * math.pi) ** -0.5
            else:
                e = torch.special.expit(a)
                d = e + a * e * torch.special.expit(-a)
            da, du = dy * u * d, dy * act(a)
            dx.append(torch.einsum("no,oi->ni", da, gate) + torch.einsum("no,oi->ni", du, up))
            dwg += torch.einsum("no,ni->oi", da, x)
            dwu += torch.einsum("no,ni->oi", du, x)
            db += torch.cat([da.sum(0), du.sum(0)])
        return torch.cat(dx), torch.cat([dwg, dwu]), db
    if op == "quantize":
        q, scale = [], []
        for x in s["x"].split(65536):
            x = x.to(f8)
            top = torch.linalg.vector_norm(x, ord=math.inf, dim=1)
            q.append(torch.div(x * 127, top.clamp(min=5e-324)[:, None]).round().to(torch.int8))
            scale.append(top / 127)
        return torch.cat(q), torch.cat(scale)
    if op == "int8":
        y, w = [], s["w"].to(f8) * s["w_scale"].to(f8)[:, None]
        for k, (x, xs) in enumerate(zip(s["x"].split(65536), s["x_scale"].split(65536))):
            z = torch.einsum("ni,oi->no", x.to(f8) * xs.to(f8)[:, None], w)
            if s["bias"] is not None:
                z += s["bias"].to(f8)
            z = act(z)
            if s["residual"] is not None:
                z = z + s["residual"][k * 65536:(k + 1) * 65536].to(f8)
            y.append(z)
        return torch.cat(y)
    # p(x) = a x + b x (x^T x) + c x (x^T x)^2, from the right
    a, b, c = COEFFICIENTS
    x = s["g"].to(f8)
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS)
    if x.shape[-2] >= x.shape[-1]:
        for _ in range(STEPS):
            r = torch.einsum("...ki,...kj->...ij", x, x)
            x = a * x + torch.matmul(torch.matmul(x, r), c * r + b * torch.eye(r.shape[-1], dtype=f8, device="cuda"))
        return x
    for _ in range(STEPS):
        r = torch.einsum("...ik,...jk->...ij", x, x)
        x = a * x + torch.matmul(c * r + b * torch.eye(r.shape[-1], dtype=f8, device="cuda"), torch.matmul(r, x))
    return x
