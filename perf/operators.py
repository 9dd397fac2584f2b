"""Cases of the framework's dense-layer and matrix-optimizer operators: what they compute in plain torch, in 64 bits,
and through the framework.

  linear          y = act(x W + b) + residual, optionally with the pre-activation z kept for the backward pass
  linear_bwd      dz = dy act'(z), dx = dz W^T, dW = x^T dz, db = column sums of dz
  newton_schulz   X = G / (|G| + eps); steps times X <- a X + (b A + c A^2) X with A = X X^T
  muon            one optimizer step over a flat parameter buffer: momentum, orthogonalised update of every matrix, Adam for the vectors
"""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
ALIGN = 64           # every tensor of a flat buffer starts on a multiple of this many floats
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
LARGEST_FLOPS = 2 * 8192 * 4096 * 8192


def listed():
    return [
        # one row through a square layer: what a served model does for every token
        dict(name="linear row bf16", op="linear", m=1, k=4096, n=4096, dtype="bf16", act="silu", residual=True, pre=False, trans_w=False),
        # the first fully connected layer of the MNIST network, at its default batch
        dict(name="linear mnist fc1 fp32", op="linear", m=128, k=3136, n=512, dtype="fp32", act="relu", residual=False, pre=True, trans_w=False),
        # a ragged batch with odd sizes through a layer kept as [out, in]
        dict(name="linear ragged fp16", op="linear", m=1003, k=1531, n=2050, dtype="fp16", act="gelu_tanh", residual=True, pre=False, trans_w=True),
        # a wide hidden layer in training: many rows, pre-activation kept
        dict(name="linear wide bf16", op="linear", m=8192, k=4096, n=8192, dtype="bf16", act="gelu", residual=False, pre=True, trans_w=False),
        # gradients of the MNIST network's first fully connected layer
        dict(name="bwd mnist fc1 fp32", op="linear_bwd", m=128, k=3136, n=512, dtype="fp32", act="relu", trans_w=False),
        # odd sizes, backward
        dict(name="bwd ragged fp16", op="linear_bwd", m=777, k=1001, n=1300, dtype="fp16", act="silu", trans_w=True),
        # gradients of a square hidden layer over a large batch
        dict(name="bwd wide bf16", op="linear_bwd", m=8192, k=4096, n=4096, dtype="bf16", act="gelu", trans_w=False),
        # the 64-channel 3x3 filters of the 20-layer CIFAR network, as [kh kw in, out] matrices
        dict(name="ns filters fp32", op="newton_schulz", batch=6, m=576, n=64, dtype="fp32", steps=5),
        # a wide projection's gradient in 16 bits
        dict(name="ns wide bf16", op="newton_schulz", batch=1, m=1024, n=4096, dtype="bf16", steps=5),
        # a large square weight
        dict(name="ns square fp32", op="newton_schulz", batch=1, m=4096, n=4096, dtype="fp32", steps=5),
        # one update of the 20-layer CIFAR network: many small filters, vectors by Adam
        dict(name="muon resnet20", op="muon", net="resnet", size=3, nesterov=True, weight_decay=0.0),
        # one update of the MNIST network: a few matrices of very different shapes
        dict(name="muon mnist", op="muon", net="mnist", size=0, nesterov=True, weight_decay=0.01),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_bwd", "linear_bwd", "newton_schulz", "newton_schulz", "muon"))
    if op in ("linear", "linear_bwd"):
        c = dict(op=op, m=_log_int(rng, 1, 8192), k=_log_int(rng, 8, 8192), n=_log_int(rng, 8, 8192),
                 dtype=rng.choice(("fp32", "bf16", "fp16")), act=rng.choice(ACTIVATIONS), trans_w=rng.random() < 0.4)
        if rng.random() < 0.5:   # half of them as sizes of 16-byte rows, the others as they fall
            c["k"], c["n"] = (c["k"] + 7) // 8 * 8, (c["n"] + 7) // 8 * 8
        if op == "linear":
            c.update(residual=rng.random() < 0.5, pre=rng.random() < 0.5)
        while work(c)["flops"] * (4 if c["dtype"] == "fp32" else 1) > LARGEST_FLOPS:
            c["m"] = max(1, c["m"] // 2)
        return c
    if op == "newton_schulz":
        c = dict(op=op, batch=rng.choice((1, 1, 2, 3, 6)), m=_log_int(rng, 1, 4096), n=_log_int(rng, 1, 4096),
                 dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), steps=rng.choice((3, 5, 5, 6)))
        most = work(dict(op=op, batch=1, m=4096, n=4096, dtype="fp32", steps=5))["flops"]
        while work(c)["flops"] > most / 2:
            c["m"] = max(1, c["m"] // 2)
        return c
    net = rng.choice(("resnet", "fc"))
    size = rng.choice([n for n in range(1, 19) if n != 3]) if net == "resnet" else _log_int(rng, 20, 1500)
    return dict(op=op, net=net, size=size, nesterov=rng.random() < 0.7, weight_decay=rng.choice((0.0, 0.01)))


# ---------------------------------------------------------------- parameter tables of the optimizer cases
def _shapes(net, size):
    if net == "mnist":
        return [(5, 5, 1, 32), (32,), (5, 5, 32, 64), (64,), (3136, 512), (512,), (512, 10), (10,)]
    if net == "fc":   # a stack of fully connected layers whose widths shrink
        widths = [784, size, max(8, size // 2 + 1), max(8, size // 3), 10]
        out = []
        for a, b in zip(widths, widths[1:]):
            out += [(a, b), (b,)]
        return out
    out, cin = [(3, 3, 3, 16), (16,), (16,)], 16
    for stage, c in enumerate((16, 32, 64)):
        for i in range(size):
            if stage or i:
                out += [(cin,), (cin,)]
            out += [(3, 3, cin, c), (c,), (c,), (3, 3, c, c)]
            cin = c
    return out + [(64,), (64,), (64, 10), (10,)]


def _layout(shapes):
    off, table = 0, []
    for s in shapes:
        table.append((off, s))
        off += (math.prod(s) + ALIGN - 1) // ALIGN * ALIGN
    return table, off


def _matrix(shape):
    return math.prod(shape[:-1]), shape[-1]


# ---------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _gradient(gen, batch, m, n):
    """Matrices like gradients: a few strong directions whose weight falls off, over a floor of noise."""
    k = min(16, m, n)
    fall = 0.5 ** torch.linspace(0, 6, k, device="cuda")
    return 1e-3 * (torch.matmul(_randn(gen, batch, m, k) * fall, _randn(gen, batch, k, n)) / math.sqrt(k) + 0.05 * _randn(gen, batch, m, n))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op in ("linear", "linear_bwd"):
        m, k, n, dt = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
        s["x"] = _randn(gen, m, k).to(dt)
        w = _randn(gen, k, n) / math.sqrt(k)
        s["w"] = (w.t().contiguous() if case["trans_w"] else w).to(dt)
        if op == "linear":
            s["bias"] = (0.1 + 0.1 * _randn(gen, n)).to(dt)
            s["res"] = _randn(gen, m, n).to(dt) if case["residual"] else None
        else:
            s["dy"] = (_randn(gen, m, n) / 16).to(dt)
            s["z"] = (0.1 + _randn(gen, m, n)).to(dt)
    elif op == "newton_schulz":
        g = _gradient(gen, case["batch"], case["m"], case["n"])
        if case["dtype"] == "fp16":
            g = g * 1024   # as a loss scale does
        s["g"] = g.to(DTYPES[case["dtype"]])
    else:
        shapes = _shapes(case["net"], case["size"])
        table, total = _layout(shapes)
        p, g, mo, v = (torch.zeros(total, device="cuda") for _ in range(4))
        for off, shape in table:
            num = math.prod(shape)
            if len(shape) > 1:
                r, c = _matrix(shape)
                p[off:off + num] = 0.1 * _randn(gen, num)
                g[off:off + num] = _gradient(gen, 1, r, c).reshape(-1)
                mo[off:off + num] = 10 * _gradient(gen, 1, r, c).reshape(-1)
            else:
                p[off:off + num] = 0.1
                g[off:off + num] = 1e-3 * _randn(gen, num)
                mo[off:off + num] = 1e-3 * _randn(gen, num)
                v[off:off + num] = 1e-6 * (0.5 + torch.rand(num, device="cuda", generator=gen))
        s.update(table=table, p=p, g=g, m=mo, v=v, t=0)
        if own:
            from distributed_tensorflow_amd.optim import FlatMuon
            from distributed_tensorflow_amd.runtime.arena import ParamArena, ParamSpec

            arena = ParamArena([ParamSpec("p%d" % i, shape, "zeros") for i, shape in enumerate(shapes)], "cuda", FlatMuon.slots)
            arena.params.copy_(p)
            arena.grads.copy_(g)
            arena.slots["m"].copy_(mo)
            arena.slots["v"].copy_(v)
            s.update(arena=arena, opt=FlatMuon(arena, nesterov=case["nesterov"], weight_decay=case["weight_decay"]))
    return s


# ---------------------------------------------------------------- the plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z))
    if act == "silu":
        q = 1 / (1 + torch.exp(-z))
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


def _linear_plain(s):
    w = s["w"].float()
    z = torch.matmul(s["x"].float(), w.t() if s["trans_w"] else w) + s["bias"].float()
    y = _act(z, s["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    dt = s["x"].dtype
    return {"y": y.to(dt), "pre": z.to(dt)} if s["pre"] else {"y": y.to(dt)}


def _linear_bwd_plain(s):
    dt, w, x = s["x"].dtype, s["w"].float(), s["x"].float()
    dz = s["dy"].float() * _act_grad(s["z"].float(), s["act"])
    dx = torch.matmul(dz, w if s["trans_w"] else w.t())
    dw = torch.matmul(dz.t(), x) if s["trans_w"] else torch.matmul(x.t(), dz)
    return {"dx": dx.to(dt), "dw": dw.to(dt), "db": dz.sum(0).to(dt)}


def _orthogonalise(g, steps):
    """[batch, m, n] in 32 bits; the norm in 64 (squares of small gradients leave the range of 32)."""
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    norm = g.double().square().sum((1, 2), keepdim=True).sqrt()
    x = x / (norm + NS_EPS).float()
    a, b, c = COEFFS
    for _ in range(steps):
        s = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(1, 2) if tall else x


LR, VECTOR_LR, GRAD_SCALE, MU = 0.02, 1e-3, 0.5, 0.95
BETA1, BETA2, ADAM_EPS = 0.9, 0.999, 1e-8


def _muon_plain(s):
    s["t"] += 1
    lr_t = VECTOR_LR * math.sqrt(1 - BETA2 ** s["t"]) / (1 - BETA1 ** s["t"])
    for off, shape in s["table"]:
        num = math.prod(shape)
        p, g, m, v = (s[q][off:off + num] for q in "pgmv")
        g = g * GRAD_SCALE
        if len(shape) > 1:
            r, c = _matrix(shape)
            m.mul_(MU).add_(g)
            u = g + MU * m if s["nesterov"] else m
            o = _orthogonalise(u.view(1, r, c), 5).reshape(-1)
            p.mul_(1 - LR * s["weight_decay"]).sub_(LR * math.sqrt(max(1.0, c / r)) * o)
        else:
            m.mul_(BETA1).add_((1 - BETA1) * g)
            v.mul_(BETA2).add_((1 - BETA2) * g * g)
            p.sub_(lr_t * m / (v.sqrt() + ADAM_EPS))
    return {"p": s["p"], "m": s["m"], "v": s["v"]}


def run(s):
    op = s["op"]
    if not own:
        if op == "linear":
            return _linear_plain(s)
        if op == "linear_bwd":
            return _linear_bwd_plain(s)
        if op == "newton_schulz":
            return {"o": _orthogonalise(s["g"], s["steps"]).to(s["g"].dtype).contiguous()}
        return _muon_plain(s)
    from distributed_tensorflow_amd.ops import native as nv

    if op == "linear":
        pre = torch.empty((s["m"], s["n"]), device="cuda", dtype=s["x"].dtype) if s["pre"] else None
        y = nv.linear(s["x"], s["w"], s["bias"], activation=s["act"], residual=s["res"], trans_w=s["trans_w"], pre=pre)
        return {"y": y, "pre": pre} if s["pre"] else {"y": y}
    if op == "linear_bwd":
        dx, dw, db = nv.linear_bwd(s["dy"], s["x"], s["w"], pre=s["z"], activation=s["act"], trans_w=s["trans_w"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "newton_schulz":
        return {"o": nv.newton_schulz(s["g"], steps=s["steps"])}
    s["opt"].step(LR, grad_scale=GRAD_SCALE, vector_lr=VECTOR_LR)
    a = s["arena"]
    return {"p": a.params, "m": a.slots["m"], "v": a.slots["v"]}


# ---------------------------------------------------------------- what a pass cannot do without
def _ns_flops(m, n, steps):
    r, c = min(m, n), max(m, n)
    return steps * (r * (r + 1) * c + r * r * (r + 1) + 2 * r * r * c)   # the two symmetric products by half


def work(case):
    op = case["op"]
    if op in ("linear", "linear_bwd"):
        m, k, n, b = case["m"], case["k"], case["n"], SIZES[case["dtype"]]
        if op == "linear":
            return {"bytes": b * (m * k + k * n + n + m * n * (1 + case["residual"] + case["pre"])), "flops": 2 * m * k * n}
        return {"bytes": b * (m * n * (1 + (case["act"] != "none")) + 2 * m * k + 2 * k * n + n), "flops": 4 * m * k * n}
    if op == "newton_schulz":
        return {"bytes": 2 * SIZES[case["dtype"]] * case["batch"] * case["m"] * case["n"], "flops": case["batch"] * _ns_flops(case["m"], case["n"], case["steps"])}
    size = flops = 0
    for shape in _shapes(case["net"], case["size"]):
        num = math.prod(shape)
        size += 4 * num * (5 if len(shape) > 1 else 7)
        flops += _ns_flops(*_matrix(shape), 5) if len(shape) > 1 else 12 * num
    return {"bytes": size, "flops": flops}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _act64(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":   # (1 + tanh u) / 2 is the logistic function of 2 u
        u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        q = torch.sigmoid(u2)
        return z * q, q + z * q * torch.sigmoid(-u2) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    if act == "silu":
        q = torch.sigmoid(z)
        return z * q, q + z * q * torch.sigmoid(-z)
    return z, torch.ones_like(z)


def _ns64(g, steps):
    """The same polynomial on the other side of the product: X (a I + S (b I + c S)), S = X^T X, with X tall."""
    x = g.double()
    flip = x.shape[0] < x.shape[1]
    x = x.t().contiguous() if flip else x
    x = x / (torch.linalg.vector_norm(x) + NS_EPS)
    eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
    a, b, c = COEFFS
    for _ in range(steps):
        s = torch.mm(x.t().contiguous(), x)
        x = torch.mm(x, a * eye + torch.mm(s, b * eye + c * s))
    return x.t().contiguous() if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        w = s["w"].double()
        z = torch.addmm(s["bias"].double(), s["x"].double(), w.t().contiguous() if case["trans_w"] else w)
        y, _ = _act64(z, case["act"])
        if case["residual"]:
            y = y + s["res"].double()
        return {"y": y, "pre": z} if case["pre"] else {"y": y}
    if op == "linear_bwd":
        dz = s["dy"].double() * _act64(s["z"].double(), case["act"])[1]
        w, x = s["w"].double(), s["x"].double()
        dw = torch.mm(x.t().contiguous(), dz)
        return {"dx": torch.mm(dz, w if case["trans_w"] else w.t().contiguous()), "dw": dw.t().contiguous() if case["trans_w"] else dw,
                "db": torch.mv(dz.t().contiguous(), torch.ones(case["m"], dtype=torch.float64, device=dz.device))}
    if op == "newton_schulz":
        return {"o": torch.stack([_ns64(g, case["steps"]) for g in s["g"]])}
    p, g, m, v = (s[q].double() for q in "pgmv")
    g = g * GRAD_SCALE
    lr_t = VECTOR_LR * math.sqrt(1 - BETA2) / (1 - BETA1)
    for off, shape in s["table"]:
        at = slice(off, off + math.prod(shape))
        if len(shape) > 1:
            r, c = _matrix(shape)
            m[at] = MU * m[at] + g[at]
            u = g[at] + MU * m[at] if case["nesterov"] else m[at]
            p[at] = p[at] - LR * case["weight_decay"] * p[at] - LR * max(1.0, c / r) ** 0.5 * _ns64(u.view(r, c), 5).reshape(-1)
        else:
            m[at] = BETA1 * m[at] + (1 - BETA1) * g[at]
            v[at] = BETA2 * v[at] + (1 - BETA2) * g[at] ** 2
            p[at] = p[at] - lr_t * m[at] / (v[at].sqrt() + ADAM_EPS)
    return {"p": p, "m": m, "v": v}
