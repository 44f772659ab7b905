"""The operators of sequence policies, as measurable cases.

A policy with memory is a stack of blocks: a linear layer into gates and
values, a gated linear recurrence over the rollout's steps, a linear layer back
with the residual. It is trained by the backward passes of both and by an
orthogonalised (Muon) update of its matrices, and it acts one step at a time.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) the tensors a program has in hand before the call
    run(state)          one pass: in plain torch, or (own) through phyz_amd.ops
    work(case)          bytes and operations a pass cannot do without
    exact(case, seed)   the pass from the operator's definition, 64 bits

Operators (a case's "op"):

    scan            h_t = c_t h_{t-1} + u_t over [steps, worlds, width], with
                    c = sigmoid(z), u = (1 - c) x ("sigmoid") or c = z, u = x
                    ("decay"); where `reset` is set, h_{t-1} counts as 0
    scan_backward   its gradients for z, x and the first state
    scan_step       one step of it, the state updated in place
    linear          y = act(x W^T + bias) + residual
    linear_backward its gradients for x, W and bias, from the saved
                    pre-activation
    orthogonalize   Newton-Schulz: X = g / |g|, then
                    X <- a X + (b A + c A^2) X with A = X X^T, five times
    muon_step       momentum, orthogonalisation and the weights' update
"""
import math

import torch

own = False

STEPS, COEF, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
BYTES = {"f32": 4, "bf16": 2}
ACTS = ("none", "tanh", "relu", "silu", "gelu")


def listed():
    return [
        # One control step of a recurrent policy on a small batch of worlds: the
        # state's update, launch latency and little else.
        {"name": "scan_step", "op": "scan_step", "dtype": "f32", "form": "sigmoid", "worlds": 1024, "width": 256,
         "reset": True},
        # Forward over a collector's rollout: 4096 worlds at the policy's hidden
        # width, episodes that end inside it.
        {"name": "scan_rollout", "op": "scan", "dtype": "f32", "form": "sigmoid", "steps": 64, "worlds": 4096,
         "width": 256, "reset": True, "batch_first": False},
        # One very long sequence: parallelism has to come from the steps.
        {"name": "scan_long", "op": "scan", "dtype": "bf16", "form": "sigmoid", "steps": 32768, "worlds": 1,
         "width": 2048, "reset": False, "batch_first": False},
        # Backward over ragged sizes, batch-major tensors, odd rows.
        {"name": "scan_backward_odd", "op": "scan_backward", "dtype": "bf16", "form": "decay", "steps": 1023,
         "worlds": 61, "width": 515, "reset": True, "batch_first": True},
        # Serving: sixteen rows through a wide layer, the weights streamed once.
        {"name": "linear_serve", "op": "linear", "dtype": "bf16", "rows": 16, "n_in": 2048, "n_out": 8192,
         "act": "silu", "bias": True, "residual": False},
        # The policy's first layer on a batch of worlds: 55 observations (rows
        # that are not aligned) into 256 hidden units.
        {"name": "linear_policy", "op": "linear", "dtype": "f32", "rows": 4096, "n_in": 55, "n_out": 256,
         "act": "tanh", "bias": True, "residual": False},
        # A wide layer over a training batch, compute bound.
        {"name": "linear_wide", "op": "linear", "dtype": "bf16", "rows": 32768, "n_in": 1024, "n_out": 4096,
         "act": "gelu", "bias": True, "residual": True},
        # The PPO minibatch's hidden layer, backward: long sums over rows into
        # small weight gradients.
        {"name": "linear_backward_hidden", "op": "linear_backward", "dtype": "f32", "rows": 16384, "n_in": 256,
         "n_out": 256, "act": "tanh"},
        # Backward at odd sizes: nothing divides a tile and half the rows are
        # not aligned.
        {"name": "linear_backward_odd", "op": "linear_backward", "dtype": "bf16", "rows": 8191, "n_in": 1000,
         "n_out": 1001, "act": "silu"},
        # Muon on the hidden layers of an actor and a critic.
        {"name": "muon_policy", "op": "muon_step", "dtype": "f32", "batch": 2, "n_out": 256, "n_in": 256},
        # A wide layer's gradient in bfloat16.
        {"name": "orthogonalize_wide", "op": "orthogonalize", "dtype": "bf16", "batch": 1, "n_out": 1024,
         "n_in": 4096},
        # A tall odd matrix in float32.
        {"name": "orthogonalize_odd", "op": "orthogonalize", "dtype": "f32", "batch": 1, "n_out": 1501,
         "n_in": 1001},
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: any operator, sizes over the ranges of the listed ones."""
    op = rng.choice(("scan_step", "scan", "scan", "scan_backward", "scan_backward", "linear", "linear", "linear_backward",
                     "linear_backward", "muon_step", "orthogonalize", "orthogonalize"))
    dtype = rng.choice(("f32", "bf16"))
    if op.startswith("scan"):
        c = {"op": op, "dtype": dtype, "form": rng.choice(("sigmoid", "decay"))}
        if op == "scan_step":
            c.update(worlds=_between(rng, 1, 16384), width=_between(rng, 16, 2048))
        else:
            most = 1 << (26 if op == "scan" else 25)  # positions
            steps, width = _between(rng, 1, 32768), _between(rng, 16, 2048)
            worlds = _between(rng, 1, max(1, min(8192, most // (steps * width))))
            c.update(steps=steps, worlds=worlds, width=width, batch_first=rng.random() < 0.5)
        c["reset"] = rng.random() < 0.5
        return c
    if op.startswith("linear"):
        c = {"op": op, "dtype": dtype, "rows": _between(rng, 1, 65536), "n_in": _between(rng, 16, 4096),
             "n_out": _between(rng, 1, 4096), "act": rng.choice(ACTS)}
        most = (1 << 37) // (8 if dtype == "f32" else 1)  # multiply-adds
        c["rows"] = max(1, min(c["rows"], most // (c["n_in"] * c["n_out"])))
        if op == "linear":
            c.update(bias=rng.random() < 0.7, residual=rng.random() < 0.5)
        return c
    top = 1900 if dtype == "bf16" and op == "orthogonalize" else 1500
    n_out, n_in = _between(rng, 16, top), _between(rng, 16, 2 * top)
    if n_out * n_in < 128 * 1024 and rng.random() < 0.5:
        batch = _between(rng, 2, 16)
    else:
        batch = 1
    return {"op": op, "dtype": "f32" if op == "muon_step" else dtype, "batch": batch, "n_out": n_out, "n_in": n_in}


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen) * scale


def _gates(case, gen, *shape):
    # Learned gates spread over memories from a few steps to some hundreds.
    z = _normal(gen, *shape) * 1.5 + 2.0
    return (z if case["form"] == "sigmoid" else torch.sigmoid(z)).to(_dtype(case))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, op = _dtype(case), case["op"]
    s = {"case": case}
    if op == "scan_step":
        b, d = case["worlds"], case["width"]
        s.update(z=_gates(case, gen, b, d), x=_normal(gen, b, d).to(dt), h=_normal(gen, b, d),
                 reset=torch.rand(b, device="cuda", generator=gen) < 0.02 if case["reset"] else None)
    elif op in ("scan", "scan_backward"):
        t, b, d = case["steps"], case["worlds"], case["width"]

        def lay(v):  # [steps, worlds, width]; batch-major tensors are strided views
            return v.transpose(0, 1) if case["batch_first"] else v

        shape = (b, t, d) if case["batch_first"] else (t, b, d)
        s.update(z=lay(_gates(case, gen, *shape)), x=lay(_normal(gen, *shape).to(dt)), h0=_normal(gen, b, d),
                 reset=torch.rand(t, b, device="cuda", generator=gen) < 0.005 if case["reset"] else None)
        if op == "scan_backward":
            # The states as a forward pass saved them: smooth values of its size.
            s.update(h=lay(_normal(gen, *shape, scale=0.7).to(dt)), dh=lay(_normal(gen, *shape, scale=0.1).to(dt)),
                     dh_last=_normal(gen, b, d, scale=0.1))
    elif op in ("linear", "linear_backward"):
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        s.update(x=_normal(gen, m, k).to(dt), w=_normal(gen, n, k, scale=1.0 / math.sqrt(k)).to(dt))
        if op == "linear":
            s.update(bias=_normal(gen, n, scale=0.1).to(dt) if case["bias"] else None,
                     residual=_normal(gen, m, n).to(dt) if case["residual"] else None)
        else:
            s.update(pre=_normal(gen, m, n).to(dt) if case["act"] != "none" else None,
                     dy=_normal(gen, m, n, scale=0.02).to(dt))
    else:
        q, m, n = case["batch"], case["n_out"], case["n_in"]
        # A gradient: noise on top of a few directions that dominate.
        r = min(8, m, n)
        g = _normal(gen, q, m, n, scale=1e-3)
        g += (_normal(gen, q, m, r, scale=1e-2)[..., None, :] * _normal(gen, q, n, r)[:, None]).sum(-1) / math.sqrt(r)
        s["g"] = g.to(dt)
        if op == "muon_step":
            s.update(w=_normal(gen, q, m, n, scale=1.0 / math.sqrt(n)), m=_normal(gen, q, m, n, scale=2e-3))
    return s


# ── the plain form: elementary torch operations in 32 bits ──────────────────

def _act(a, p):
    if a == "tanh":
        return torch.tanh(p)
    if a == "relu":
        return torch.clamp(p, min=0)
    if a == "silu":
        return p * torch.sigmoid(p)
    if a == "gelu":
        return 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p * p * p)))
    return p


def _act_grad(a, p):
    if a == "tanh":
        y = torch.tanh(p)
        return 1 - y * y
    if a == "relu":
        return (p > 0).to(p.dtype)
    if a == "silu":
        g = torch.sigmoid(p)
        return g * (1 + p * (1 - g))
    c = math.sqrt(2 / math.pi)
    y = torch.tanh(c * (p + 0.044715 * p * p * p))
    return 0.5 * (1 + y) + 0.5 * p * (1 - y * y) * c * (1 + 3 * 0.044715 * p * p)


def _recur(c, u):
    """h_t = c_t h_{t-1} + u_t along the first axis, by doubling."""
    s = 1
    while s < u.shape[0]:
        u = torch.cat([u[:s], torch.addcmul(u[s:], c[s:], u[:-s])])
        c = torch.cat([c[:s], c[s:] * c[:-s]])
        s *= 2
    return u


def _coefficients(s):
    """(c with resets in it, c without, u) in 32 bits."""
    z, x = s["z"].float(), s["x"].float()
    if s["case"]["form"] == "sigmoid":
        f = torch.sigmoid(z)
        u = torch.sigmoid(-z) * x
    else:
        f, u = z, x
    c = f if s["reset"] is None else torch.where(s["reset"][..., None], torch.zeros_like(f), f)
    return c, f, u


def _plain_scan(s):
    c, _, u = _coefficients(s)
    u = torch.cat([(u[0] + c[0] * s["h0"])[None], u[1:]])
    h = _recur(c, u)
    return {"h": h.to(s["x"].dtype), "h_last": h[-1].clone()}


def _plain_scan_backward(s):
    c, f, _ = _coefficients(s)
    dt = s["x"].dtype
    dh = s["dh"].float()
    dh = torch.cat([dh[:-1], (dh[-1] + s["dh_last"])[None]])
    back = torch.cat([torch.zeros_like(c[:1]), c[1:].flip(0)])  # the factor from step t + 1
    e = _recur(back, dh.flip(0)).flip(0)
    before = torch.cat([s["h0"][None], s["h"][:-1].float()])
    if s["reset"] is not None:
        before = torch.where(s["reset"][..., None], torch.zeros_like(before), before)
    dh0 = c[0] * e[0]
    if s["case"]["form"] == "sigmoid":
        g = torch.sigmoid(-s["z"].float())
        return {"dz": (e * (before - s["x"].float()) * f * g).to(dt), "dx": (e * g).to(dt), "dh0": dh0}
    return {"dz": (e * before).to(dt), "dx": e.to(dt), "dh0": dh0}


def _plain_step(s):
    c, _, u = _coefficients(s)
    s["h"].copy_(c * s["h"] + u)
    return s["h"]


def _plain_linear(s):
    p = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        p = p + s["bias"].float()
    y = _act(s["case"]["act"], p)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_linear_backward(s):
    dt, dz = s["x"].dtype, s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _act_grad(s["case"]["act"], s["pre"].float())
    return {"dx": (dz @ s["w"].float()).to(dt), "dw": (dz.t() @ s["x"].float()).to(dt), "db": dz.sum(0).to(dt)}


def _newton_schulz(g):
    a, b, c = COEF
    x = g / ((g * g).sum((-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    for _ in range(STEPS):
        p = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * p + c * torch.matmul(p, p), x)
    return x.transpose(-2, -1).contiguous() if tall else x


def _plain_muon(s):
    w, g, m = s["w"], s["g"], s["m"]
    m.copy_(MOMENTUM * m + g)
    o = _newton_schulz(g + MOMENTUM * m)
    scale = math.sqrt(max(1.0, w.shape[-2] / w.shape[-1]))
    w.copy_(w * (1 - LR * DECAY) - LR * scale * o)
    return {"w": w, "m": m}


# ── the framework's operators ───────────────────────────────────────────────

_ops = []


def _handle():
    if not _ops:
        from phyz_amd.ops import Ops
        _ops.append(Ops(device=0))
    return _ops[0]


def _own(s):
    ops, c = _handle(), s["case"]
    if c["op"] == "scan_step":
        return ops.gated_step(s["z"], s["x"], s["h"], reset=s["reset"], form=c["form"])
    if c["op"] == "scan":
        h, last = ops.gated_scan(s["z"], s["x"], h0=s["h0"], reset=s["reset"], form=c["form"])
        return {"h": h, "h_last": last}
    if c["op"] == "scan_backward":
        dz, dx, dh0 = ops.gated_scan_backward(s["dh"], s["z"], s["x"], s["h"], h0=s["h0"], reset=s["reset"],
                                              dh_last=s["dh_last"], form=c["form"])
        return {"dz": dz, "dx": dx, "dh0": dh0}
    if c["op"] == "linear":
        return ops.linear(s["x"], s["w"], bias=s["bias"], act=c["act"], residual=s["residual"])
    if c["op"] == "linear_backward":
        dx, dw, db = ops.linear_backward(s["dy"], s["x"], s["w"], pre=s["pre"], act=c["act"])
        return {"dx": dx, "dw": dw, "db": db}
    if c["op"] == "orthogonalize":
        return ops.orthogonalize(s["g"], steps=STEPS, coef=COEF, eps=EPS)
    ops.muon_step(s["w"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS,
                  coef=COEF, eps=EPS)
    return {"w": s["w"], "m": s["m"]}


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    if op == "orthogonalize":
        return _newton_schulz(s["g"].float()).to(s["g"].dtype)
    return {"scan_step": _plain_step, "scan": _plain_scan, "scan_backward": _plain_scan_backward, "linear": _plain_linear,
            "linear_backward": _plain_linear_backward, "muon_step": _plain_muon}[op](s)


# ── what a pass cannot do without ───────────────────────────────────────────

def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "scan_step":
        n = case["worlds"] * case["width"]
        return {"bytes": n * (2 * e + 8) + (case["worlds"] if case["reset"] else 0), "flops": 4 * n}
    if op in ("scan", "scan_backward"):
        row = case["worlds"] * case["width"]
        n = case["steps"] * row
        mask = case["steps"] * case["worlds"] if case["reset"] else 0
        if op == "scan":
            return {"bytes": 3 * n * e + 2 * 4 * row + mask, "flops": 4 * n}
        reads = 4 if case["form"] == "sigmoid" else 3  # the decay form's gradients do not need x
        return {"bytes": (reads + 2) * n * e + 3 * 4 * row + mask, "flops": 8 * n}
    if op == "linear":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        return {"bytes": e * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)),
                "flops": 2 * m * n * k}
    if op == "linear_backward":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        return {"bytes": e * (m * n * (1 if case["act"] == "none" else 2) + 2 * m * k + 2 * n * k + n),
                "flops": 4 * m * n * k}
    q, m, n = case["batch"], min(case["n_out"], case["n_in"]), max(case["n_out"], case["n_in"])
    # A and A^2 are symmetric: half of their products is enough.
    flops = q * STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    return {"bytes": q * m * n * (2 * e if op == "orthogonalize" else 5 * 4), "flops": flops}


# ── 64 bits, from the definitions ───────────────────────────────────────────

def _exact_gate(case, z, x):
    """(c, 1 - c or None, u) of one step or of all."""
    if case["form"] == "sigmoid":
        c, g = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
        return c, g, g * x
    return z, None, x


def _exact_act(a, p):
    """(act, its derivative)."""
    one = torch.ones_like(p)
    if a == "tanh":
        return torch.tanh(p), 1 / torch.cosh(p) ** 2
    if a == "relu":
        return torch.where(p > 0, p, 0 * one), torch.where(p > 0, one, 0 * one)
    if a == "silu":
        d = 1 + torch.exp(-p)
        return p / d, (d + p * torch.exp(-p)) / d ** 2
    if a == "gelu":
        # 0.5 (1 + tanh(v)) = 1 / (1 + exp(-2 v))
        c = math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-2 * c * (p + 0.044715 * p ** 3)))
        return p * s, s + p * s * (1 - s) * 2 * c * (1 + 0.134145 * p ** 2)
    return p, one


def _exact_orthogonal(g):
    outs = []
    for x in g.double():
        x = x / (torch.linalg.matrix_norm(x) + EPS)
        for _ in range(STEPS):
            # On whichever side is shorter: p(X X^T) X = X p(X^T X).
            if x.shape[0] <= x.shape[1]:
                y = x @ x.T
                x = COEF[0] * x + COEF[1] * (y @ x) + COEF[2] * (y @ (y @ x))
            else:
                y = x.T @ x
                x = COEF[0] * x + COEF[1] * (x @ y) + COEF[2] * ((x @ y) @ y)
        outs.append(x)
    return torch.stack(outs)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    op = case["op"]
    keep = None if d.get("reset") is None else (~d["reset"]).double()[..., None]
    if op == "scan_step":
        c, _, u = _exact_gate(case, d["z"], d["x"])
        return c * (d["h"] if keep is None else d["h"] * keep) + u
    if op == "scan":
        h, out = d["h0"], torch.empty_like(d["x"], memory_format=torch.contiguous_format)
        for t in range(case["steps"]):
            c, _, u = _exact_gate(case, d["z"][t], d["x"][t])
            h = c * (h if keep is None else h * keep[t]) + u
            out[t] = h
        return {"h": out, "h_last": h}
    if op == "scan_backward":
        e = d["dh_last"]
        dz = torch.empty_like(d["x"], memory_format=torch.contiguous_format)
        dx = torch.empty_like(dz)
        for t in reversed(range(case["steps"])):
            c, g, _ = _exact_gate(case, d["z"][t], d["x"][t])
            e = e + d["dh"][t]
            before = d["h"][t - 1] if t else d["h0"]
            if keep is not None:
                before = before * keep[t]
            if g is None:
                dz[t], dx[t] = e * before, e
            else:
                dz[t], dx[t] = e * (before - d["x"][t]) * c * g, e * g
            e = c * e if keep is None else c * e * keep[t]
        return {"dz": dz, "dx": dx, "dh0": e}
    if op == "linear":
        p = torch.mm(d["x"], d["w"].T)
        if d["bias"] is not None:
            p += d["bias"]
        y = _exact_act(case["act"], p)[0]
        return y if d["residual"] is None else y + d["residual"]
    if op == "linear_backward":
        dz = d["dy"] if d["pre"] is None else d["dy"] * _exact_act(case["act"], d["pre"])[1]
        return {"dx": torch.mm(dz, d["w"]), "dw": torch.mm(dz.T, d["x"]), "db": dz.sum(0)}
    if op == "orthogonalize":
        return _exact_orthogonal(s["g"])
    m = MOMENTUM * d["m"] + d["g"]
    o = _exact_orthogonal(d["g"] + MOMENTUM * m)
    ratio = max(1.0, case["n_out"] / case["n_in"])
    return {"w": d["w"] * (1 - LR * DECAY) - LR * math.sqrt(ratio) * o, "m": m}
