"""Operators of attending policies and of their training, as measurable cases.

A policy's memory may be a matrix for each head instead of a vector: queries
read it, keys and values write it, and a gate of each head lets it fade. Over a
rollout that is linear attention with a decay, acting it is one step of it.
Queries and keys carry their position in the episode as a rotation. Such a
policy's parameters are many tensors of all sizes, and one AdamW step takes
them all.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) the tensors a program has in hand before the call
    run(state)          one pass: in plain torch, or (own) through phyz_amd.ops
    work(case)          bytes and operations a pass cannot do without
    exact(case, seed)   the pass from the operator's definition, 64 bits

Operators (a case's "op"):

    attend           S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t over
                     [steps, worlds, heads * size]; where `reset` is set, S_{t-1}
                     counts as 0. q, k and v may have fewer heads than g.
    attend_backward  its gradients for q, k, v, g and the first state
    attend_step      one step of it, the state updated in place
    rotary           the first `rot` elements of each head turned by its position,
                     in pairs (i, i + rot / 2) ("half") or (2i, 2i + 1)
                     ("interleaved"); the other way round for gradients
    adamw            one AdamW step over all tensors of a list, its two moments
                     held in 32 bits or in 8 with an exponent for each 256
"""
import math

import torch

own = False

CHUNK = 64
BLOCK = 256
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
BYTES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # One control step of an attending policy on a batch of worlds: every
        # head's state once through the chip.
        _attend("step_worlds", "attend_step", "f32", 1, 1024, 4, 64, 64, reset=True),
        # Serving a few sequences: launch latency and little else.
        _attend("step_serve", "attend_step", "bf16", 1, 8, 8, 128, 128),
        # Forward over a collector's rollout: 4096 worlds at the policy's hidden
        # width, episodes that end inside it.
        _attend("attend_rollout", "attend", "f32", 64, 4096, 4, 64, 64, reset=True),
        # One very long sequence: parallelism has to come from the steps.
        _attend("attend_long", "attend", "bf16", 32768, 1, 8, 128, 128),
        # Ragged sizes, batch-major tensors, queries and keys shared by all heads.
        _attend("attend_odd", "attend", "bf16", 1023, 61, 5, 40, 72, qh=1, kh=1, reset=True, batch_first=True),
        # The training pass over a rollout.
        _attend("backward_rollout", "attend_backward", "f32", 64, 2048, 4, 64, 64, reset=True),
        # The same where keys and values are shared by three heads each.
        _attend("backward_odd", "attend_backward", "bf16", 777, 37, 6, 48, 80, kh=2, vh=2, reset=True, batch_first=True),
        # Queries and keys of a rollout, both in one buffer.
        {"name": "rotary_rollout", "op": "rotary", "dtype": "bf16", "steps": 64, "worlds": 4096, "heads": 8, "size": 64,
         "rot": 64, "layout": "half", "inverse": False, "far": 1000, "stretch": 1.0},
        # One step of a batch of worlds far inside their episodes, half of each
        # head turned, positions stretched.
        {"name": "rotary_step", "op": "rotary", "dtype": "f32", "steps": 1, "worlds": 1024, "heads": 4, "size": 64,
         "rot": 32, "layout": "interleaved", "inverse": False, "far": 1000000, "stretch": 8.0},
        # The recurrent policy's eight tensors.
        {"name": "adamw_policy", "op": "adamw", "dtype": "f32", "grads": "f32", "bits": 32, "step": 100,
         "shapes": "256x55 256 512x256 512 256x256 256 8x256 8"},
        # Wide layers in bfloat16 products: f32 masters, bf16 gradients, moments
        # in 8 bits.
        {"name": "adamw_wide", "op": "adamw", "dtype": "f32", "grads": "bf16", "bits": 8, "step": 1000,
         "shapes": "8192x2048 8192 2048x8192 2048 8192x2048 8192 2048x8192 2048"},
        # Many tensors of odd sizes, first step.
        {"name": "adamw_many", "op": "adamw", "dtype": "f32", "grads": "f32", "bits": 32, "step": 0,
         "shapes": " ".join(f"{17 + 29 * i}x{5 + (37 * i) % 613} {17 + 29 * i}" for i in range(40))},
    ]


def _attend(name, op, dtype, steps, worlds, heads, size_k, size_v, qh=None, kh=None, vh=None, reset=False,
            batch_first=False):
    c = {"op": op, "dtype": dtype, "steps": steps, "worlds": worlds, "heads": heads, "size_k": size_k, "size_v": size_v,
         "q_heads": qh or heads, "k_heads": kh or heads, "v_heads": vh or heads, "reset": reset, "batch_first": batch_first}
    return {"name": name, **c} if name else c


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: any operator, sizes over the ranges of the listed ones."""
    op = rng.choice(("attend_step", "attend", "attend", "attend", "attend_backward", "attend_backward", "rotary", "rotary",
                     "adamw", "adamw"))
    dtype = rng.choice(("f32", "bf16"))
    if op.startswith("attend"):
        heads = rng.choice((1, 2, 3, 4, 5, 6, 8))
        shared = [h for h in range(1, heads + 1) if heads % h == 0]
        sizes = [rng.choice((rng.randint(8, 128), 32, 64, 128)) for _ in range(2)]
        most = 1 << (26 if op == "attend" else 24)  # elements of keys and values together
        steps = 1 if op == "attend_step" else _between(rng, 1, 32768)
        one = heads * sum(sizes)
        steps = min(steps, max(1, most // one))
        worlds = _between(rng, 1, max(1, min(4096, most // (steps * one))))
        qh, kh, vh = (heads if rng.random() < 0.7 else rng.choice(shared) for _ in range(3))
        return _attend(None, op, dtype, steps, worlds, heads, *sizes, qh=qh, kh=kh, vh=vh, reset=rng.random() < 0.5,
                       batch_first=rng.random() < 0.5)
    if op == "rotary":
        size = rng.choice((rng.randint(2, 128), 32, 64, 128))
        heads = rng.randint(1, 12)
        steps = _between(rng, 1, 4096)
        worlds = _between(rng, 1, max(1, min(4096, (1 << 27) // (steps * heads * size))))
        return {"op": op, "dtype": dtype, "steps": steps, "worlds": worlds, "heads": heads, "size": size,
                "rot": size // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, size // 2),
                "layout": rng.choice(("half", "interleaved")), "inverse": rng.random() < 0.4,
                "far": _between(rng, 10, 1 << 22), "stretch": rng.choice((1.0, 1.0, 2.0, 8.0))}
    bits = rng.choice((32, 8))
    count = _between(rng, 1, 48)
    shapes, left = [], 1 << 26
    for _ in range(count):
        m, n = _between(rng, 1, 8192), _between(rng, 1, 4096)
        if rng.random() < 0.4 or m * n > left:
            n = 1
        left -= m * n
        shapes.append(f"{m}x{n}" if n > 1 else f"{m}")
    return {"op": op, "dtype": dtype, "grads": rng.choice((dtype, "bf16")), "bits": bits, "step": rng.choice((0, 1, 100, 20000)),
            "shapes": " ".join(shapes)}


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen) * scale


def _frequencies(case):
    """Radians a position for each pair. Stretched, the slow pairs' (those that
    turn less than once in 1024 positions) are divided by the factor, the fast
    ones' (32 times or more) kept, those between blended; in 64 bits."""
    n = case["rot"] // 2
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    if case["stretch"] != 1.0:
        keep = ((f * 1024 / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * (keep + (1 - keep) / case["stretch"])
    return f


def _sizes(case):
    """[(shape, elements, offset)] of a list of tensors in one buffer, each at a
    multiple of 64 elements."""
    out, at = [], 0
    for s in case["shapes"].split():
        shape = tuple(int(v) for v in s.split("x"))
        n = math.prod(shape)
        out.append((shape, n, at))
        at += -(-n // 64) * 64
    return out, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op.startswith("attend"):
        dt = _dtype(case["dtype"])
        t, b, h, dk, dv = (case[k] for k in ("steps", "worlds", "heads", "size_k", "size_v"))

        def lay(v):  # [steps, worlds, ...]; batch-major tensors are strided views
            return v.transpose(0, 1) if case["batch_first"] else v

        one = (b, t) if case["batch_first"] else (t, b)
        s.update(q=lay(_normal(gen, *one, case["q_heads"] * dk).to(dt)),
                 k=lay(_normal(gen, *one, case["k_heads"] * dk, scale=dk ** -0.5).to(dt)),
                 v=lay(_normal(gen, *one, case["v_heads"] * dv).to(dt)),
                 # Learned gates, of memories from a few steps to some hundreds.
                 g=lay(torch.nn.functional.logsigmoid(_normal(gen, *one, h) * 1.5 + 3.0)),
                 s0=_normal(gen, b, h, dk, dv, scale=0.5),
                 reset=lay(torch.rand(*one, device="cuda", generator=gen) < 0.01) if case["reset"] else None)
        if op == "attend_backward":
            s.update(do=lay(_normal(gen, *one, h * dv, scale=0.1).to(dt)), ds=_normal(gen, b, h, dk, dv, scale=0.05))
        if op == "attend_step":
            for k in ("q", "k", "v", "g", "reset"):
                s[k] = None if s[k] is None else s[k][0]
    elif op == "rotary":
        t, b, h, d = (case[k] for k in ("steps", "worlds", "heads", "size"))
        s["x"] = _normal(gen, t, b, h * d).to(_dtype(case["dtype"]))
        # Each world somewhere in its episode, and a step further at each step.
        first = torch.randint(0, case["far"], (b,), device="cuda", generator=gen)
        s["positions"] = first + torch.arange(t, device="cuda")[:, None]
        s["freq"] = _frequencies(case).cuda()
        # What a stretched rotation is scaled by.
        s["scale"] = 0.1 * math.log(case["stretch"]) + 1.0
    else:
        sizes, n = _sizes(case)
        # Weights and gradients of all scales, one a tensor.
        sc = torch.exp(_normal(gen, len(sizes)))
        w, g = _normal(gen, n, scale=0.05), _normal(gen, n, scale=1e-3)
        m, v = _normal(gen, n, scale=3e-4), _normal(gen, n, scale=1e-3).square()
        if case["step"] == 0:
            m, v = torch.zeros_like(m), torch.zeros_like(v)
        for (_, k, at), f in zip(sizes, sc.tolist()):
            for x, y in ((g, f), (m, f), (v, f * f)):
                x[at:at + k] *= y
        s.update(w=w.to(_dtype(case["dtype"])), g=g.to(_dtype(case["grads"])), seed=seed & 0xffff,
                 step=torch.full((1,), case["step"], dtype=torch.int64, device="cuda"))
        cut = lambda x: [x[at:at + k].view(shape) for shape, k, at in sizes]  # noqa: E731
        if case["bits"] == 32:
            s.update(m=m, v=v)
        else:
            # Moments as a program holds them after some steps.
            s.update(m=torch.zeros(n, dtype=torch.uint8, device="cuda"), v=torch.zeros(n, dtype=torch.uint8, device="cuda"),
                     exponents=[torch.zeros(2, -(-k // BLOCK), dtype=torch.uint8, device="cuda") for _, k, _ in sizes],
                     m_values=torch.zeros(n, dtype=torch.bfloat16, device="cuda"),
                     v_values=torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
            for (_, k, at), e in zip(sizes, s["exponents"]):
                half = torch.zeros(k, dtype=torch.int64, device="cuda") + (1 << 19)
                s["m"][at:at + k], e[0] = _encode(m[at:at + k], half, 14, True)
                s["v"][at:at + k], e[1] = _encode(v[at:at + k], half, 30, False)
            s.update(ms=cut(s["m_values"]), vs=cut(s["v_values"]))
        s.update(lists=[cut(s[k]) for k in ("w", "g", "m", "v")])
    return s


# ── the plain form: elementary torch operations in 32 bits ──────────────────

def _recur(c, u):
    """h_t = c_t h_{t-1} + u_t along the first axis, by doubling."""
    s = 1
    while s < u.shape[0]:
        u = torch.cat([u[:s], torch.addcmul(u[s:], c[s:], u[:-s])])
        c = torch.cat([c[:s], c[s:] * c[:-s]])
        s *= 2
    return u


def _chunks(x, heads, of):
    """[chunks, worlds, of, CHUNK, size] in 32 bits of [steps, worlds, heads * size],
    heads repeated to `of`, steps that are missing 0."""
    t, b, w = x.shape
    n = -(-t // CHUNK)
    y = torch.zeros(n * CHUNK, b, w, dtype=torch.float32, device=x.device)
    y[:t] = x
    y = y.view(n, CHUNK, b, heads, w // heads).permute(0, 2, 3, 1, 4)
    return y.repeat_interleave(of // heads, 2).contiguous()


def _merge(y, heads, like):
    """The other way: [steps, worlds, heads * size] in the type of `like`, repeated
    heads summed."""
    n, b, of, c, d = y.shape
    y = y.view(n, b, heads, of // heads, c, d).sum(3)
    y = y.permute(0, 3, 1, 2, 4).reshape(n * c, b, heads * d)[:like.shape[0]]
    return y.to(like.dtype)


def _decays(s):
    """Within each chunk: the decay from step to step [.., t, s], from its start, to
    its end, and over all of it. Sums of logarithms in 64 bits, as differences of
    long ones are taken."""
    c = s["case"]
    t, b, h = s["g"].shape
    n = -(-t // CHUNK)
    g = torch.zeros(n * CHUNK, b, h, dtype=torch.float64, device="cuda")
    g[:t] = s["g"]
    g = g.view(n, CHUNK, b, h).permute(0, 2, 3, 1).cumsum(-1)
    part = torch.zeros(n * CHUNK, b, dtype=torch.int64, device="cuda")
    if c["reset"]:
        part[:t] = s["reset"]
    part = part.view(n, CHUNK, b).permute(0, 2, 1).cumsum(-1)[:, :, None]
    zero = torch.zeros((), device="cuda")
    within = (g[..., :, None] - g[..., None, :]).float().exp()
    i = torch.arange(CHUNK, device="cuda")
    within = torch.where((part[..., :, None] == part[..., None, :]) & (i[:, None] >= i), within, zero)
    start = torch.where(part == 0, g.float().exp(), zero)
    end = torch.where(part == part[..., -1:], (g[..., -1:] - g).float().exp(), zero)
    return within, start, end, start[..., -1]


def _states(total, add, first):
    """The state before each chunk, and after the last."""
    total = total[..., None, None]
    add = torch.cat([(add[0] + total[0] * first)[None], add[1:]])
    after = _recur(total.expand_as(add).contiguous(), add)
    return torch.cat([first[None], after[:-1]]), after[-1].clone()


def _plain_attend(s):
    c = s["case"]
    h, scale = c["heads"], c["size_k"] ** -0.5
    q, k, v = (_chunks(s[x], c[x + "_heads"], h) for x in "qkv")
    within, start, end, total = _decays(s)
    add = torch.matmul((k * end[..., None]).transpose(-1, -2).contiguous(), v)
    before, last = _states(total, add, s["s0"])
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * within, v)
    o = scale * (o + start[..., None] * torch.matmul(q, before))
    return {"o": _merge(o, h, s["v"]), "s": last}


def _plain_attend_backward(s):
    c = s["case"]
    h, scale = c["heads"], c["size_k"] ** -0.5
    q, k, v = (_chunks(s[x], c[x + "_heads"], h) for x in "qkv")
    do = _chunks(s["do"], h, h) * scale
    within, start, end, total = _decays(s)
    turned = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    before, _ = _states(total, torch.matmul(turned(k * end[..., None]), v), s["s0"])
    add = torch.matmul(turned(q * start[..., None]), do)
    after, ds0 = _states(total.flip(0), add.flip(0), s["ds"])
    after = after.flip(0)  # the loss's gradient for the state after each chunk
    a = torch.matmul(q, turned(k)) * within
    w = torch.matmul(do, turned(v))
    da = w * within
    q_far = start[..., None] * torch.matmul(do, turned(before))
    k_far = end[..., None] * torch.matmul(v, turned(after))
    dq = torch.matmul(da, k) + q_far
    dk = torch.matmul(turned(da), q) + k_far
    dv = torch.matmul(turned(a), do) + end[..., None] * torch.matmul(k, after)
    # A gate at t is on the way from each step before it to each step from it on.
    ways = torch.tril(a * w, -1)
    ways = (ways.flip(-2).cumsum(-2).flip(-2).cumsum(-1) - ways.flip(-2).cumsum(-2).flip(-2)).diagonal(dim1=-2, dim2=-1)
    dg = ways + (q * q_far).sum(-1).flip(-1).cumsum(-1).flip(-1)
    kf = (k * k_far).sum(-1)
    dg = dg + kf.cumsum(-1) - kf + (total * (before * after).sum((-1, -2)))[..., None]
    t = s["g"].shape[0]
    dg = dg.permute(0, 3, 1, 2).reshape(-1, c["worlds"], h)[:t].contiguous()
    return {"dq": _merge(dq, c["q_heads"], s["q"]), "dk": _merge(dk, c["k_heads"], s["k"]),
            "dv": _merge(dv, c["v_heads"], s["v"]), "dg": dg, "ds0": ds0}


def _plain_attend_step(s):
    c = s["case"]
    b, h = c["worlds"], c["heads"]
    q, k, v = (s[x].float().view(b, c[x + "_heads"], -1).repeat_interleave(h // c[x + "_heads"], 1) for x in "qkv")
    a = s["g"].exp()
    if s["reset"] is not None:
        a = torch.where(s["reset"][:, None], torch.zeros_like(a), a)
    s["s0"].copy_(a[..., None, None] * s["s0"] + k[..., None] * v[..., None, :])
    o = (q[..., None] * s["s0"]).sum(-2) * c["size_k"] ** -0.5
    return {"o": o.reshape(b, -1).to(s["v"].dtype), "s": s["s0"]}


def _plain_rotary(s):
    c = s["case"]
    t, b, h, d, r = (c[k] for k in ("steps", "worlds", "heads", "size", "rot"))
    x = s["x"].view(t, b, h, d).float()
    # Angles in 64 bits: a far position's is thousands of turns.
    angle = (s["positions"].double()[..., None] * s["freq"])[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if c["inverse"]:
        sin = -sin
    turn = x[..., :r]
    if c["layout"] == "half":
        x0, x1 = turn[..., :r // 2], turn[..., r // 2:]
    else:
        x0, x1 = turn[..., 0::2], turn[..., 1::2]
    y0, y1 = (x0 * cos - x1 * sin) * s["scale"], (x0 * sin + x1 * cos) * s["scale"]
    y = torch.cat([y0, y1], -1) if c["layout"] == "half" else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1).view(t, b, h * d).to(s["x"].dtype)


_LOW = 0xffffffff


def _mix(x):
    """32 bits to 32 bits, each of the result's depending on all of them."""
    x = ((x ^ (x >> 16)) * 0xb504f335) & _LOW
    x = ((x ^ (x >> 15)) * 0xb7e15163) & _LOW
    return x ^ (x >> 16)


def _dither(seed, step, tensor, n):
    """Random bits of a tensor's elements: (20 bits for m, 20 for v)."""
    key = _mix((_mix((step & _LOW) ^ 0x9e3779b9) + seed) & _LOW)  # a tensor: the step is on the device
    key = _mix((key + tensor * 0x243f6a89) & _LOW)
    h = _mix((torch.arange(n, device="cuda") * 0x9e3779b9 & _LOW) ^ key)
    return (h & 0xffff) * 16 + 8, (h >> 16) * 16 + 8


def _encode(x, dither, top, signed):
    """(codes, a block's exponent): x in blocks of 256 as numbers of four digits
    (three beside the leading one) and an exponent of its own below the block's,
    rounded up where the digits cut off and the dither carry. The block's exponent
    is that of its largest element, at code exponent `top`; the smallest numbers
    share one exponent. 0x80 (signed) or 0xff stands for what is not finite; what
    is positive and unsigned does not become 0."""
    n = x.numel()
    size = x.abs()
    bits = size.view(torch.int32).long()
    fine = bits < 0x7f800000
    padded = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.int64, device="cuda")
    padded[:n] = torch.where(fine, bits, 0)
    block = torch.clamp(padded.view(-1, BLOCK).amax(1) >> 23, min=40)
    e = block.repeat_interleave(BLOCK)[:n]
    normal = ((bits + dither) >> 20) - ((e - top) << 3)
    # Below: whole multiples of the least step, 2^(e - top - 2 - 127).
    unit = ((129 + top - e + 20 + 1023) << 52).view(torch.float64)
    small = ((torch.where(fine, size, 0.0).double() * unit).long() + dither) >> 20
    code = torch.where((bits >> 23) - e + top >= 1, normal, small)
    if signed:
        code = torch.where(fine, code + 128 * ((x < 0) & (code > 0)), 0x80)
    else:
        code = torch.where(fine, torch.where(bits > 0, code.clamp(min=1), 0), 0xff)
    return code.to(torch.uint8), block.to(torch.uint8)


def _decode(code, block, top, signed):
    n = code.numel()
    e = block.long().repeat_interleave(BLOCK)[:n]
    c = code.long()
    bad = c == (0x80 if signed else 0xff)
    size = c & 0x7f if signed else c
    exp = size >> 3
    digits = torch.where(exp > 0, 8 + (size & 7), size).float()
    value = digits * ((e - top + torch.clamp(exp, min=1) - 3) << 23).int().view(torch.float32)
    if signed:
        value = torch.where(c > 128, -value, value)
    return torch.where(bad, torch.full_like(value, math.nan), value)


def _plain_adamw(s):
    c = s["case"]
    b1, b2 = BETAS
    s["step"] += 1
    t = s["step"].double()
    fix1, fix2 = (1 - b1 ** t).float(), (1 - b2 ** t).float()
    out = s if c["bits"] == 32 else {"m": s["m_values"], "v": s["v_values"]}
    step = s["step"]
    for i, (_, n, at) in enumerate(_sizes(c)[0]):
        w, g = s["w"][at:at + n], s["g"][at:at + n].float()
        if c["bits"] == 32:
            m, v = s["m"][at:at + n], s["v"][at:at + n]
        else:
            e = s["exponents"][i]
            m, v = _decode(s["m"][at:at + n], e[0], 14, True), _decode(s["v"][at:at + n], e[1], 30, False)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        w.copy_(w.float() * (1 - LR * DECAY) - (m / fix1) * LR / ((v / fix2).sqrt() + EPS))
        if c["bits"] == 32:
            s["m"][at:at + n], s["v"][at:at + n] = m, v
        else:
            dm, dv = _dither(s["seed"], step, i, n)
            s["m"][at:at + n], e[0] = _encode(m, dm, 14, True)
            s["v"][at:at + n], e[1] = _encode(v, dv, 30, False)
            out["m"][at:at + n] = _decode(s["m"][at:at + n], e[0], 14, True)
            out["v"][at:at + n] = _decode(s["v"][at:at + n], e[1], 30, False)
    return {"w": s["w"], "m": out["m"], "v": out["v"], "step": s["step"]}


# ── the framework's operators ───────────────────────────────────────────────

_ops = []


def _handle():
    if not _ops:
        from phyz_amd.ops import Ops
        _ops.append(Ops(device=0))
    return _ops[0]


def _own(s):
    ops, c = _handle(), s["case"]
    if c["op"].startswith("attend"):
        sizes = {"size_k": c["size_k"], "size_v": c["size_v"], "scale": c["size_k"] ** -0.5, "reset": s["reset"]}
        if c["op"] == "attend_step":
            return {"o": ops.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["s0"], **sizes), "s": s["s0"]}
        if c["op"] == "attend":
            o, last = ops.linear_attention(s["q"], s["k"], s["v"], s["g"], s0=s["s0"], **sizes)
            return {"o": o, "s": last}
        dq, dk, dv, dg, ds0 = ops.linear_attention_backward(s["do"], s["q"], s["k"], s["v"], s["g"], s0=s["s0"], ds=s["ds"], **sizes)
        return {"dq": dq, "dk": dk, "dv": dv, "dg": dg, "ds0": ds0}
    if c["op"] == "rotary":
        return ops.rotary(s["x"], s["positions"], s["freq"], heads=c["heads"], layout=c["layout"], scale=s["scale"],
                          inverse=c["inverse"])
    w, g, m, v = s["lists"]
    more = {"lr": LR, "betas": BETAS, "eps": EPS, "weight_decay": DECAY, "seed": s["seed"]}
    if c["bits"] == 32:
        ops.adamw_step(w, g, m, v, s["step"], **more)
        return {"w": s["w"], "m": s["m"], "v": s["v"], "step": s["step"]}
    ops.adamw_step(w, g, m, v, s["step"], exponents=s["exponents"], **more)
    ops.adamw_values(m, v, s["exponents"], out=(s["ms"], s["vs"]))
    return {"w": s["w"], "m": s["m_values"], "v": s["v_values"], "step": s["step"]}


def run(s):
    if own:
        return _own(s)
    return {"attend": _plain_attend, "attend_backward": _plain_attend_backward, "attend_step": _plain_attend_step,
            "rotary": _plain_rotary, "adamw": _plain_adamw}[s["case"]["op"]](s)


# ── what a pass cannot do without ───────────────────────────────────────────

def work(case):
    op = case["op"]
    if op.startswith("attend"):
        e = BYTES[case["dtype"]]
        t, b, h, dk, dv = (case[k] for k in ("steps", "worlds", "heads", "size_k", "size_v"))
        rows, states = t * b, 4 * b * h * dk * dv
        q, k, v = case["q_heads"] * dk, case["k_heads"] * dk, case["v_heads"] * dv
        mask = rows if case["reset"] else 0
        if op == "attend_backward":
            return {"bytes": rows * (e * (2 * (q + k + v) + h * dv) + 2 * 4 * h) + mask + 3 * states,
                    "flops": rows * h * dk * dv * 14}
        return {"bytes": rows * (e * (q + k + v + h * dv) + 4 * h) + mask + 2 * states, "flops": rows * h * dk * dv * 5}
    if op == "rotary":
        rows, r = case["steps"] * case["worlds"], case["rot"]
        return {"bytes": rows * (2 * BYTES[case["dtype"]] * case["heads"] * case["size"] + 8) + 4 * r,
                "flops": rows * case["heads"] * r * 4}
    n = sum(k for _, k, _ in _sizes(case)[0])
    # 8 bits: the moments read and written, and their values written.
    state = 16 if case["bits"] == 32 else 4 + 4
    return {"bytes": n * (2 * BYTES[case["dtype"]] + BYTES[case["grads"]] + state), "flops": 15 * n}


# ── 64 bits, from the definitions ───────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    wide = lambda v: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v  # noqa: E731
    if op == "rotary":
        t, b, h, d, r = (case[k] for k in ("steps", "worlds", "heads", "size", "rot"))
        x = s["x"].double().view(t * b, h, d)
        turn = torch.exp(1j * (-1.0 if case["inverse"] else 1.0) * s["positions"].double().view(-1, 1) * s["freq"])
        if case["layout"] == "half":
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn[:, None] * s["scale"]
            return torch.cat([z.real, z.imag, x[..., r:]], -1).view(t, b, h * d)
        z = torch.view_as_complex(x[..., :r].contiguous().view(t * b, h, r // 2, 2)) * turn[:, None] * s["scale"]
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1).view(t, b, h * d)
    if op == "adamw":
        b1, b2 = BETAS
        w, g = s["w"].double(), s["g"].double()
        if case["bits"] == 32:
            m, v = s["m"].double(), s["v"].double()
        else:
            m, v = torch.zeros_like(w), torch.zeros_like(w)
            for (_, n, at), e in zip(_sizes(case)[0], s["exponents"]):
                m[at:at + n] = _decode(s["m"][at:at + n], e[0], 14, True)
                v[at:at + n] = _decode(s["v"][at:at + n], e[1], 30, False)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        n = case["step"] + 1
        w1 = w - LR * DECAY * w - LR * (m / (1 - b1 ** n)) / (torch.sqrt(v / (1 - b2 ** n)) + EPS)
        for (_, k, at), (_, _, then) in zip(_sizes(case)[0], _sizes(case)[0][1:] + [(0, 0, w.numel())]):
            for x, y in ((w1, w), (m, s["m"]), (v, s["v"])):
                x[at + k:then] = y[at + k:then]  # between the tensors
        # What 8 bits hold goes by the rounding's own bits.
        return {"w": w1, "m": m if case["bits"] == 32 else None, "v": v if case["bits"] == 32 else None, "step": s["step"] + 1}
    t, b, h, dk, dv = (case[k] for k in ("steps", "worlds", "heads", "size_k", "size_v"))
    if op == "attend_step":
        for k in ("q", "k", "v", "g", "reset"):
            s[k] = None if s[k] is None else s[k][None]
    d = {k: wide(v) for k, v in s.items()}
    q, k, v = (d[x].reshape(t, b, case[x + "_heads"], -1).repeat_interleave(h // case[x + "_heads"], 2) for x in "qkv")
    keep = torch.exp(d["g"])
    if d["reset"] is not None:
        keep = keep * (~d["reset"]).double()[..., None]
    state, scale = d["s0"], dk ** -0.5
    if op != "attend_backward":
        out = torch.empty(t, b, h, dv, dtype=torch.float64, device="cuda")
        for i in range(t):
            state = keep[i][..., None, None] * state + k[i][..., :, None] * v[i][..., None, :]
            out[i] = scale * (q[i][..., None, :] @ state)[..., 0, :]
        return {"o": out.view(t, b, h * dv)[0] if op == "attend_step" else out.view(t, b, h * dv), "s": state}
    do = d["do"].reshape(t, b, h, dv)
    dq, dkk, dvv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for i in range(t):
        state = keep[i][..., None, None] * state + k[i][..., :, None] * v[i][..., None, :]
        dq[i] = scale * (state @ do[i][..., None])[..., 0]
    # <E_t, S_t> = q_t dq_t + dg_{t+1} = dg_t + k_t dk_t, E_t the loss's gradient for S_t
    grad, later, dg = d["ds"], (d["ds"] * state).sum((-1, -2)), torch.empty_like(keep)
    for i in reversed(range(t)):
        grad = grad + scale * q[i][..., :, None] * do[i][..., None, :]
        dkk[i] = (grad @ v[i][..., None])[..., 0]
        dvv[i] = (k[i][..., None, :] @ grad)[..., 0, :]
        later = (later + (q[i] * dq[i]).sum(-1) - (k[i] * dkk[i]).sum(-1)) * (keep[i] != 0).double()
        dg[i] = later
        grad = keep[i][..., None, None] * grad

    def total(x, name):
        n = case[name + "_heads"]
        return x.view(t, b, n, h // n, -1).sum(3).view(t, b, -1)

    return {"dq": total(dq, "q"), "dk": total(dkk, "k"), "dv": total(dvv, "v"), "dg": dg, "ds0": grad}
