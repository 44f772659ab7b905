"""Linear attention, rotary positions and AdamW in 64 bits on the CPU, with bounds
on how far a correct 32-bit implementation may be off, element by element.

Linear attention and its four gradients are one recurrence,
    s <- a s + key val^T,  out = s^T read
over the steps in one direction. Each product key val is carried on by exp(the
sum of the gates since); a 32-bit implementation has that factor to (2 + |sum|) U
of itself (U = 2^-24), and adds at most N of such products and partial sums of
them one after the other, each addition U of the magnitudes. So beside the state
stand its magnitude, M <- a M + |key| |val|, and the same weighted by age,
A <- a (A + |g| M) + |key| |val|; the state is off by at most U (N M + 4 A).
In bf16 the products may take the state and the scores in two pieces, to 2^-16 of
themselves; results are rounded once.
"""
import math

import torch

U32, U_BF16 = 2.0 ** -24, 2.0 ** -8


def d64(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def split(x, n, heads):
    """[steps, worlds, heads, n] from [steps, worlds, own heads * n], repeated."""
    x = d64(x)
    own = x.shape[-1] // n
    return x.reshape(*x.shape[:-1], own, n).repeat_interleave(heads // own, -2)


def gates(g, reset):
    """(a, |g| where it carries on)."""
    g = d64(g)
    forget = g < -104
    if reset is not None:
        forget = forget | reset.cpu().bool()[..., None]
    return torch.where(forget, torch.zeros_like(g), torch.exp(g)), torch.where(forget, torch.zeros_like(g), g.abs())


def sweep(read, key, val, a, age, first, back=False):
    """(out, its bound in U of the products' errors, (s, M, A) after every step)."""
    T, B, H, n = key.shape
    m = val.shape[-1]
    s = torch.zeros(B, H, n, m, dtype=torch.float64) if first is None else first
    M, A = s.abs(), s.abs()
    out, mag, aged, states = (torch.empty(T, B, H, m, dtype=torch.float64) for _ in range(3)), None, None, []
    out, mag, aged = out
    for i in range(T):
        t = T - 1 - i if back else i
        tg = t + 1 if back else t
        if tg < T:
            f, x = a[tg][..., None, None], age[tg][..., None, None]
            # What a reset cuts off may be anything.
            s, M, A = (torch.where(f == 0, torch.zeros_like(v), f * v) for v in (s, M, A + x * M))
        kv = key[t][..., :, None] * val[t][..., None, :]
        s, M, A = s + kv, M + kv.abs(), A + kv.abs()
        r = read[t][..., None, :]
        out[t], mag[t], aged[t] = (r @ s)[..., 0, :], (r.abs() @ M)[..., 0, :], (r.abs() @ A)[..., 0, :]
        states.append((s, M, A))
    return out, (mag, aged), states


def _terms(steps, nk, nv):
    return nk + nv + 160 + steps // 16


def _bound(out, mags, scale, terms, dtype, pieces=True):
    mag, aged = mags
    b = abs(scale) * U32 * (terms * mag + 4 * aged)
    if dtype != torch.float32:
        b = b + (abs(scale) * 3 * 2.0 ** -16 * mag if pieces else 0) + U_BF16 * out.abs() * 1.01
    return b + 1e-37


def merge(x, own, summed=True):
    """[steps, worlds, own * n]: heads that share one summed."""
    T, B, H, n = x.shape
    return x.reshape(T, B, own, H // own, n).sum(3).reshape(T, B, own * n)


def attention(q, k, v, g, s0, reset, nk, nv, scale):
    """((o, s), bounds)."""
    H = g.shape[-1]
    dtype = q.dtype
    q, k, v = split(q, nk, H), split(k, nk, H), split(v, nv, H)
    a, age = gates(g, reset)
    out, mags, states = sweep(q, k, v, a, age, d64(s0))
    T, B = out.shape[:2]
    n = _terms(T, nk, nv)
    s, M, A = states[-1]
    o = scale * out
    return (o.reshape(T, B, -1), s), (_bound(o, mags, scale, n, dtype).reshape(T, B, -1), U32 * (n * M + 4 * A) + 1e-37)


def attention_backward(do, q, k, v, g, s0, reset, ds, nk, nv, scale):
    """((dq, dk, dv, dg, ds0), bounds)."""
    H, dtype = g.shape[-1], q.dtype
    own = q.shape[-1] // nk, k.shape[-1] // nk, v.shape[-1] // nv
    do, q, k, v = split(do, nv, H), split(q, nk, H), split(k, nk, H), split(v, nv, H)
    T, B = q.shape[:2]
    a, age = gates(g, reset)
    s0, ds = d64(s0), d64(ds)
    n = _terms(T, nk, nv)
    turned = lambda s: None if s is None else s.transpose(-1, -2)  # noqa: E731
    dq, mq, S = sweep(do, v, k, a, age, turned(s0))                      # states transposed
    dv, mv, E = sweep(k, scale * q, do, a, age, ds, back=True)
    dk, mk, _ = sweep(v, scale * do, q, a, age, turned(ds), back=True)
    E = E[::-1]
    dg, x = torch.empty_like(a), torch.empty_like(a)
    zero = torch.zeros(B, H, nv, nk, dtype=torch.float64)
    for t in range(T):
        s, M, A = S[t - 1] if t else ((zero,) * 3 if s0 is None else (turned(s0), turned(s0).abs(), turned(s0).abs()))
        e, Me, Ae = (turned(v_) for v_ in E[t])
        f = a[t]
        dg[t] = torch.where(f == 0, torch.zeros_like(f), f * (e * torch.where(f[..., None, None] == 0, zero, s)).sum((-1, -2)))
        x[t] = torch.where(f == 0, torch.zeros_like(f), f * (Me * (M * 1.0) + Me * A + Ae * M).sum((-1, -2)))
    # A gate's gradient may be found from its neighbours' in a chunk of steps, by
    # sums of their magnitudes.
    near = torch.nn.functional.max_pool1d(x.permute(1, 2, 0).reshape(B * H, 1, T), 129, 1, 64).reshape(B, H, T).permute(2, 0, 1)
    e, M, A = E[0]
    f, y = a[0][..., None, None], age[0][..., None, None]
    ds0 = torch.where(f == 0, torch.zeros_like(e), f * e)
    bs = U32 * (n * f * M + 4 * f * (A + y * M)) + 1e-37
    dq = scale * dq
    bq, bk, bv = _bound(dq, mq, scale, n, dtype), _bound(dk, mk, 1.0, n, dtype), _bound(dv, mv, 1.0, n, dtype)
    if dtype != torch.float32:  # sums over heads are rounded once
        bq, bk, bv = (b + U_BF16 * 0 for b in (bq, bk, bv))
    bg = U32 * (n + 64) * near + (3 * 2.0 ** -16 * near if dtype != torch.float32 else 0) + 1e-37
    return ((merge(dq, own[0]), merge(dk, own[1]), merge(dv, own[2]), dg, ds0),
            (merge(bq, own[0]), merge(bk, own[1]), merge(bv, own[2]), bg, bs))


def rotary(x, positions, freq, heads, layout, scale, inverse):
    """(y, bound): angles to 2^-52 of themselves and 2^-24 of a turn at the end, sine
    and cosine to 3 U, products and one sum."""
    dtype, x, f = x.dtype, d64(x), d64(freq)
    shape = x.shape
    x = x.reshape(*shape[:-1], heads, shape[-1] // heads)
    n = f.shape[0]
    angle = (positions.cpu().double()[..., None] * f)[..., None, :]
    c, s = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
    x0, x1 = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    y, b = x.clone(), torch.zeros_like(x)
    mag = abs(scale) * (x0.abs() + x1.abs())
    off = mag * (12 * U32 + 2.0 ** -50 * angle.abs()) + 1e-37
    for i, v in enumerate((scale * (x0 * c - x1 * s), scale * (x0 * s + x1 * c))):
        at = slice(i * n, (i + 1) * n) if layout == "half" else slice(i, 2 * n, 2)
        y[..., at] = v
        b[..., at] = off + (U_BF16 * 1.01 * v.abs() if dtype != torch.float32 else 0)
    return y.reshape(shape), b.reshape(shape)


def adamw(w, g, m, v, t, lr, betas, eps, weight_decay):
    """((w, m, v), bounds): a few roundings each."""
    dtype = w.dtype
    w, g, m, v = (d64(x) for x in (w, g, m, v))
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    bm = 3 * U32 * (b1 * m.abs() + (1 - b1) * g.abs()) + 1e-45
    bv = 4 * U32 * v1 + 1e-45
    step = lr * (m1 / (1 - b1 ** t)) / (torch.sqrt(v1 / (1 - b2 ** t)) + eps)
    # The step's own: what m is off by, half of what v is off by, and ten roundings.
    # A v below f32's range counts as 0 to within its smallest number.
    most = lr * ((m1.abs() + bm) / (1 - b1 ** t)) / (torch.sqrt((v1 - bv).clamp(min=0) / (1 - b2 ** t)) + eps)
    w1 = w * (1 - lr * weight_decay) - step
    bw = (most - step.abs()).abs() + 12 * U32 * most + 3 * U32 * w.abs() + 1e-45
    if dtype != torch.float32:
        bw = bw + U_BF16 * 1.01 * w1.abs()
    return (w1, m1, v1), (bw, bm, bv)


def mix(x):
    x = ((x ^ (x >> 16)) * 0xb504f335) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0xb7e15163) & 0xffffffff
    return x ^ (x >> 16)


def dither(seed, t, tensor, i):
    key = mix((mix((mix((t & 0xffffffff) ^ 0x9e3779b9) + seed) & 0xffffffff) + tensor * 0x243f6a89) & 0xffffffff)
    h = mix(((i * 0x9e3779b9) & 0xffffffff) ^ key)
    return ((h & 0xffff) * 16 + 8) / 2 ** 20, ((h >> 16) * 16 + 8) / 2 ** 20


def code_values(e, top, signed):
    """What every code stands for below a block's exponent e, as Python floats."""
    out = []
    for c in range(256):
        size = c & 127 if signed else c
        x, d = size >> 3, size & 7
        value = (8 + d) * 2.0 ** (e - top - 130 + x) if x else d * 2.0 ** (e - top - 129)
        out.append(-value if signed and c > 128 else value)
    out[128 if signed else 255] = math.nan
    return out


def encode(x, e, top, signed, r):
    """The code of one finite f32 value: rounded down or up between its neighbours,
    up where the part of the way that is above the lower one and r come to 1."""
    values = code_values(e, top, signed)
    size = abs(x)
    last = 127 if signed else 254
    low = max(c for c in range(last + 1) if values[c] <= size)
    if low == last:
        code = low
    else:
        part = (size - values[low]) / (values[low + 1] - values[low])
        # The part of the way is known to 20 bits.
        code = low + (math.floor(part * 2 ** 20) / 2 ** 20 + r >= 1.0)
    if signed:
        return code + 128 if x < 0 and code else code
    return max(code, 1) if size > 0 else 0


def within(got, want, bound, what):
    got = d64(got)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    if not want.numel():
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"
