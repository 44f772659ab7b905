"""The sequence operators in 64 bits on the CPU, with bounds on how far a
correct 32-bit implementation may be off, element by element.

Bounds follow the arithmetic. U is half the spacing of f32 (or of the stored
type) at 1. A recurrence's error obeys the recurrence itself: what a step adds
is a few U of the magnitudes it handles (a gate costs 2|z| + 16 of them: its
exponential's argument is off by |z| U), and the steps after it carry it on. A
dot product of length K is off by at most (K + 32) U of the products'
magnitudes.
"""
import math

import torch

U32, U_BF16 = 2.0 ** -24, 2.0 ** -8


def unit(dtype):
    return U_BF16 if dtype == torch.bfloat16 else U32


def d64(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def gate(z, form):
    """(c, the factor of x, the relative cost of both in U)."""
    if form == "sigmoid":
        return torch.sigmoid(z), torch.sigmoid(-z), 2 * z.abs() + 16
    return z, torch.ones_like(z), torch.full_like(z, 4.0)


def scan(z, x, h0, reset, form, dtype):
    """(h, h_last, bound of h, bound of h_last)."""
    z, x = d64(z), d64(x)
    T, B, D = x.shape
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else d64(h0)
    mag, err = h.abs(), torch.zeros(B, D, dtype=torch.float64)
    out, bound = torch.empty_like(x), torch.empty_like(x)
    for t in range(T):
        c, w, cost = gate(z[t], form)
        if reset is not None:
            r = reset[t].cpu().bool()[:, None]
            h, mag, err = (torch.where(r, 0.0, v) for v in (h, mag, err))
        h = c * h + w * x[t]
        mag = c.abs() * mag + w * x[t].abs()
        err = c.abs() * err + U32 * cost * mag
        out[t], bound[t] = h, err + (unit(dtype) * h.abs() if dtype != torch.float32 else 0)
    return out, h, bound, err


def scan_backward(dh, z, x, h, h0, reset, dh_last, form, dtype):
    """((dz, dx, dh0), their bounds), from the stored h."""
    dh, z, x, h = d64(dh), d64(z), d64(x), d64(h)
    T, B, D = x.shape
    zero = torch.zeros(B, D, dtype=torch.float64)
    k = zero if dh_last is None else d64(dh_last)
    first = zero if h0 is None else d64(h0)
    kmag, kerr = k.abs(), zero.clone()
    dz, dx, bz, bx = (torch.empty_like(x) for _ in range(4))
    rnd = unit(dtype) if dtype != torch.float32 else 0.0
    for t in reversed(range(T)):
        c, w, cost = gate(z[t], form)
        e, emag = dh[t] + k, dh[t].abs() + kmag
        eerr = kerr + 2 * U32 * emag
        hp = h[t - 1] if t else first
        r = None
        if reset is not None:
            r = reset[t].cpu().bool()[:, None]
            hp = torch.where(r, 0.0, hp)
        slope, away, far = (c * w, hp - x[t], hp.abs() + x[t].abs()) if form == "sigmoid" else (1.0, hp, hp.abs())
        dz[t], dx[t] = e * away * slope, e * w
        bz[t] = (eerr + U32 * 2 * cost * emag) * far * slope + rnd * dz[t].abs()
        bx[t] = (eerr + U32 * cost * emag) * w + rnd * dx[t].abs()
        k, kmag = c * e, c.abs() * emag
        kerr = c.abs() * eerr + U32 * cost * kmag
        if r is not None:
            k, kmag, kerr = (torch.where(r, 0.0, v) for v in (k, kmag, kerr))
    return (dz, dx, k), (bz, bx, kerr + 1e-30)


_G = math.sqrt(2 / math.pi)


def act(name, p):
    if name == "tanh":
        return torch.tanh(p)
    if name == "relu":
        return torch.relu(p)
    if name == "silu":
        return p * torch.sigmoid(p)
    if name == "gelu":
        return 0.5 * p * (1 + torch.tanh(_G * (p + 0.044715 * p ** 3)))
    return p


def act_grad(name, p):
    if name == "tanh":
        return 1 - torch.tanh(p) ** 2
    if name == "relu":
        return (p > 0).double()
    if name == "silu":
        s = torch.sigmoid(p)
        return s * (1 + p * (1 - s))
    if name == "gelu":
        y = torch.tanh(_G * (p + 0.044715 * p ** 3))
        return 0.5 * (1 + y) + 0.5 * p * (1 - y * y) * _G * (1 + 0.134145 * p ** 2)
    return torch.ones_like(p)


def linear(x, w, bias, residual, name, dtype):
    """(y, pre, bound of y, bound of pre)."""
    x, w = d64(x), d64(w)
    p, mag = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        p, mag = p + d64(bias), mag + d64(bias).abs()
    ep = (x.shape[1] + 32) * U32 * mag + 1e-37
    y = act(name, p)
    # Slopes are at most 1.13; an activation costs a few U and 2|p| of its gate.
    ey = 1.13 * ep + U32 * (4 * p.abs() + 16) * y.abs()
    if residual is not None:
        y = y + d64(residual)
        ey = ey + U32 * 2 * (y.abs() + d64(residual).abs())
    rnd = unit(dtype) if dtype != torch.float32 else 0.0
    return y, p, ey + rnd * y.abs() + 1e-37, ep + rnd * p.abs()


def linear_backward(dy, x, w, pre, name, dtype):
    """((dx, dw, db), their bounds)."""
    dy, x, w = d64(dy), d64(x), d64(w)
    m, n = dy.shape
    p = torch.zeros_like(dy) if pre is None else d64(pre)
    dz = dy * act_grad(name, p)
    # dz: the derivative's cost, 8 |p| + 32 of U (p itself multiplies a gate's
    # error), and bf16's rounding where the products take it in bf16.
    ez = U32 * (8 * p.abs() + 32) * dy.abs() if name != "none" else torch.zeros_like(dy)
    eb = ez.clone()
    if dtype != torch.float32 and name != "none":
        ez = ez + U_BF16 * dz.abs()
    rnd = unit(dtype) if dtype != torch.float32 else 0.0
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    bx = ez @ w.abs() + (n + 32) * U32 * (dz.abs() @ w.abs()) + rnd * dx.abs() + 1e-37
    bw = ez.T @ x.abs() + (m + 32) * U32 * (dz.abs().T @ x.abs()) + rnd * dw.abs() + 1e-37
    bb = eb.sum(0) + (m + 32) * U32 * dz.abs().sum(0) + rnd * db.abs() + 1e-37
    return (dx, dw, db), (bx, bw, bb)


COEF = (3.4445, -4.7750, 2.0315)


def orthogonalize(g, steps=5, coef=COEF, eps=1e-7):
    g = d64(g)
    x = g / (torch.sqrt((g * g).sum((-2, -1), keepdim=True)) + eps)
    for _ in range(steps):
        a = x @ x.transpose(-2, -1)
        x = coef[0] * x + (coef[1] * a + coef[2] * a @ a) @ x
    return x


def muon(w, g, m, lr, momentum, nesterov, weight_decay, **kw):
    w, g, m = d64(w), d64(g), d64(m)
    m = momentum * m + g
    o = orthogonalize(g + momentum * m if nesterov else m, **kw)
    return w * (1 - lr * weight_decay) - lr * math.sqrt(max(1.0, w.shape[-2] / w.shape[-1])) * o, m


def within(got, want, bound, what):
    """Every element within its bound, and not-finite where the reference is."""
    got = d64(got)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    if not want.numel():
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() / (bound + 1e-38)
    worst = float(over.max())
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"
