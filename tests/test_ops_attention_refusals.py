"""What linear attention, rotary positions and AdamW refuse, on a handle without a
GPU, and their 64-bit references against autograd and plain rounding."""
import ctypes as C

import pytest
import torch

from phyz_amd import _lib
from phyz_amd.ops import Ops, OpsError, rotary_frequencies
from tests import attend_ref as R

F32, BF16, F64, I64, U8 = torch.float32, torch.bfloat16, torch.float64, torch.int64, torch.uint8


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


def attend(o, q=(6, 2, 12), k=(6, 2, 12), v=(6, 2, 15), g=(6, 2, 3), **kw):
    put = lambda x: t(*x) if isinstance(x, tuple) else x  # noqa: E731
    return o.linear_attention(put(q), put(k), put(v), put(g), **kw)


def back(o, do=(6, 2, 15), **kw):
    return o.linear_attention_backward(t(*do), t(6, 2, 12), t(6, 2, 12), t(6, 2, 15), t(6, 2, 3), **kw)


def step(o, s, **kw):
    return o.linear_attention_step(t(2, 12), t(2, 12), t(2, 15), t(2, 3), s, **kw)


def adamw(o, w=None, g=None, m=None, v=None, s=None, **kw):
    one = lambda x: [t(5)] if x is None else x  # noqa: E731
    return o.adamw_step(one(w), one(g), one(m), one(v), t(1, dtype=I64) if s is None else s, **kw)


def rot(o, x=None, p=None, f=None, **kw):
    return o.rotary(t(4, 2, 12) if x is None else x, t(4, 2, dtype=I64) if p is None else p, t(2, dtype=F64) if f is None else f, **kw)


def test_valid_calls_reach_the_device_check(ops):
    x = t(4, 2, 12)
    for call in (lambda: attend(ops, s0=t(2, 3, 4, 5), reset=t(6, 2, dtype=torch.bool)),
                 lambda: attend(ops, g=t(3)), lambda: attend(ops, q=t(6, 2, 4), v=t(6, 2, 5), size_k=4, size_v=5),
                 lambda: attend(ops, q=t(2, 6, 12).transpose(0, 1)), lambda: attend(ops, out=(t(6, 2, 15), None)),
                 lambda: back(ops, ds=t(2, 3, 4, 5), need_dg=False), lambda: step(ops, t(2, 3, 4, 5)),
                 lambda: step(ops, t(2, 3, 4, 5), reset=t(2, dtype=U8), out=t(2, 15)),
                 lambda: rot(ops, heads=3), lambda: rot(ops, x=x, out=x), lambda: rot(ops, p=t(4, 2, dtype=torch.int32)),
                 lambda: rot(ops, x=t(4, 12), p=t(4, dtype=I64)), lambda: adamw(ops), lambda: adamw(ops, [], [], [], []),
                 lambda: adamw(ops, [t(2, 3), t(4, dtype=BF16)], [t(2, 3, dtype=BF16), t(4)], [t(6), t(4)], [t(3, 2), t(4)]),
                 lambda: adamw(ops, m=[t(5, dtype=U8)], v=[t(5, dtype=U8)], exponents=[t(2, 1, dtype=U8)]),
                 lambda: ops.adamw_values([t(5, dtype=U8)], [t(5, dtype=U8)], [t(2, 1, dtype=U8)])):
        with pytest.raises(OpsError, match="host-only"):
            call()


@pytest.mark.parametrize("call, message", [
    (lambda o: attend(o, q=(6, 12)), "q has 2 dimensions, expected 3"),
    (lambda o: attend(o, q=t(6, 2, 12, dtype=F64)), "q is f64, expected f32 or bf16"),
    (lambda o: attend(o, q=t(6, 2, 12, dtype=torch.int32)), "q is i32, expected f32 or bf16"),
    (lambda o: attend(o, k=t(6, 2, 12, dtype=BF16)), "k is bf16, expected f32"),
    (lambda o: attend(o, k=(5, 2, 12)), "k has 5 elements along axis 0, expected 6"),
    (lambda o: attend(o, k=(6, 2, 8)), "k has 8 elements along axis 2: heads of 4, as many as g's 3 or a divisor"),
    (lambda o: attend(o, v=(6, 2, 0), size_v=5), "v has 0 elements along axis 2"),
    (lambda o: attend(o, v=(6, 2, 16)), "v has 16 elements along axis 2: heads of 5"),
    (lambda o: attend(o, q=t(6, 12, 2).transpose(1, 2)), "q: the last axis has to be dense"),
    (lambda o: attend(o, g=t(6, 2, 3, dtype=BF16)), "g is bf16, expected f32"),
    (lambda o: attend(o, g=(6, 3, 3)), "g has 3 elements along axis 1, expected 2"),
    (lambda o: attend(o, g=(6, 2, 0)), "g has no heads"),
    (lambda o: attend(o, q=(6, 2, 387)), "size_k and size_v have to be 1 to 128, not 129 and 5"),
    (lambda o: attend(o, size_v=0), "size_k and size_v have to be 1 to 128"),
    (lambda o: attend(o, scale=float("nan")), "scale has to be finite"),
    (lambda o: attend(o, s0=t(2, 3, 5, 4)), "s0 has 5 elements along axis 2, expected 4"),
    (lambda o: attend(o, s0=t(2, 3, 20)), "s0 has to be a tensor"),
    (lambda o: attend(o, s0=t(2, 3, 5, 4).transpose(2, 3)), "s0: each head's state has to be dense"),
    (lambda o: attend(o, s0=t(3, 3, 4, 5)), "s0 has 3 elements along axis 0, expected 2"),
    (lambda o: attend(o, s0=t(2, 3, 4, 5, dtype=BF16)), "s0 is bf16, expected f32"),
    (lambda o: attend(o, reset=t(2, 6, dtype=U8)), "reset has 2 elements along axis 0"),
    (lambda o: attend(o, reset=t(6, 2)), "reset is f32, expected u8"),
    (lambda o: attend(o, out=(t(6, 2, 14), None)), "o has 14 elements along axis 2, expected 15"),
    (lambda o: attend(o, out=(t(6, 1, 15).expand(6, 2, 15), None)), "o is broadcast"),
    (lambda o: attend(o, q=7), "q has to be a torch tensor"),
    (lambda o: back(o, do=(6, 2, 14)), "do has 14 elements along axis 2, expected 15"),
    (lambda o: back(o, ds=t(2, 3, 4, 4)), "ds has 4 elements along axis 3, expected 5"),
    (lambda o: back(o, out=(t(6, 2, 12), t(6, 2, 4), t(6, 2, 15), None, None)), "dk has 4 elements along axis 2, expected 12"),
    (lambda o: back(o, out=(t(6, 2, 12), t(6, 2, 12), t(6, 2, 15), t(6, 2, 1).expand(6, 2, 3), None)), "dg is broadcast"),
    (lambda o: step(o, t(2, 3, 4, 4)), "s has 4 elements along axis 3, expected 5"),
    (lambda o: step(o, None), "s has to be a torch tensor"),
    (lambda o: step(o, t(1, 3, 4, 5).expand(2, 3, 4, 5)), "s is broadcast"),
    (lambda o: rot(o, layout="whole"), "unknown layout 'whole'"),
    (lambda o: rot(o, heads=5), "x has 12 elements along axis 2, not 5 heads"),
    (lambda o: rot(o, heads=0), "not 0 heads"),
    (lambda o: rot(o, f=t(4, dtype=F64), heads=2), "freq has 4 pairs, more than fit heads of 6"),
    (lambda o: rot(o, f=t(2)), "freq is f32, expected f64"),
    (lambda o: rot(o, p=t(4, 2)), "positions is f32, expected i32 or i64"),
    (lambda o: rot(o, p=t(2, 4, dtype=I64)), "positions has 2 elements along axis 0"),
    (lambda o: rot(o, x=t(4, 2, 12, dtype=F64)), "x is f64"),
    (lambda o: rot(o, scale=float("inf")), "scale has to be finite"),
    (lambda o: rot(o, x=t(4, 12, 2).transpose(1, 2), p=t(4, 2, dtype=I64)), "x: the last axis has to be dense"),
    (lambda o: adamw(o, w=t(5)), "w has to be a list of tensors, not Tensor"),
    (lambda o: adamw(o, g=[t(5), t(5)]), "g has 2 tensors, w has 1"),
    (lambda o: adamw(o, g=[t(4)]), r"g\[0\] has 4 elements along axis 0, expected 5"),
    (lambda o: adamw(o, w=[t(5, dtype=F64)]), r"w\[0\] is f64, expected f32 or bf16"),
    (lambda o: adamw(o, w=[t(5).half()]), r"w\[0\] is torch.float16"),
    (lambda o: adamw(o, w=[t(5, 2).t()], g=[t(10)], m=[t(10)], v=[t(10)]), r"w\[0\] is not contiguous"),
    (lambda o: adamw(o, w=[3.0]), r"w\[0\] has to be a torch tensor"),
    (lambda o: adamw(o, m=[t(5, dtype=BF16)]), r"m\[0\] is bf16, expected f32"),
    (lambda o: adamw(o, v=[t(5, dtype=U8)]), r"v\[0\] is u8, expected f32"),
    (lambda o: adamw(o, m=[t(5, dtype=U8)], v=[t(5, dtype=U8)]), "exponents are missing"),
    (lambda o: adamw(o, exponents=[t(2, 1, dtype=U8)]), "exponents are given"),
    (lambda o: adamw(o, m=[t(5, dtype=U8)], v=[t(5, dtype=U8)], exponents=[t(2, 2, dtype=U8)]), r"exponents\[0\] has 4 elements"),
    (lambda o: adamw(o, s=t(1)), "step is f32, expected i64"),
    (lambda o: adamw(o, s=t(2, dtype=I64)), "step has 2 elements"),
    (lambda o: adamw(o, s=3), "step has to be a torch tensor"),
    (lambda o: adamw(o, lr=float("inf")), "lr and weight_decay have to be finite"),
    (lambda o: adamw(o, betas=(1.0, 0.9)), r"betas have to be in \[0, 1\)"),
    (lambda o: adamw(o, eps=-1.0), "eps has to be finite"),
    (lambda o: o.adamw_state([t(3)], bits=4), "moments have 32 or 8 bits, not 4"),
    (lambda o: o.adamw_values([t(5)], [t(5, dtype=U8)], [t(2, 1, dtype=U8)]), r"m\[0\] is f32, expected u8"),
    (lambda o: rotary_frequencies(5), "has to be even"),
    (lambda o: rotary_frequencies(4, base=-1.0), "base and stretch"),
    (lambda o: rotary_frequencies(4, turns=(3, 2), context=10), "turns have to be"),
])
def test_refusals(ops, call, message):
    with pytest.raises(OpsError, match=message):
        call(ops)


def test_overlapping_outputs(ops):
    v, q, s = t(6, 2, 15), t(6, 2, 12), t(2, 3, 4, 5)
    for call, message in (
            (lambda: attend(ops, v=v, out=(v, None)), "o overlaps v"),
            (lambda: attend(ops, s0=s, out=(t(6, 2, 15), s)), "s_last overlaps s0"),
            (lambda: back(ops, out=(q, q, v, None, None)), "dq overlaps dk"),
            (lambda: back(ops, ds=s, out=(t(6, 2, 12), q, v, None, s)), "ds0 overlaps ds"),
            (lambda: step(ops, s, out=s.view(-1)[:30].view(2, 15)), "s overlaps o"),
            (lambda: rot(ops, x=t(5, 2, 12)[:4], out=None), "host-only"),
            (lambda: adamw(ops, w=[v], g=[t(180)], m=[t(180)], v=[v.view(-1)]), r"v\[0\] overlaps w\[0\]|w\[0\] overlaps v\[0\]"),
            (lambda: adamw(ops, w=[v, v], g=[t(180)] * 2, m=[t(180), t(180)], v=[t(180), t(180)]), "overlaps w"),
            (lambda: adamw(ops, w=[t(180)], g=[v], m=[v], v=[t(180)]), r"m\[0\] overlaps g\[0\]")):
        with pytest.raises(OpsError, match=message):
            call()
    buf = t(5, 2, 12)
    with pytest.raises(OpsError, match="y overlaps x"):
        rot(ops, x=buf[:4], out=buf[1:])
    shared = [t(180)] * 2  # gradients may be shared
    with pytest.raises(OpsError, match="host-only"):
        adamw(ops, w=[t(180), t(180)], g=shared, m=[t(180), t(180)], v=[t(180), t(180)])


def test_gradients_that_would_be_lost_are_refused(ops):
    p = lambda *s: torch.zeros(*s, requires_grad=True)  # noqa: E731
    for name, call in (("q", lambda: attend(ops, q=p(6, 2, 12))), ("g", lambda: attend(ops, g=p(6, 2, 3))),
                       ("x", lambda: rot(ops, x=p(4, 2, 12))), ("s", lambda: step(ops, p(2, 3, 4, 5)))):
        with pytest.raises(OpsError, match=f"^{name} requires gradients"):
            call()
        with torch.no_grad(), pytest.raises(OpsError, match="host-only"):
            call()
    with pytest.raises(OpsError, match="host-only"):
        adamw(ops, w=[p(5)])


def test_c_interface_refuses_nulls():
    L = _lib.load()
    h = C.c_void_p()
    assert L.phz_ops_create(-1, C.byref(h)) == 0
    n = [None] * 13
    a, r, w = _lib.AttentionCfg(1.0, 4, 4), _lib.RotaryCfg(1.0, 1, 0, 0), _lib.AdamWCfg(0.1, 0.9, 0.99, 0.0, 0.0, 0)
    for call in (lambda c: L.phz_linear_attention(h, None, c, *n[:8]), lambda c: L.phz_linear_attention_backward(h, None, c, *n),
                 lambda c: L.phz_linear_attention_step(h, None, c, *n[:7])):
        assert call(None) != 0 and L.phz_ops_last_error(h) == b"configuration is missing"
        assert call(C.byref(a)) != 0 and L.phz_ops_last_error(h) == b"q is missing"
    assert L.phz_linear_attention(None, None, C.byref(a), *n[:8]) != 0
    assert L.phz_rotary(h, None, None, *n[:4]) != 0 and L.phz_ops_last_error(h) == b"configuration is missing"
    assert L.phz_rotary(h, None, C.byref(r), *n[:4]) != 0 and L.phz_ops_last_error(h) == b"x is missing"
    assert L.phz_adamw_step(h, None, None, 0, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"configuration is missing"
    assert L.phz_adamw_step(h, None, C.byref(w), 1, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"a list of tensors is missing"
    assert L.phz_adamw_step(h, None, C.byref(w), 0, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"step is missing"
    assert L.phz_adamw_values(h, None, -1, *n[:5]) != 0 and L.phz_ops_last_error(h) == b"too many tensors"
    L.phz_ops_destroy(h)


def test_frequencies():
    f = rotary_frequencies(8, base=100.0)
    assert f.dtype == F64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=F64), rtol=1e-15)
    assert torch.equal(rotary_frequencies(8, stretch=4.0), rotary_frequencies(8) / 4)
    g = rotary_frequencies(64, stretch=8.0, turns=(1, 32), context=1024)
    whole = rotary_frequencies(64)
    assert g[0] == whole[0] and g[-1] == whole[-1] / 8 and bool((g <= whole).all()) and bool((g >= whole / 8).all())
    assert rotary_frequencies(0).numel() == 0


# ── the references themselves ──

def test_attention_reference_gradients_are_autograd_s():
    gen = torch.Generator().manual_seed(1)
    T, B, H, nk, nv = 9, 2, 4, 3, 5
    rnd = lambda *s: torch.randn(*s, generator=gen, dtype=F64)  # noqa: E731
    q, k, v, g, s0 = rnd(T, B, 2 * nk), rnd(T, B, H * nk), rnd(T, B, nv), -rnd(T, B, H).abs(), rnd(B, H, nk, nv)
    reset = torch.rand(T, B, generator=gen) < 0.3
    do, ds = rnd(T, B, H * nv), rnd(B, H, nk, nv)
    for x in (q, k, v, g, s0):
        x.requires_grad_()
    split = lambda x, n: x.reshape(T, B, -1, n).repeat_interleave(H * n // x.shape[-1], 2)  # noqa: E731
    s, o = s0, []
    for i in range(T):
        a = torch.exp(g[i]) * (~reset[i]).double()[:, None]
        s = a[..., None, None] * s + split(k, nk)[i][..., :, None] * split(v, nv)[i][..., None, :]
        o.append(0.3 * (split(q, nk)[i][..., None, :] @ s)[..., 0, :].reshape(B, -1))
    o = torch.stack(o)
    ((o * do).sum() + (s * ds).sum()).backward()
    (ro, rs), _ = R.attention(q, k, v, g, s0, reset, nk, nv, 0.3)
    assert torch.allclose(ro, o.detach(), rtol=1e-12, atol=1e-13) and torch.allclose(rs, s.detach(), rtol=1e-12, atol=1e-13)
    grads, _ = R.attention_backward(do, q, k, v, g, s0, reset, ds, nk, nv, 0.3)
    for got, x in zip(grads, (q, k, v, g, s0)):
        assert torch.allclose(got, x.grad, rtol=1e-11, atol=1e-12)


def test_code_reference():
    """Codes rise with their values, and a value rounds to one of its neighbours."""
    for top, signed, last in ((14, True, 127), (30, False, 254)):
        values = R.code_values(130, top, signed)[:last + 1]
        assert all(a < b for a, b in zip(values, values[1:])) and values[0] == 0
        assert values[top * 8] == 8.0 and values[top * 8 + 7] == 15.0  # 2^(130 - 127) and up
        for c in (1, 5, 8, 9, 50, 100):
            assert R.encode(values[c], 130, top, signed, 0.5) == c
            mid = (values[c] + values[c + 1]) / 2
            assert R.encode(mid, 130, top, signed, 0.49) == c and R.encode(mid, 130, top, signed, 0.51) == c + 1
    assert R.encode(1e-30, 130, 30, False, 0.0) == 1 and R.encode(0.0, 130, 30, False, 0.99) == 0
