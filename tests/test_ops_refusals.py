"""What the sequence operators refuse, on a handle without a GPU, and the
64-bit references that the device tests compare with, against autograd and
plain rounding."""
import ctypes as C

import pytest
import torch

from phyz_amd import _lib
from phyz_amd.ops import Ops, OpsError
from tests import ops_ref as R

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype)


def test_valid_calls_reach_the_device_check(ops):
    """A host-only handle refuses last: the arguments were right."""
    x = t(6, 2, 5)
    for call in (lambda: ops.gated_scan(x, x.clone(), h0=t(2, 5), reset=t(6, 2, dtype=torch.bool)),
                 lambda: ops.gated_scan_backward(x, x, x, x, h0=t(2, 5), dh_last=t(2, 5)),
                 lambda: ops.gated_step(t(2, 5), t(2, 5), t(2, 5), reset=t(2, dtype=torch.uint8)),
                 lambda: ops.linear(t(4, 3), t(7, 3), bias=t(7), residual=t(4, 7), act="gelu"),
                 lambda: ops.linear(t(2, 4, 3), t(7, 3), save_pre=True),
                 lambda: ops.linear_backward(t(4, 7), t(4, 3), t(7, 3), pre=t(4, 7), act="silu"),
                 lambda: ops.orthogonalize(t(3, 4, 5, dtype=BF16)),
                 lambda: ops.muon_step(t(4, 5), t(4, 5, dtype=BF16), t(4, 5)),
                 lambda: ops.reserve(100)):
        with pytest.raises(OpsError, match="host-only"):
            call()
    assert ops.workspace_bytes == 0


@pytest.mark.parametrize("call, message", [
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 4)), "x has 4 elements along axis 2, expected 5"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5, dtype=BF16)), "x is bf16, expected f32"),
    (lambda o: o.gated_scan(t(2, 5), t(2, 5)), "z has 2 dimensions, expected 3"),
    (lambda o: o.gated_scan(t(6, 2, 5, dtype=torch.uint8), t(6, 2, 5)), "z is u8, expected f32 or bf16"),
    (lambda o: o.gated_scan(t(6, 2, 5, dtype=torch.float64), t(6, 2, 5)), "z is f64"),
    (lambda o: o.gated_scan(t(6, 2, 5).half(), t(6, 2, 5)), "z is torch.float16"),
    (lambda o: o.gated_scan(t(6, 5, 2).transpose(1, 2), t(6, 2, 5)), "the last axis has to be dense"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), h0=t(2, 5, dtype=BF16)), "h0 is bf16, expected f32"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), h0=t(5, 2)), "h0 has 5 elements along axis 0"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), reset=t(2, 6, dtype=torch.bool)), "reset has 2 elements"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), reset=t(6, 2)), "reset is f32, expected u8"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), form="lstm"), "unknown gate form 'lstm'"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), out=(t(6, 1, 5).expand(6, 2, 5), t(2, 5))), "h is broadcast"),
    (lambda o: o.gated_scan(t(6, 2, 5), t(6, 2, 5), out=(torch.as_strided(t(99), (6, 2, 5), (10, 4, 1)), t(2, 5))),
     "h overlaps itself"),
    (lambda o: o.gated_scan(7, t(6, 2, 5)), "z has to be a torch tensor"),
    (lambda o: o.gated_scan_backward(t(6, 2, 5), t(6, 2, 5), t(6, 2, 5), t(5, 2, 5)), "h has 5 elements along axis 0"),
    (lambda o: o.gated_scan_backward(t(6, 2, 5), t(6, 2, 5), t(6, 2, 5), t(6, 2, 5), dh_last=t(2, 6)), "dh_last has 6"),
    (lambda o: o.gated_step(t(2, 5), t(2, 5), t(2, 5, dtype=BF16)), "h is bf16, expected f32"),
    (lambda o: o.gated_step(t(2, 5), t(2, 5), t(2, 5), reset=t(3, dtype=torch.bool)), "reset has 3 elements"),
    (lambda o: o.linear(t(4, 3), t(7, 4)), "w has 4 elements along axis 1, expected 3"),
    (lambda o: o.linear(t(4, 3), t(7)), "w has 1 dimensions, expected 2"),
    (lambda o: o.linear(t(4, 3), t(7, 3), bias=t(4)), "bias has 4 elements along axis 0, expected 7"),
    (lambda o: o.linear(t(4, 3), t(7, 3), residual=t(4, 3)), "residual has 3 elements along axis 1, expected 7"),
    (lambda o: o.linear(t(4, 3), t(7, 3), act="swish"), "unknown activation 'swish'"),
    (lambda o: o.linear(t(4, 3, dtype=BF16), t(7, 3)), "w is f32, expected bf16"),
    (lambda o: o.linear(t(3, 4).t(), t(7, 3)), "x: the last axis has to be dense"),
    (lambda o: o.linear_backward(t(4, 7), t(4, 3), t(7, 3), act="tanh"), "pre is missing"),
    (lambda o: o.linear_backward(t(5, 7), t(4, 3), t(7, 3)), "dy has 5 elements along axis 0, expected 4"),
    (lambda o: o.orthogonalize(t(5)), "g has 1 dimensions, expected a matrix"),
    (lambda o: o.orthogonalize(t(5, 5), steps=-1), "steps is -1"),
    (lambda o: o.orthogonalize(t(5, 5), coef=(1.0, float("nan"), 0.0)), "coefficients have to be finite"),
    (lambda o: o.orthogonalize(t(5, 5), eps=-1.0), "eps has to be finite"),
    (lambda o: o.muon_step(t(4, 5), t(4, 5), t(5, 4)), "m has 5 elements along axis 0, expected 4"),
    (lambda o: o.muon_step(t(4, 5, dtype=BF16), t(4, 5), t(4, 5)), "w is bf16, expected f32"),
    (lambda o: o.muon_step(t(4, 5), t(4, 5), t(4, 5), lr=float("inf")), "lr, momentum and weight_decay"),
])
def test_refusals(ops, call, message):
    with pytest.raises(OpsError, match=message):
        call(ops)


def test_overlapping_outputs(ops):
    x = t(6, 2, 5)
    with pytest.raises(OpsError, match="h overlaps x"):
        ops.gated_scan(t(6, 2, 5), x, out=(x, t(2, 5)))
    with pytest.raises(OpsError, match="h_last overlaps h0"):
        h0 = t(2, 5)
        ops.gated_scan(t(6, 2, 5), x, h0=h0, out=(t(6, 2, 5), h0))
    with pytest.raises(OpsError, match="dz overlaps dx"):
        g = t(6, 2, 5)
        ops.gated_scan_backward(x, x, x, x, out=(g, g, t(2, 5)))
    with pytest.raises(OpsError, match="h overlaps z"):
        h = t(2, 5)
        ops.gated_step(h, t(2, 5), h)
    both = t(6, 2, 12)
    with pytest.raises(OpsError, match="dz overlaps dx"):  # halves that share a column
        ops.gated_scan_backward(x, x, x, x, out=(both[..., 0:5], both[..., 4:9], t(2, 5)))
    with pytest.raises(OpsError, match="host-only"):       # halves that do not
        ops.gated_scan_backward(x, x, x, x, out=(both[..., 0:5], both[..., 5:10], t(2, 5)))
    y = t(4, 8)
    with pytest.raises(OpsError, match="y overlaps x"):
        ops.linear(y[:, :3], t(8, 3), out=y)
    with pytest.raises(OpsError, match="y overlaps residual"):
        wide = t(4, 9)
        ops.linear(t(4, 3), t(8, 3), residual=wide[:, :8], out=wide[:, 1:])
    with pytest.raises(OpsError, match="host-only"):
        ops.linear(t(4, 3), t(8, 3), residual=y, out=y)
    w = t(4, 5)
    with pytest.raises(OpsError, match="w overlaps m"):
        ops.muon_step(w, t(4, 5), w)
    with pytest.raises(OpsError, match="o overlaps g"):
        ops.orthogonalize(w, out=w)


def test_c_interface_refuses_nulls():
    L = _lib.load()
    h = C.c_void_p()
    assert L.phz_ops_create(-1, None) != 0
    assert b"null output pointer" in L.phz_ops_last_error(None)
    assert L.phz_ops_create(-1, C.byref(h)) == 0
    n = [None] * 10
    assert L.phz_gated_scan(None, None, 0, *n[:6]) != 0
    assert L.phz_gated_scan(h, None, 5, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"unknown gate form"
    assert L.phz_gated_scan(h, None, 0, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"z is missing"
    assert L.phz_gated_scan_backward(h, None, 0, *n[:10]) != 0 and L.phz_ops_last_error(h) == b"z is missing"
    assert L.phz_gated_step(h, None, 0, *n[:4]) != 0 and L.phz_ops_last_error(h) == b"z is missing"
    assert L.phz_linear(h, None, 9, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"unknown activation"
    assert L.phz_linear(h, None, 0, *n[:6]) != 0 and L.phz_ops_last_error(h) == b"x is missing"
    assert L.phz_linear_backward(h, None, 0, *n[:7]) != 0 and L.phz_ops_last_error(h) == b"x is missing"
    cfg = _lib.MuonCfg(1.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1, 0)
    assert L.phz_orthogonalize(h, None, None, None, None) != 0
    assert L.phz_ops_last_error(h) == b"configuration is missing"
    assert L.phz_orthogonalize(h, None, C.byref(cfg), None, None) != 0 and L.phz_ops_last_error(h) == b"g is missing"
    assert L.phz_muon_step(h, None, C.byref(cfg), None, None, None) != 0 and L.phz_ops_last_error(h) == b"g is missing"
    L.phz_ops_destroy(h)
    L.phz_ops_destroy(None)


# ── the references themselves ──

@pytest.mark.parametrize("form", ["sigmoid", "decay"])
def test_scan_reference_gradients_are_autograd_s(form):
    g = torch.Generator().manual_seed(1)
    T, B, D = 9, 2, 3
    z, x = (torch.randn(T, B, D, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    h0 = torch.randn(B, D, generator=g, dtype=torch.float64, requires_grad=True)
    dh, dl = torch.randn(T, B, D, generator=g).double(), torch.randn(B, D, generator=g).double()
    reset = torch.rand(T, B, generator=g) < 0.2
    h, hs = h0, []
    for t_ in range(T):
        c = torch.sigmoid(z[t_]) if form == "sigmoid" else z[t_]
        h = c * torch.where(reset[t_][:, None], torch.zeros_like(h), h) + ((1 - c) if form == "sigmoid" else 1) * x[t_]
        hs.append(h)
    hs = torch.stack(hs)
    ((hs * dh).sum() + (h * dl).sum()).backward()
    got, _ = R.scan_backward(dh, z, x, hs, h0, reset, dl, form, F32)
    for a, b in zip(got, (z.grad, x.grad, h0.grad)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)
    want = R.scan(z, x, h0, reset, form, F32)
    assert torch.allclose(want[0], hs, rtol=1e-13, atol=1e-14) and torch.allclose(want[1], h, rtol=1e-13, atol=1e-14)


@pytest.mark.parametrize("name", ["none", "tanh", "relu", "silu", "gelu"])
def test_linear_reference_gradients_are_autograd_s(name):
    g = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((6, 4), (5, 4), (5,)))
    dy = torch.randn(6, 5, generator=g).double()
    p = x @ w.T + b
    y = {"gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": torch.nn.functional.silu,
         "tanh": torch.tanh, "relu": torch.relu, "none": lambda v: v}[name](p)
    (y * dy).sum().backward()
    got, _ = R.linear_backward(dy, x, w, p, name, F32)
    for a, v in zip(got, (x, w, b)):
        assert torch.allclose(a, v.grad, rtol=1e-11, atol=1e-12)
    assert torch.allclose(R.linear(x, w, b, None, name, F32)[0], y, rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_unit_is_what_rounding_costs(dtype):
    """Rounding to the stored type stays within R.unit of the value, and reaches it."""
    u = R.unit(dtype)
    v = torch.cat([torch.linspace(1, 2, 5001, dtype=torch.float64), torch.tensor([1 + u], dtype=torch.float64)])
    rel = ((v.to(dtype).double() - v) / v).abs()
    assert float(rel.max()) <= u and float(rel.max()) > 0.9 * u


def test_orthogonalize_reference_is_near_orthogonal():
    g = torch.randn(20, 30, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    s = torch.linalg.svdvals(R.orthogonalize(g, steps=8))
    assert float(s.min()) > 0.6 and float(s.max()) < 1.3
