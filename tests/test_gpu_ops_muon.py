"""Orthogonalised updates on the device against 64 bits.

Singular values lie within a factor of four, so no direction's error grows
against its signal by more than that: five steps, each with a few roundings U of
the largest singular value, leave a relative error (Frobenius) below 80 U, where
U is 2^-23 for f32 (what the matrix cores are given of an f32 is good to 22
bits, and sums round once more) and 2^-12 for bf16 (11 bits), whose output is
rounded to bf16 besides."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = {F32: 80 * 2.0 ** -23, BF16: 80 * 2.0 ** -12 + 2.0 ** -9}
SHAPES = [(1, 1), (1, 9), (7, 1), (2, 3), (16, 16), (31, 33), (64, 64), (65, 64), (64, 200), (129, 100), (256, 256),
          (8, 256), (256, 67), (130, 1000), (515, 140), (700, 300), (384, 384), (513, 1030)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def matrices(batch, rows, cols, dtype, seed=0, scale=1e-3):
    """Random singular vectors, singular values from 1/4 to 1."""
    g = torch.Generator().manual_seed(seed)
    k = min(rows, cols)
    out = []
    for _ in range(batch):
        u, _ = torch.linalg.qr(torch.randn(rows, k, generator=g, dtype=torch.float64))
        v, _ = torch.linalg.qr(torch.randn(cols, k, generator=g, dtype=torch.float64))
        s = 0.25 + 0.75 * torch.rand(k, generator=g, dtype=torch.float64)
        out.append(scale * (u * s) @ v.T)
    return torch.stack(out).to("cuda", dtype)


def off(got, want):
    got = R.d64(got)
    assert torch.isfinite(got).all()
    return float(torch.linalg.norm(got - want) / torch.linalg.norm(want))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(ops, shape, dtype):
    batch = 1 if max(shape) > 256 else 3
    g = matrices(batch, *shape, dtype)
    o = ops.orthogonalize(g)
    assert o.dtype == dtype and o.shape == g.shape
    assert off(o, R.orthogonalize(g)) <= TOL[dtype]
    if batch == 1:
        assert torch.equal(ops.orthogonalize(g[0]), o[0])
    assert torch.equal(ops.orthogonalize(g), o)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(128, 160), (160, 128), (129, 160), (128, 161), (96, 281), (64, 530), (530, 64),
                                   (32, 1150), (1150, 17), (20, 3000), (100, 100)], ids=str)
def test_sizes_about_one_workgroup(ops, shape, dtype):
    """What one workgroup holds, and what it just does not; a batch of each."""
    g = matrices(5, *shape, dtype, seed=6)
    o = ops.orthogonalize(g)
    for k in range(5):
        assert off(o[k], R.orthogonalize(g[k])) <= TOL[dtype]
    assert torch.equal(ops.orthogonalize(g[3]), o[3])


@pytest.mark.parametrize("steps", [0, 1, 2, 7])
def test_steps_and_coefficients(ops, steps):
    g = matrices(2, 40, 72, F32)
    for coef in (R.COEF, (1.875, -1.25, 0.375)):
        o = ops.orthogonalize(g, steps=steps, coef=coef, eps=1e-3)
        assert off(o, R.orthogonalize(g, steps, coef, 1e-3)) <= TOL[F32]


def test_coefficients_beyond_f16(ops):
    """Steps that raise every singular value a hundredfold: the iterates leave
    f16's range and the f32 products take over. a X alone is exact to a few U;
    its error here is that of one rounding a step."""
    for shape in ((40, 72), (72, 40), (200, 150)):
        g = matrices(2, *shape, F32)
        o = ops.orthogonalize(g, steps=4, coef=(100.0, 0.0, 0.0))
        assert off(o, R.orthogonalize(g, 4, (100.0, 0.0, 0.0))) <= TOL[F32]


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e12, 1e30])
def test_any_magnitude(ops, scale):
    """The norm's squares leave f32's range; the result does not depend on it."""
    g = matrices(1, 48, 64, F32, scale=1.0) * scale
    assert off(ops.orthogonalize(g, eps=0.0), R.orthogonalize(g, eps=0.0)) <= TOL[F32]


def test_zero_and_nan(ops):
    g = torch.zeros(2, 30, 20, device="cuda")
    assert not ops.orthogonalize(g).any()
    g[1] = matrices(1, 30, 20, F32)[0]
    o = ops.orthogonalize(g)
    assert not o[0].any() and off(o[1], R.orthogonalize(g[1])) <= TOL[F32]
    g[0, 3, 4] = float("nan")  # one matrix's NaN stays in it
    o2 = ops.orthogonalize(g)
    assert torch.isnan(o2[0]).all() and torch.equal(o2[1], o[1])
    assert ops.orthogonalize(torch.zeros(0, 4, 4, device="cuda")).shape == (0, 4, 4)
    assert ops.orthogonalize(torch.zeros(4, 0, device="cuda")).shape == (4, 0)


@pytest.mark.parametrize("gtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(2, 256, 256), (1, 67, 31), (3, 20, 50), (1, 300, 520), (2, 1, 40)], ids=str)
def test_muon_step(ops, shape, nesterov, gtype):
    g, m = matrices(*shape, gtype, seed=1), matrices(*shape, F32, seed=2, scale=2e-3)
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(3)).cuda()
    kw = dict(lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    ww, wm = R.muon(w, g, m, **kw)
    before = w.clone()
    ops.muon_step(w, g, m, **kw)
    # m: two roundings of its terms. w: its own roundings, and the update's
    # error (in norm), of u's singular values within a factor of 16.
    assert off(m, wm) <= 4 * R.U32
    step = 0.05 * max(1.0, shape[1] / shape[2]) ** 0.5
    room = 4 * R.U32 * float(before.double().norm()) + 4 * TOL[F32] * step * (shape[0] * min(shape[1:])) ** 0.5
    assert float((R.d64(w) - ww).norm()) <= room


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(33, 45), (128, 64), (300, 257)], ids=str)
def test_strided_views(ops, shape, dtype):
    g = matrices(2, *shape, dtype)
    wide = torch.full((2, shape[0] + 3, shape[1] + 5), 3.0, dtype=dtype, device="cuda")
    v = wide[:, 1:1 + shape[0], 2:2 + shape[1]]
    v.copy_(g)
    o = ops.orthogonalize(g)
    assert torch.equal(ops.orthogonalize(v), o)
    ops.orthogonalize(g, out=v)
    assert torch.equal(v, o)
    v.fill_(3.0)
    assert (wide == 3).all()


def test_graph_replays(ops):
    g = matrices(2, 100, 60, F32)
    side = torch.cuda.Stream()
    o = torch.empty_like(g)
    with torch.cuda.stream(side):
        ops.orthogonalize(g, out=o)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.orthogonalize(g, out=o)
    for k in range(4):
        g.add_(1e-4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ops.orthogonalize(g)), k
