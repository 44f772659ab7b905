"""Rotary positions on the device against rotations in 64 bits."""
import pytest
import torch

from tests import attend_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def inputs(T, B, H, size, pairs, dtype, far, seed=0, ints=torch.int64):
    from phyz_amd.ops import rotary_frequencies
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, B, H * size, generator=g).to(dtype).cuda()
    p = torch.randint(-far, far + 1, (T, B), generator=g).to(ints).cuda()
    return x, p, rotary_frequencies(2 * pairs).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T, B, H, size, pairs, far", [
    (1, 1, 1, 2, 1, 5), (3, 5, 2, 7, 3, 1000), (2, 3, 4, 64, 32, 100), (5, 2, 3, 64, 16, 1 << 24), (4, 3, 1, 33, 0, 10),
    (2, 2, 2, 130, 65, 1 << 20), (1, 1024, 4, 64, 16, 10 ** 6), (7, 3, 5, 80, 20, 1), (3, 2, 2, 6, 2, (1 << 31) - 1),
    (2, 2, 12, 128, 64, 5000), (1, 3, 1, 300, 150, 99)])
def test_turns(ops, T, B, H, size, pairs, far, layout, dtype):
    for ints in (torch.int32, torch.int64):
        x, p, f = inputs(T, B, H, size, pairs, dtype, far, seed=size, ints=ints)
        for inverse, scale in ((False, 1.0), (True, 1.3)):
            y = ops.rotary(x, p, f, heads=H, layout=layout, scale=scale, inverse=inverse)
            want, bound = R.rotary(x, p, f, H, layout, scale, inverse)
            R.within(y, want, bound + 1e-37, f"{ints} inverse={inverse}")


def test_far_positions(ops):
    """Positions past 2^31, where a position times a frequency is 2^40 turns."""
    x, _, f = inputs(4, 3, 2, 32, 16, F32, 1)
    p = torch.tensor([[0, 1, -1], [1 << 31, -(1 << 31) - 1, (1 << 31) + 1], [1 << 40, 3, 1 << 42], [5, 1 << 35, 7]]).cuda()
    y = ops.rotary(x, p, f, heads=2)
    want, bound = R.rotary(x, p, f, 2, "half", 1.0, False)
    # 2^42 turns leave 2^-10 of them in f64: bound's second part.
    R.within(y, want, bound, "y")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_views(ops, layout, dtype):
    """Heads in the middle of a buffer's rows, turned where they stand; the rest of
    the rows and elements behind the pairs stay."""
    x, p, f = inputs(9, 5, 3, 20, 7, dtype, 1000)
    want = ops.rotary(x, p, f, heads=3, layout=layout)
    wide = torch.full((5, 9, 67), 4.0, dtype=dtype, device="cuda")
    view = wide.transpose(0, 1)[..., 3:63]
    view.copy_(x)
    q = torch.stack([p, p + 1], -1)[..., 0]
    got = ops.rotary(view, q, f, heads=3, layout=layout, out=view)
    assert got is view and torch.equal(view, want)
    assert bool((wide[..., :3] == 4).all()) and bool((wide[..., 63:] == 4).all())
    tail = x.view(9, 5, 3, 20)[..., 14:]
    assert torch.equal(want.view(9, 5, 3, 20)[..., 14:], tail)
    one = ops.rotary(x[0], p[0], f, heads=3, layout=layout)
    assert torch.equal(one, want[0])


def test_there_and_back(ops):
    """The inverse takes a rotation back, and is its gradient: both to the roundings
    of two rotations."""
    x, p, f = inputs(6, 4, 2, 64, 32, F32, 10 ** 6)
    y = ops.rotary(x, p, f, heads=2)
    back = ops.rotary(y, p, f, heads=2, inverse=True)
    assert float((back - x).abs().max()) <= 60 * R.U32 * float(x.abs().max())
    d = torch.randn_like(x)
    dx = ops.rotary(d, p, f, heads=2, inverse=True)
    a, b = float((d.double() * y.double()).sum()), float((dx.double() * x.double()).sum())
    assert abs(a - b) <= 24 * R.U32 * float((d.double().abs() * y.double().abs()).sum() + (dx.double() * x.double()).abs().sum())


def test_streams_graphs_and_empty(ops):
    x, p, f = inputs(8, 3, 2, 64, 32, BF16, 100)
    want = ops.rotary(x, p, f, heads=2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    y, graph = torch.empty_like(x), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.rotary(x, p, f, heads=2, out=y)
    for k in range(3):
        y.zero_()
        p.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.rotary(x, p, f, heads=2))
        assert k or not torch.equal(y, want)
    assert ops.rotary(x[:0], p[:0], f, heads=2).shape == (0, 3, 128)
    assert torch.equal(ops.rotary(x, p, f[:0], heads=2), x)
