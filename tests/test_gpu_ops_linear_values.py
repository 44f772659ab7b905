"""What the linear layer's large f32 products, cut in bf16 pieces, make of
values at the ends of f32: infinite and NaN ones wherever they stand, and
numbers of one sign."""
import pytest
import torch

from tests import ops_ref as R

pytestmark = pytest.mark.gpu

F32 = torch.float32
INF = float("inf")
#: 2^33 multiply-adds and more, from where operands are cut; the second with
#: sums in splits.
SHAPES = [(4100, 2056, 1032), (1030, 8200, 1032)]


@pytest.fixture(scope="module")
def ops():
    from phyz_amd.ops import Ops
    return Ops(0)


def data(m, k, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g).cuda(), (torch.randn(n, k, generator=g) * k ** -0.5).cuda(),
            torch.randn(m, n, generator=g).cuda())


def same(got, want, rows, what):
    """Rows `rows` of `got` as the 64-bit product has them: the same infinities and NaN."""
    got, want = got[rows].cpu().double(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    bad = ~torch.isfinite(want)
    assert torch.equal(got[bad & ~torch.isnan(want)], want[bad & ~torch.isnan(want)]), what
    assert torch.isfinite(got[~bad]).all(), what


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_infinite_and_nan_operands_in_pieces(ops, shape):
    m, k, n = shape
    x, w, dy = data(*shape)
    x[3, 17], x[5, 40], x[7, 3], x[9, 60] = INF, -INF, float("nan"), INF
    x[11, 20], x[11, 21] = INF, -INF          # a row of both
    x[9, 61] = -INF
    w[4, 17], w[6, 17], w[8, 17] = 0.0, INF, -INF   # infinity times 0, times infinities
    w[10, 60], w[10, 61] = INF, -INF          # two infinite products of one sign
    w[12, 100], x[13] = float("nan"), 0.0     # NaN times 0
    rows = torch.tensor([0, 3, 5, 7, 9, 11, 13, m - 1])
    y = ops.linear(x, w)
    same(y, x[rows.cuda()].double().cpu() @ w.double().cpu().T, rows, "y")
    clean = torch.tensor([j for j in range(n) if j not in (6, 8, 10, 12)])
    assert torch.isfinite(y[0, clean.cuda()]).all()
    dy[2, 5], dy[4, 6], dy[4, 7] = INF, float("nan"), -INF
    dx, dw, db = ops.linear_backward(dy, x, w)
    rows = torch.tensor([0, 2, 4, m - 1])
    same(dx, dy[rows.cuda()].double().cpu() @ w.double().cpu(), rows, "dx")
    rows = torch.tensor([0, 5, 6, 7, n - 1])
    same(dw, dy[:, rows.cuda()].double().cpu().T @ x.double().cpu(), rows, "dw")
    assert db[5] == INF and torch.isnan(db[6]) and db[7] == -INF


@pytest.mark.parametrize("value", [float("nan"), INF], ids=["nan", "inf"])
def test_operands_wholly_not_finite(ops, value):
    """A diverged run: every product is NaN, or an infinity of the weight's sign."""
    x, w, dy = data(*SHAPES[0])
    x.fill_(value)
    y = ops.linear(x, w.abs() + 1)
    assert torch.isnan(y).all() if value != value else bool((y == INF).all())
    dx, dw, db = ops.linear_backward(torch.full_like(dy, value), x, w)
    assert torch.isnan(dx).all() and (torch.isnan(dw).all() if value != value else bool((dw == INF).all()))
    assert not torch.isfinite(db).any()


def test_a_diverged_run_costs_what_a_healthy_one_does(ops):
    """The time of an all-NaN product beside a clean one's: the same instructions,
    so about the same time; a factor of ten leaves room for clocks."""
    x, w, dy = data(*SHAPES[0])

    def ms(x, dy):
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.linear(x, w)
            ops.linear_backward(dy, x, w)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean = ms(x, dy)
    assert ms(torch.full_like(x, float("nan")), torch.full_like(dy, float("nan"))) <= 10 * clean


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_pieces_lean_to_no_side(ops, shape):
    """Operands of one sign whose lower bits are all set, where pieces that are cut
    off leave out most, and always low. What rounded pieces leave out is at most
    2^-24 of a product and of either sign, and so are the sums' roundings: the mean
    over 128 x 1032 sums of 2056 and more is within 2^-25 of them."""
    m, k, n = shape
    g = torch.Generator().manual_seed(3)
    x, w = ((1 + 2.0 ** -7 * (1 - torch.rand(r, k, generator=g) * 2.0 ** -6)).cuda() for r in (m, n))
    y = ops.linear(x, w)[:128].double().cpu()
    want = x[:128].double().cpu() @ w.double().cpu().T
    assert abs(float(((y - want) / want).mean())) <= 2.0 ** -25


def test_cut_at_the_ends_of_f32(ops):
    """Numbers that round up to infinity in bf16, powers of two, f32's largest, and
    small ones: one product each of a long sum of zeros is exact to f32's unit."""
    m, k, n = SHAPES[0]
    v = torch.tensor([3.4028234663852886e38, -3.4e38, 3.3961775292304601e38, 2.0 ** 127, 1.5, 1 + 2.0 ** -23,
                      1 + 2.0 ** -8 + 2.0 ** -23, 2 - 2.0 ** -23, -(1 + 2.0 ** -8), 3.0e-33, 2.0 ** -100 * (2 - 2.0 ** -23)])
    x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    x[:len(v), 77] = v.cuda()
    u = torch.tensor([1.0, -1.0, 0.5, 1 - 2.0 ** -24, 2.0 ** -20 * (1 + 2.0 ** -23), 0.7])
    w[:len(u), 77] = u.cuda()
    y = ops.linear(x, w)[:len(v), :len(u)].double().cpu()
    want = v.double()[:, None] * u.double()[None]
    # Six products, at most 2^-24 left out, and as many roundings of sums below
    # the value: four units of 2^-24; and a result below f32's normal numbers
    # (3e-33 x 2^-20) is half its spacing there, 2^-150, off.
    assert bool(((y - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -150).all())
