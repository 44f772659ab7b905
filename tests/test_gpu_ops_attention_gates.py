"""Gradients of linear attention's gates and of its first state where a head's steps
are not all finite: what the recurrence says of them is right, to the step."""
import pytest
import torch

from tests import attend_ref as R
from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
# Within the first chunk, on a chunk's border, in a chunk of one segment among many
# (1500 steps of 4 heads), in heads of other sizes than the tiles'.
@pytest.mark.parametrize("T, bad, nk, nv", [(40, 12, 32, 32), (150, 64, 33, 20), (150, 95, 128, 100), (1500, 700, 24, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_its_own_steps(ops, T, bad, nk, nv, value, dtype):
    """dg_t = exp(g_t) <E_t, S_{t-1}>: keys and values of a step are seen by the gates
    behind it, queries and the outputs' gradients by those up to it, gates by all of
    their episode, and none by another episode or head."""
    x = A.inputs(T, 2, 2, nk, nv, dtype, 11, reset=0)
    x["reset"] = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    x["reset"][bad + 10] = x["reset"][bad - 7] = True
    grads, bounds = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], x["ds"], nk, nv, nk ** -0.5)
    first, last = bad - 6, bad + 9  # gates of the episode that carry something on
    seen = {"k": (bad + 1, last), "v": (bad + 1, last), "q": (first, bad), "do": (first, bad), "g": (first, last)}
    for name, (lo, hi) in seen.items():
        y = dict(x)
        y[name] = x[name].clone()
        y[name][bad, 0, 1 if name != "g" else 0] = value
        dq, dk, dv, dg, ds0 = A.backward(ops, y, nk, nv)
        clean = torch.ones(T, 2, 2, dtype=torch.bool)
        clean[lo:hi + 1, 0, 0] = False
        R.within(dg.cpu()[clean], grads[3][clean], bounds[3][clean], f"{name}: dg")
        assert not torch.isfinite(dg[lo:hi + 1, 0, 0]).any(), name
        R.within(ds0, grads[4], bounds[4], f"{name}: ds0")  # a reset stands before the step
        for got, w, b, what in zip((dq, dk, dv), grads, bounds, ("dq", "dk", "dv")):
            n = nv if what == "dv" else nk
            for part in ((slice(None), 1), (slice(None), 0, slice(n, 2 * n)), (slice(bad + 10, None), 0), (slice(0, bad - 7), 0)):
                R.within(got[part], w[part], b[part], f"{name}: {what}")


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
def test_the_first_state_s_gradient_without_a_reset(ops, dtype):
    """ds0 sees queries and the outputs' gradients, not keys and values."""
    x = A.inputs(70, 1, 2, 32, 48, dtype, 12, reset=0)
    grads, bounds = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], None, x["ds"], 32, 48, 32 ** -0.5)
    for name in ("k", "v"):
        y = dict(x)
        y[name] = x[name].clone()
        y[name][20, 0, 3] = float("inf")
        dq, dk, dv, dg, ds0 = A.backward(ops, y, 32, 48)
        R.within(ds0, grads[4], bounds[4], f"{name}: ds0")
        R.within(dg[:21], grads[3][:21], bounds[3][:21], f"{name}: dg")
        R.within(dg[:, 0, 1], grads[3][:, 0, 1], bounds[3][:, 0, 1], f"{name}: dg of the other head")
        assert not torch.isfinite(dg[21:, 0, 0]).any()


def test_shared_heads_and_several_bad_steps(ops):
    """Two bad steps in one episode, of keys and then of queries: between them both are
    seen, before the first only the queries', behind the second only the keys'."""
    x = A.inputs(130, 1, 4, 16, 24, A.F32, 13, qh=2, kh=1, reset=0)
    grads, bounds = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], None, x["ds"], 16, 24, 0.25)
    y = dict(x, v=x["v"].clone(), do=x["do"].clone())
    y["v"][50, 0, 2], y["do"][40, 0, 1] = float("nan"), float("nan")  # head 0
    dg, ds0 = A.backward(ops, y, 16, 24)[3:]
    R.within(dg[41:51], grads[3][41:51], bounds[3][41:51], "dg between")
    R.within(dg[..., 1:], grads[3][..., 1:], bounds[3][..., 1:], "dg of other heads")
    R.within(ds0[:, 1:], grads[4][:, 1:], bounds[4][:, 1:], "ds0 of other heads")
    assert torch.isnan(dg[:41, 0, 0]).all() and torch.isnan(dg[51:, 0, 0]).all()


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [2, 33, 100, 1500])
def test_gates_that_close(ops, T, dtype):
    """Gates that leave little have gradients as little, also beside keys and values
    whose own weight in the last state's gradient is not."""
    x = A.inputs(T, 2, 2, 24, 32, dtype, 14, reset=0)
    x["g"].fill_(-12.0)
    want, bound = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], None, x["ds"], 24, 32, 24 ** -0.5)
    R.within(A.backward(ops, x, 24, 32)[3], want[3], bound[3], "dg")
