"""What decays leave of states that are large or not finite: rollouts, single steps
and the recurrence in 64 bits agree down to what f32 holds."""
import pytest
import torch

from tests import attend_ref as R
from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops
# Gates before the others, which are of the usual size: one below f32's normal
# numbers, several whose product is (within a tile of 16, over two, over a chunk).
GATES = {"one": {0: -90.0}, "the least": {0: -103.5}, "two": {0: -50.0, 3: -50.0}, "two tiles": {5: -60.0, 20: -70.0},
         "many": {t: -4.0 for t in range(30)}, "over chunks": {10: -45.0, 70: -45.0, 140: -45.0}}


def sizes_of_gates_sums(x, nk, nv, scale):
    """exp(g_t) times the sum of |E_t| |S_{t-1}| over the state, which a 32-bit dg's
    partial sums reach at most."""
    H = x["g"].shape[-1]
    do, q, k, v = (R.split(x[n], m, H) for n, m in (("do", nv), ("q", nk), ("k", nk), ("v", nv)))
    a, age = R.gates(x["g"], x["reset"])
    S = R.sweep(q, k, v, a, age, R.d64(x["s0"]))[2]
    E = R.sweep(k, scale * q, do, a, age, R.d64(x["ds"]), back=True)[2][::-1]
    before = [R.d64(x["s0"])] + [s for s, _, _ in S[:-1]]
    return torch.stack([a[t] * (E[t][0].abs() * before[t].abs()).sum((-1, -2)) for t in range(len(S))])


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gates", GATES)
# In one piece, and in segments of the steps.
@pytest.mark.parametrize("T", [12, 150, 1500])
def test_large_first_states(ops, T, gates, dtype):
    """Of a first state of 1e37 something is left behind all of these, and the same of
    the last state's gradient from the other end. Gates' gradients are sums of 1280
    products of both: where those pass f32's range there is no answer in 32 bits."""
    x = A.inputs(T, 1, 2, 32, 40, dtype, 21, reset=0)
    for t, v in GATES[gates].items():
        if t < T:
            x["g"][t] = v
            x["g"][T - 1 - t] = v
    x["s0"] *= 1e37
    A.check_forward(A.forward(ops, x, 32, 40), x, 32, 40)
    x["s0"] /= 1e37
    x["ds"] *= 1e37
    want, bound = R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], None, x["ds"], 32, 40, 32 ** -0.5)
    held = sizes_of_gates_sums(x, 32, 40, 32 ** -0.5) < 3e38
    assert held.any()
    for got, w, b, n in zip(A.backward(ops, x, 32, 40), want, bound, ("dq", "dk", "dv", "dg", "ds0")):
        if n == "dg":
            got, w, b = got.cpu()[held], w[held], b[held]
        R.within(got, w, b, n)


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
def test_steps_of_large_states(ops, dtype):
    for g in (-86.0, -90.0, -100.0, -103.9):
        x = A.inputs(1, 3, 2, 16, 24, dtype, 22, reset=0)
        x["s0"] *= 1e37
        x["g"].fill_(g)
        s = x["s0"].clone()
        o = ops.linear_attention_step(x["q"][0], x["k"][0], x["v"][0], x["g"][0], s)
        A.check_forward((o[None], s), x, 16, 24)
        A.check_forward(A.forward(ops, x, 16, 24), x, 16, 24)


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gates", GATES)
def test_infinite_first_states(ops, gates, dtype):
    """An infinity stays one whatever the decays, until a reset."""
    T = 200
    x = A.inputs(T, 2, 2, 16, 16, dtype, 23, reset=0)
    x["reset"] = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    x["reset"][170] = True
    for t, v in GATES[gates].items():
        x["g"][t] = v
    want, bound = R.attention(x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], 16, 16, 0.25)
    x["s0"][0, 1, 3, 5] = float("inf")
    o, s = A.forward(ops, x, 16, 16)
    assert not torch.isfinite(o[:170, 0, 16 + 5]).any()
    clean = torch.ones(o.shape, dtype=torch.bool)
    clean[:170, 0, 16 + 5] = False
    R.within(o.cpu()[clean], want[0][clean], bound[0][clean], "o")
    R.within(s, want[1], bound[1], "s")
    state, outs = x["s0"].clone(), []
    for t in range(T):
        outs.append(ops.linear_attention_step(x["q"][t], x["k"][t], x["v"][t], x["g"][t], state, reset=x["reset"][t]))
    assert torch.equal(torch.isfinite(torch.stack(outs)), torch.isfinite(o))


def test_infinite_gradients_of_the_last_state(ops):
    T = 150
    x = A.inputs(T, 1, 2, 16, 16, A.F32, 24, reset=0)
    x["g"][T - 1] = -90.0
    x["g"][T - 40:T - 35] = -50.0
    x["ds"][0, 0, 3, 5] = float("inf")
    dq, dk, dv, dg, ds0 = A.backward(ops, x, 16, 16)
    assert not torch.isfinite(dk[:, 0, 3]).any() and not torch.isfinite(dv[:, 0, 5]).any()
    assert not torch.isfinite(dg[1:, 0, 0]).any() and not torch.isfinite(ds0[0, 0, 3, 5])
    assert torch.isfinite(dk[..., 16:]).all() and torch.isfinite(dg[..., 1]).all() and torch.isfinite(dq).all()
