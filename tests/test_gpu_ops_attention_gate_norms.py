"""Gates' gradients by the norm: the element-wise bounds of tests/attend_ref.py add up
magnitudes over 128 steps and leave room for faults of a percent."""
import math

import pytest
import torch

from tests import attend_ref as R
from tests import test_gpu_ops_attention as A

SIZES = [(1, 3, 2, 64, 64), (33, 1, 2, 64, 31), (100, 1, 2, 128, 128), (257, 1, 1, 40, 72), (700, 1, 2, 64, 64), (1100, 1, 1, 128, 64),
         (70, 30, 4, 8, 16)]


def most_off(T, nk, nv):
    """dg = exp(g_t) <E_t, S_{t-1}>. E and S are sums of up to n products one after the
    other, off by sqrt(n / 3) U of their size (U = 2^-24, each addition by up to U of it,
    evenly spread); their product's sum by both and its own additions, less than sqrt(3)
    of one. Decays are off by U of their logarithm, less than 16 where anything is left
    that counts. Twice all that."""
    return 2 * (math.sqrt(3 * R._terms(T, nk, nv) / 3) + 16) * R.U32


def off(got, want):
    """The largest of a head's norms of got - want, in want's."""
    got, want = got.double().cpu(), want.double()
    return float(((got - want).norm(dim=0) / want.norm(dim=0)).max())


def reference(x, nk, nv):
    return R.attention_backward(x["do"], x["q"], x["k"], x["v"], x["g"], x["s0"], x["reset"], x["ds"], nk, nv, nk ** -0.5)[0][3]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T, B, H, nk, nv", SIZES)
def test_by_the_norm(T, B, H, nk, nv, dtype):
    """In bf16 too: q, k and v are given, dg is f32."""
    from phyz_amd.ops import Ops
    x = A.inputs(T, B, H, nk, nv, dtype, seed=T + nv, reset=0.01 if T > 1 else 0)
    got = off(A.backward(Ops(0), x, nk, nv)[3], reference(x, nk, nv))
    assert got <= most_off(T, nk, nv), f"{got:.3g}, more than {most_off(T, nk, nv):.3g}"


@pytest.mark.parametrize("T, B, H, nk, nv", SIZES[1:4])
def test_faults_that_it_sees(monkeypatch, T, B, H, nk, nv):
    """States rounded to bf16, and a hundredth too much; three pieces of bf16 are within."""
    monkeypatch.setattr(torch.Tensor, "cuda", lambda t, *a, **k: t)
    x = A.inputs(T, B, H, nk, nv, A.BF16, seed=T + nv, reset=0.01)
    want = reference(x, nk, nv)
    bound = most_off(T, nk, nv)
    assert off(want.float(), want) < bound < off(1.01 * want, want)
    do, q, k, v = (R.split(x[n], m, H) for n, m in (("do", nv), ("q", nk), ("k", nk), ("v", nv)))
    a, age = R.gates(x["g"], x["reset"])
    S = R.sweep(q, k, v, a, age, R.d64(x["s0"]))[2]
    E = R.sweep(k, nk ** -0.5 * q, do, a, age, R.d64(x["ds"]), back=True)[2][::-1]
    before = [R.d64(x["s0"])] + [s for s, _, _ in S[:-1]]

    def cut(s, pieces):
        out = torch.zeros_like(s)
        for _ in range(pieces):
            out = out + (s - out).to(torch.bfloat16).double()
        return out

    for pieces, seen in ((1, True), (3, False)):
        dg = torch.stack([a[t] * (cut(E[t][0], pieces) * cut(before[t], pieces)).sum((-1, -2)) for t in range(T)])
        assert (off(dg, want) > bound) == seen, (pieces, off(dg, want), bound)
