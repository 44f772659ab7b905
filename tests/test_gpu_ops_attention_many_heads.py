"""Linear attention of more heads of all worlds than a launch has workgroups for."""
import pytest
import torch

from tests import test_gpu_ops_attention as A

pytestmark = pytest.mark.gpu
ops = A.ops


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
def test_steps_of_many_heads(ops, dtype):
    """2^24 and some more heads of one element each, in rows with gaps."""
    B, H = (1 << 22) + 3, 5
    gen = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    q, k, v = (rnd(B, H + 1).to(dtype)[:, :H] for _ in range(3))
    g, s0, reset = -rnd(B, H).abs(), rnd(B, H, 1, 1), torch.rand(B, device="cuda", generator=gen) < 0.1
    s = s0.clone()
    o = ops.linear_attention_step(q, k, v, g, s, reset=reset, scale=0.5)
    a = torch.where(reset[:, None], 0.0, g.double().exp())
    want = a * s0[..., 0, 0].double() + k.double() * v.double()
    size = a * s0[..., 0, 0].double().abs() + (k.double() * v.double()).abs()
    # exp to 2^-23 of itself and its argument's 2^-24, a product, a sum: (4 + |g|) U.
    off = 2.0 ** -24 * (4 + g.double().abs()) * size + 1e-37
    assert bool(((s[..., 0, 0].double() - want).abs() <= off).all())
    out = 0.5 * q.double() * want
    step = 2.0 ** -24 if dtype == A.F32 else 2.0 ** -8
    assert bool(((o.double() - out).abs() <= 0.5 * q.double().abs() * 2 * off + 1.01 * step * out.abs() + 1e-37).all())


@pytest.mark.parametrize("dtype", [A.F32, A.BF16], ids=["f32", "bf16"])
def test_rollouts_of_many_heads(ops, dtype):
    """2^22 and some more: the same as the last worlds alone, to the bit, and as the
    bounds for those and the first ones. Batch-major, q shared."""
    T, B, H, n = 2, (1 << 20) + 3, 5, 2
    gen = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = {"q": rnd(B, T, n).to(dtype).transpose(0, 1), "k": rnd(T, B, H * n).to(dtype), "v": rnd(T, B, H).to(dtype),
         "g": -rnd(T, B, H).abs(), "s0": rnd(B, H, n, 1), "reset": torch.rand(T, B, device="cuda", generator=gen) < 0.1,
         "do": rnd(T, B, H).to(dtype), "ds": rnd(B, H, n, 1)}
    whole = (*A.forward(ops, x, n, 1), *A.backward(ops, x, n, 1))
    state = {"s0", "ds"}
    for part in (slice(0, 1000), slice(838860 - 500, 838860 + 500), slice(B - 1000, B)):
        y = {m: t[part] if m in state else t[:, part] for m, t in x.items()}
        alone = (*A.forward(ops, y, n, 1), *A.backward(ops, y, n, 1))
        for i, (a, b) in enumerate(zip(whole, alone)):
            assert torch.equal(a[part] if i in (1, 6) else a[:, part], b), i
        A.check_forward(alone[:2], y, n, 1)
        A.check_backward(alone[2:], y, n, 1)
    last = ops.linear_attention(x["q"][:0], x["k"][:0], x["v"][:0], x["g"][:0], s0=x["s0"], size_k=n, size_v=1)[1]
    assert torch.equal(last, x["s0"])


def test_no_steps_of_many_heads(ops):
    B, H = (1 << 24) + 5, 1
    none = torch.empty(0, B, H, device="cuda")
    s0 = torch.arange(B, device="cuda").float().view(B, H, 1, 1)
    assert torch.equal(ops.linear_attention(none, none, none, none, s0=s0)[1], s0)
