"""The recurrent policy with a matrix memory, and AdamW over all its parameters:
linear layers, rotary positions, linear attention and the update together."""
import pytest
import torch

from tests import attend_ref as R
from tests.test_gpu_recurrent import task

pytestmark = pytest.mark.gpu
CASES = [("attention", "muon", 32), ("attention", "adamw", 32), ("attention", "adamw", 8), ("gates", "adamw", 8)]


def policy_of(*args, **kw):
    from phyz_amd.recurrent import RecurrentPolicy
    return RecurrentPolicy(*args, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("memory, optimizer, bits", CASES)
def test_trains_and_acts(memory, optimizer, bits, dtype):
    """Updates change every parameter and leave all of them finite."""
    obs, actions, reset = task()
    policy = policy_of(11, 48, 3, seed=1, memory=memory, heads=3, optimizer=optimizer, moment_bits=bits, dtype=dtype)
    start = {k: v.clone() for k, v in [*policy.w.items(), *(("b_" + k, v) for k, v in policy.b.items())]}
    for _ in range(3):
        loss = policy.imitate(obs, actions, reset=reset)
        assert bool(torch.isfinite(loss))
    for k, v in start.items():
        now = policy.b[k[2:]] if k.startswith("b_") else policy.w[k]
        assert bool(torch.isfinite(now).all()) and not torch.equal(now, v), k
    policy.begin(64)
    assert bool(torch.isfinite(policy.act(obs[0], reset[0])).all())


@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 1e-1)], ids=["f32", "bf16"])
def test_acting_is_the_attention_step_by_step(dtype, tol):
    """The same actions either way. f32: sums of up to 100 terms of size up to 10 in
    another order, 100 * 10 * 2^-24 in all, and angles within 2^-22. bf16: outputs
    are rounded once either way, so neighbours differ by a unit, 2^-8 of 8, and pass
    two more products."""
    obs, _, reset = task(worlds=70)
    policy = policy_of(11, 96, 3, dtype=dtype, seed=2, memory="attention", heads=4)
    whole, _ = policy.forward(obs, reset)
    policy.begin(70)
    for t in range(obs.shape[0]):
        assert float((policy.act(obs[t], reset[t]).float() - whole[t].float()).abs().max()) <= tol


def test_a_rollout_in_two_parts():
    """The memory behind the first part is where the second begins."""
    obs, _, reset = task(steps=50, worlds=9)
    policy = policy_of(11, 64, 3, seed=3, memory="attention", heads=2)
    whole, _ = policy.forward(obs, reset)
    first, c = policy.forward(obs[:23], reset[:23])
    second, _ = policy.forward(obs[23:], reset[23:], h0=c["last"])
    assert float((torch.cat([first, second]) - whole).abs().max()) <= 2e-5


def test_forward_against_64_bits():
    """The whole policy from its formulas, in 64 bits."""
    obs, _, reset = task(steps=30, worlds=5)
    policy = policy_of(11, 48, 3, seed=4, memory="attention", heads=2)
    got, _ = policy.forward(obs, reset)
    w = {k: v.double().cpu() for k, v in policy.w.items()}
    b = {k: v.double().cpu() for k, v in policy.b.items()}
    x = torch.tanh(obs.double().cpu() @ w["embed"].T + b["embed"])
    y = x @ w["gate"].T + b["gate"]
    n, size = 48, 24
    freq = 10000.0 ** (-torch.arange(size // 2, dtype=torch.float64) * 2 / size)
    s = torch.zeros(5, 2, size, size, dtype=torch.float64)
    place, out = torch.zeros(5, dtype=torch.int64), []
    for t in range(30):
        place = torch.where(reset[t].cpu(), 0, place)
        turn = torch.exp(1j * place[:, None, None] * freq)

        def turned(v):
            v = v.reshape(5, 2, size)
            z = torch.complex(v[..., :size // 2], v[..., size // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k, v = turned(y[t, :, :n]), turned(y[t, :, n:2 * n]), y[t, :, 2 * n:3 * n].reshape(5, 2, size)
        a = torch.sigmoid(y[t, :, 3 * n:]) * (~reset[t].cpu()).double()[:, None]
        s = a[..., None, None] * s + k[..., :, None] * v[..., None, :]
        out.append((q[..., None, :] @ s)[..., 0, :].reshape(5, n) * size ** -0.5)
        place = place + 1
    h = x + torch.stack(out) @ w["out"].T + b["out"]
    want = h @ w["act"].T + b["act"]
    # Four layers' sums of up to 100 terms, each result's relative error below 100 * 2^-24.
    assert float((got.double().cpu() - want).abs().max()) <= 4 * 100 * R.U32 * float(want.abs().max() + 10)


def test_gradients_against_differences():
    """Each parameter's gradient along a random direction against the loss's central
    difference: f32 sums over 40 x 64 x 3 errors, step 1e-3 of unit directions, 2e-3
    of the gradient's size."""
    obs, actions, reset = task()
    policy = policy_of(11, 32, 3, seed=3, memory="attention", heads=2)

    def loss():
        a, c = policy.forward(obs, reset)
        return float((a.double() - actions.double()).square().sum()), a, c

    _, a, c = loss()
    grads = policy.backward(2 * (a - actions), c)
    gen = torch.Generator().manual_seed(4)
    for name in grads:
        p = policy.b[name[2:]] if name.startswith("b_") else policy.w[name]
        d = torch.randn(p.shape, generator=gen).cuda()
        d /= d.norm()
        keep, s = p.clone(), 1e-3
        p.copy_(keep + s * d)
        up = loss()[0]
        p.copy_(keep - s * d)
        down = loss()[0]
        p.copy_(keep)
        along = float((grads[name].double() * d.double()).sum())
        assert abs((up - down) / (2 * s) - along) <= 2e-3 * float(grads[name].double().norm()), name


def test_a_captured_update_is_the_eager_one():
    """Forward, backward and AdamW in one graph, replayed between eager work."""
    obs, actions, reset = task(steps=20, worlds=16)
    kw = {"seed": 5, "memory": "attention", "heads": 2, "optimizer": "adamw", "moment_bits": 8}
    eager, captured = policy_of(11, 32, 3, **kw), policy_of(11, 32, 3, **kw)

    def step(p):
        a, c = p.forward(obs, reset)
        p.update(p.backward((a - actions) * 0.01, c))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured)
    torch.cuda.current_stream().wait_stream(side)
    step(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(captured)
    for _ in range(4):
        graph.replay()
        step(eager)
        torch.cuda.synchronize()
        for k in eager.w:
            assert torch.equal(eager.w[k], captured.w[k]) and torch.equal(eager.b[k], captured.b[k]), k
