"""The recurrent policy: its operators together, as a program uses them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def task(steps=40, worlds=64, n_in=11, n_out=3, seed=0):
    """Actions that follow a leaky average of past observations: nothing that one
    step's observation tells."""
    g = torch.Generator().manual_seed(seed)
    obs = torch.randn(steps, worlds, n_in, generator=g)
    reset = torch.rand(steps, worlds, generator=g) < 0.05
    reset[0] = True
    mix = torch.randn(n_in, n_out, generator=g) / n_in ** 0.5
    h, out = torch.zeros(worlds, n_in), []
    for t in range(steps):
        h = torch.where(reset[t][:, None], 0.0, h) * 0.8 + 0.2 * obs[t]
        out.append(h @ mix)
    return obs.cuda(), torch.stack(out).cuda(), reset.cuda()


def test_learns_what_needs_memory():
    from phyz_amd.recurrent import RecurrentPolicy
    obs, actions, reset = task()
    policy = RecurrentPolicy(11, 64, 3, seed=1)
    losses = [float(policy.imitate(obs, actions, reset=reset, lr=0.02 * (1 - k / 200))) for k in range(200)]
    assert losses[-1] < 0.1 * float(actions.var()) < losses[0]


@pytest.mark.parametrize("dtype, tol", [(torch.float32, 1e-5), (torch.bfloat16, 6e-2)], ids=["f32", "bf16"])
def test_acting_is_the_scan_step_by_step(dtype, tol):
    """The same actions either way: in f32 up to the order of sums; in bf16 the
    scan's states are rounded where they are stored, a step's when they are used,
    and the products' inputs in both: a few units of 2^-8 of sums of size 1 to 4."""
    from phyz_amd.recurrent import RecurrentPolicy
    obs, _, reset = task(worlds=70)
    policy = RecurrentPolicy(11, 96, 3, dtype=dtype, seed=2)
    whole, _ = policy.forward(obs, reset)
    policy.begin(70)
    for t in range(obs.shape[0]):
        assert float((policy.act(obs[t], reset[t]).float() - whole[t].float()).abs().max()) <= tol


def test_gradients_against_differences():
    """Each parameter's gradient along a random direction against the loss's
    central difference: f32 sums over 40 x 64 x 3 errors, step 1e-3 of unit
    directions, 2e-3 of the gradient's size."""
    from phyz_amd.recurrent import RecurrentPolicy
    obs, actions, reset = task()
    policy = RecurrentPolicy(11, 32, 3, seed=3)

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
