"""AdamW with an eps that f32 does not hold."""
import pytest
import torch

from tests import attend_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-37, 1e-39, 1e-45, 1e-60])
def test_weights_without_gradients_decay_alone(eps, bits):
    """0 / (sqrt(0) + eps) is 0; beside them, steps as ever."""
    from phyz_amd.ops import Ops
    ops = Ops(0)
    gen = torch.Generator().manual_seed(1)
    w, g = [torch.randn(700, generator=gen).cuda()], [torch.randn(700, generator=gen).cuda()]
    g[0][::3] = 0
    start = w[0].clone()
    m, v, e, step = ops.adamw_state(w, bits=bits)
    ops.adamw_step(w, g, m, v, step, exponents=e, lr=1e-2, betas=(0.9, 0.99), eps=eps, weight_decay=0.1)
    want, bound = R.adamw(start, g[0], torch.zeros(700), torch.zeros(700), 1, 1e-2, (0.9, 0.99), eps, 0.1)
    R.within(w[0], want[0], bound[0], "w")
