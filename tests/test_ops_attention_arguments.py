"""Arguments of the attending operators that are of the wrong kind altogether: an
OpsError that names them, on a handle without a GPU."""
import pytest
import torch

from phyz_amd.ops import Ops, OpsError

F32, I64, F64 = torch.float32, torch.int64, torch.float64


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def t(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def attend(o, v=(6, 2, 15), g=(6, 2, 3), **kw):
    return o.linear_attention(t(6, 2, 12), t(6, 2, 12), t(*v), t(*g) if g is not None else None, **kw)


def rot(o, **kw):
    return o.rotary(t(4, 2, 12), t(4, 2, dtype=I64), t(2, dtype=F64), **kw)


def adamw(o, w="", **kw):
    one = [t(5)]
    return o.adamw_step([t(5)] if w == "" else w, [t(5)], one, [t(5)], t(1, dtype=I64), **kw)


@pytest.mark.parametrize("call, message", [
    (lambda o: attend(o, g=()), "g has 0 dimensions, expected 3"),
    (lambda o: attend(o, v=()), "v has 0 dimensions, expected 3"),
    (lambda o: attend(o, g=None), "g has to be a torch tensor"),
    (lambda o: attend(o, size_k=1.5), "size_k has to be a whole number, not 1.5"),
    (lambda o: attend(o, size_v="5"), "size_v has to be a whole number, not '5'"),
    (lambda o: attend(o, size_v=1 << 32), "size_v has to be a whole number"),
    (lambda o: attend(o, scale="much"), "scale has to be a number, not 'much'"),
    (lambda o: o.linear_attention_step(t(2, 12), t(2, 12), t(), t(2, 3), t(2, 3, 4, 5)), "v has 0 dimensions, expected 2"),
    (lambda o: o.linear_attention_step(t(2, 12), t(2, 12), t(2, 15), t(), t(2, 3, 4, 5)), "g has 0 dimensions, expected 2"),
    (lambda o: o.linear_attention_backward(t(6, 2, 15), t(6, 2, 12), t(6, 2, 12), t(6, 2, 15), t()), "g has 0 dimensions, expected 3"),
    (lambda o: rot(o, heads=1.5), "heads has to be a whole number, not 1.5"),
    (lambda o: rot(o, heads=(1 << 32) + 1), "heads has to be a whole number"),
    (lambda o: rot(o, heads=None), "heads has to be a whole number, not None"),
    (lambda o: rot(o, scale=None), "scale has to be a number, not None"),
    (lambda o: adamw(o, w=None), "w has to be a list of tensors, not NoneType"),
    (lambda o: adamw(o, betas=0.9), "betas have to be two numbers"),
    (lambda o: adamw(o, betas=(0.9, "a")), "betas has to be a number, not 'a'"),
    (lambda o: adamw(o, lr="fast"), "lr has to be a number, not 'fast'"),
    (lambda o: adamw(o, seed="a"), "seed has to be a whole number, not 'a'"),
    (lambda o: o.adamw_values(None, [t(5)], [t(2, 1)], out=([t(5)], [t(5)])), "m has to be a list of tensors, not NoneType"),
    (lambda o: o.adamw_state([3.0]), "params has to be a torch tensor"),
])
def test_refusals(ops, call, message):
    with pytest.raises(OpsError, match=message):
        call(ops)


def test_numbers_of_other_types_are_taken(ops):
    for call in (lambda: rot(ops, heads=3.0), lambda: rot(ops, heads=torch.tensor(3), scale=torch.tensor(2.0)),
                 lambda: attend(ops, size_k=torch.tensor(4), scale=1), lambda: adamw(ops, betas=[0, torch.tensor(0.5)], seed=-1)):
        with pytest.raises(OpsError, match="host-only"):
            call()
