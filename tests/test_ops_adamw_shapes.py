"""AdamW's gradients have their weights' shapes, or are vectors: on a handle without a
GPU."""
import pytest
import torch

from phyz_amd.ops import Ops, OpsError


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def step(ops, w, g):
    flat = [torch.zeros(torch.Size(s).numel()) for s in w]
    ops.adamw_step([torch.zeros(s) for s in w], [torch.zeros(s) for s in g], flat, [t.clone() for t in flat],
                   torch.zeros(1, dtype=torch.int64))


@pytest.mark.parametrize("w, g", [((2, 3), (3, 2)), ((2, 3, 4), (6, 4)), ((4, 6), (2, 3, 4)), ((1, 2, 3), (3, 1, 2)),
                                  ((2, 2, 3), (2, 3, 2)), ((2, 6), (2, 3, 2))])
def test_other_shapes_are_refused(ops, w, g):
    message = rf"g\[1\] has the shape \({', '.join(map(str, g))}\), w\[1\] \({', '.join(map(str, w))}\)"
    with pytest.raises(OpsError, match=message):
        step(ops, [(5,), w, (2, 2)], [(5,), g, (2, 2)])


@pytest.mark.parametrize("w, g", [((2, 3), (2, 3)), ((2, 3), (6,)), ((6,), (2, 3)), ((1, 2, 3), (2, 1, 3)), ((), (1, 1)), ((1,), ()),
                                  ((5, 1), (1, 5)), ((0, 3), (3, 0)), ((0, 3), (0, 3)), ((2, 3, 4), (2, 1, 3, 4)), ((1, 6), (2, 3))])
def test_the_same_places_are_taken(ops, w, g):
    with pytest.raises(OpsError, match="host-only"):
        step(ops, [w, (4, 4)], [g, (4, 4)])


def test_what_is_no_tensor_is_named(ops):
    one = [torch.zeros(2, 3)]
    for w, g, name in (([3], one, "w"), (one, [3], "g"), (one, [torch.zeros(3, 2).t()], "g")):
        with pytest.raises(OpsError, match=rf"{name}\[0\]"):
            ops.adamw_step(w, g, one, [torch.ones(2, 3)], torch.zeros(1, dtype=torch.int64))
    with pytest.raises(OpsError, match=r"g\[0\] has 4 elements along axis 0, expected 6"):
        ops.adamw_step(one, [torch.zeros(2, 2)], [torch.zeros(6)], [torch.ones(6)], torch.zeros(1, dtype=torch.int64))
