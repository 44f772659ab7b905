"""Which views of one buffer the sequence operators take as apart, on a handle
without a GPU: never two that share an element, and not refused are those that
lie beside each other within a stride."""
import random

import pytest
import torch

from phyz_amd.ops import Ops, OpsError

F32 = torch.float32


@pytest.fixture(scope="module")
def ops():
    return Ops(device=-1)


def taken(call):
    """True where only the missing device is refused, False for an overlap."""
    with pytest.raises(OpsError) as e:
        call()
    message = str(e.value)
    assert "host-only" in message or "overlaps" in message, message
    return "host-only" in message


@pytest.mark.parametrize("T, B, D", [(6, 3, 5), (1, 2, 4), (7, 1, 1)])
def test_a_record_of_states(ops, T, B, D):
    """Worlds' states in one record [worlds, steps + 1, width]: the first is h0, the
    others are written, or the last is h_last."""
    z = torch.zeros(T, B, D)
    record = torch.zeros(B, T + 1, D)
    later, first = record[:, 1:].transpose(0, 1), record[:, 0]
    last = torch.zeros(B, D)
    assert taken(lambda: ops.gated_scan(z, z.clone(), h0=first, out=(later, last)))
    assert taken(lambda: ops.gated_scan(z, z.clone(), out=(record[:, :T].transpose(0, 1), record[:, T])))
    assert not taken(lambda: ops.gated_scan(z, z.clone(), h0=record[:, 1], out=(later, last)))
    assert not taken(lambda: ops.gated_scan(z, z.clone(), out=(record[:, :T].transpose(0, 1), record[:, T - 1])))


def test_columns_of_a_wide_buffer(ops):
    """Outputs between the columns of inputs of other widths and row strides."""
    wide = torch.zeros(8, 30)
    assert taken(lambda: ops.linear(wide[:, :7], torch.zeros(9, 7), residual=wide[:, 7:16], out=wide[:, 16:25]))
    assert taken(lambda: ops.linear(wide[::2, :7], torch.zeros(9, 7), out=wide[1::2, 3:12]))
    assert taken(lambda: ops.linear(wide[:4, :7], torch.zeros(9, 7), out=wide[::2, 16:25]))
    assert not taken(lambda: ops.linear(wide[:4, :7], torch.zeros(9, 7), out=wide[::2, 6:15]))


def test_random_views_against_their_elements(ops):
    """No two views that share an element pass, of random sizes, strides and offsets;
    of equal strides, all that share none do."""
    rng = random.Random(4)
    buffer = torch.zeros(4000)
    seen = [0, 0, 0]
    while min(seen) < 300:
        rows, cols = rng.randint(1, 6), rng.randint(1, 5)
        batch = rng.randint(1, 3)

        def view(strides):
            return torch.as_strided(buffer, (batch, rows, cols), (*strides, 1), rng.randint(0, 60))

        def steps():
            row = rng.randint(cols, 14)
            return row * rng.randint(rows, rows + 4) if rng.random() < 0.7 else row * rows + rng.randint(0, 5), row

        out_steps = steps()
        equal = rng.random() < 0.5
        o, g = view(out_steps), view(out_steps if equal else steps())

        def elements(v):
            at = torch.arange(4000).as_strided(v.shape, v.stride(), v.storage_offset())
            return set(at.flatten().tolist())

        share = bool(elements(o) & elements(g))
        ok = taken(lambda: ops.orthogonalize(g, out=o))
        assert not (ok and share), (o.shape, o.stride(), o.storage_offset(), g.stride(), g.storage_offset())
        seen[0] += share
        seen[1] += ok
        if equal and out_steps[0] % out_steps[1] == 0 and not share and batch * rows > 1:
            # Within a row's stride beside each other, or one wholly after the other,
            # or rows between rows: the first two are taken.
            off = (g.storage_offset() - o.storage_offset()) % out_steps[1]
            if off >= cols and out_steps[1] - off >= cols and rows > 1:
                assert ok
                seen[2] += 1
