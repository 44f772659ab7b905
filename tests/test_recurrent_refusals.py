"""What the recurrent policy refuses, before it needs a GPU."""
import pytest

from phyz_amd.ops import OpsError
from phyz_amd.recurrent import RecurrentPolicy


@pytest.mark.parametrize("kw, message", [
    ({"memory": "lstm"}, "unknown memory 'lstm'"),
    ({"optimizer": "sgd"}, "optimizer 'sgd'"),
    ({"memory": "attention", "heads": 5}, "heads of an even size have to divide the width 32, not 5"),
    ({"memory": "attention", "heads": 32}, "not 32"),
    ({"memory": "attention", "heads": 0}, "not 0"),
    ({"memory": "attention", "heads": 1, "width": 258}, "at most 128"),
    ({"optimizer": "adamw", "moment_bits": 16}, "32 or 8 bits, not 16"),
])
def test_refusals(kw, message):
    kw = {"width": 32, **kw}
    with pytest.raises(OpsError, match=message):
        RecurrentPolicy(4, kw.pop("width"), 2, **kw)
