"""AdamW's largest tensors, by descriptions alone: on a handle without a GPU."""
import ctypes as C

import pytest

from phyz_amd import _lib


class Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("size", C.c_int64 * 3), ("stride", C.c_int64 * 3), ("dtype", C.c_int32), ("ndim", C.c_int32)]


def vector(size, dtype, at):
    return Tensor(at, (size, 0, 0), (1, 0, 0), dtype, 1)


@pytest.mark.parametrize("size, message", [(((1 << 24) - 1) * 4096, b"host-only handle (device -1)"),
                                           (((1 << 24) - 1) * 4096 + 1, b"w[0] is too large")])
def test_a_tensor_s_workgroups_fit_a_launch(size, message):
    """Fewer than 2^32 threads, 256 for 4096 elements."""
    L = _lib.load()
    h = C.c_void_p()
    assert L.phz_ops_create(-1, C.byref(h)) == 0
    cfg = _lib.AdamWCfg(0.1, 0.9, 0.99, 1e-8, 0.0, 0)
    w, g, m, v = (vector(size, 0, (i + 1) << 44) for i in range(4))
    step = vector(1, 5, 1 << 40)
    assert L.phz_adamw_step(h, None, C.byref(cfg), 1, *[C.byref(t) for t in (w, g, m, v)], None, C.byref(step)) != 0
    assert L.phz_ops_last_error(h) == message
    L.phz_ops_destroy(h)
