"""Operators of sequence policies on the device, over the C ABI of
phyz_amd/csrc/phz_scan.hip, phz_linear.hip and phz_muon.hip.

A policy with memory is a stack of blocks: a linear layer into gates and
values, a gated linear recurrence over the rollout's steps, and a linear layer
back with the residual. These are those operators with their gradients, the
recurrence's single step for acting, and the orthogonalised (Muon) update of
weight matrices:

    ops = Ops(device=0)
    pre = ops.linear(x, w_in, bias=b_in)                      # gates and values
    h, h_last = ops.gated_scan(pre[..., :n], pre[..., n:], h0=h0, reset=reset)
    y = ops.linear(h, w_out, residual=x)
    dh, dw_out, _ = ops.linear_backward(dy, h, w_out)
    dz, dx, dh0 = ops.gated_scan_backward(dh, z, x, h, h0=h0, reset=reset)
    ops.muon_step(w_out, dw_out, momentum_out, lr=0.02)

Arguments are torch tensors on the handle's GPU; calls enqueue their work on
torch's current stream and return without waiting. Errors raise OpsError with
the library's message. There is no host fallback: the kernels run on a HIP
device or not at all. Ops(device=-1) checks arguments only (of CPU tensors)
and then raises.

Autograd records none of this: gradients come from the _backward calls. The
forward operators refuse tensors that require gradients while it is recording
(call them under torch.no_grad(), or on detached tensors); the _backward calls
and muon_step take them as they are. What a call writes in place or into `out`
counts as changed for graphs that saved it.
"""
from __future__ import annotations

import ctypes as C
import math
import os

import torch

from . import _lib

FORMS = {"sigmoid": 0, "decay": 1}
ACTS = {"none": 0, "tanh": 1, "relu": 2, "silu": 3, "gelu": 4}
# Muon's quintic: five steps take singular values in about (0.002, 1) to within
# 0.7 to 1.2.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

_DTYPES = (torch.float32, torch.float64, torch.bfloat16, torch.uint8, torch.bool)
# The entry points, in the order of phz_describe.cpp's table.
_ENTRIES = ("phz_gated_scan", "phz_gated_scan_backward", "phz_gated_step", "phz_linear", "phz_linear_backward",
            "phz_orthogonalize", "phz_muon_step")
_SCAN, _SCAN_BACKWARD, _STEP, _LINEAR, _LINEAR_BACKWARD, _ORTHOGONALIZE, _MUON = range(7)
_describe = None


def _bound():
    """The module that hands tensors to the library, bound to its entry points."""
    global _describe
    if _describe is None:
        if not os.path.exists(os.path.join(_lib.HERE, "_describe.so")):
            raise ImportError("phyz_amd/_describe.so is not built; run `python -m phyz_amd.build`")
        from . import _describe as module
        L = _lib.load()
        module.bind(tuple(C.cast(getattr(L, name), C.c_void_p).value for name in _ENTRIES), _DTYPES)
        _describe = module
    return _describe


def _current_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The same without the Stream object, where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


# Tells autograd that tensors were written to, so that a graph which saved their
# values refuses to use them.
_written = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


class OpsError(RuntimeError):
    pass


class Ops:
    """A handle: one GPU's operators and their workspaces, one per stream and one
    per captured graph. A handle whose workspace a captured graph holds is kept to
    the end of the process, so that the graph outlives the last reference to it."""

    def __init__(self, device: int = 0):
        self._L = _lib.load()
        self._call = _bound().call
        self.device = int(device)
        h = C.c_void_p()
        if self._L.phz_ops_create(self.device, C.byref(h)) != 0:
            raise OpsError(self._L.phz_ops_last_error(None).decode())
        self._h = h.value

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            if not self._L.phz_ops_graph_bytes(h):
                self._L.phz_ops_destroy(h)
            self._h = None

    # ── calls ──
    def _run(self, op: int, head: int, names: str, *tensors):
        """One entry point on the current stream; `names` are the tensors'."""
        stream = _raw_stream(self.device) if self.device >= 0 else 0
        rc = self._call(op, self._h, stream, self.device, head, tensors, False)
        if rc < -100:
            if torch.is_grad_enabled():
                raise OpsError(f"{names.split()[-101 - rc]} requires gradients, which these operators do not record: call under "
                               "torch.no_grad() or with detach(), and take the gradients from the _backward calls")
            rc = self._call(op, self._h, stream, self.device, head, tensors, True)
        if rc > 0:
            raise OpsError(self._L.phz_ops_last_error(self._h).decode())
        if rc < 0:
            self._complain(names.split()[-1 - rc], tensors[-1 - rc])

    def _complain(self, name: str, t):
        if not isinstance(t, torch.Tensor):
            raise OpsError(f"{name} has to be a torch tensor, not {type(t).__name__}")
        if t.get_device() != self.device:
            where = "a host-only handle checks CPU tensors" if self.device < 0 else f"the handle's GPU is cuda:{self.device}"
            raise OpsError(f"{name} is on {t.device}: {where}")
        if t.dtype not in _DTYPES:
            raise OpsError(f"{name} is {t.dtype}, expected float32, bfloat16 or a mask of uint8 or bool")
        if not 1 <= t.dim() <= 3:
            raise OpsError(f"{name} has {t.dim()} dimensions, expected 1 to 3")
        raise OpsError(f"{name} has no strided memory to read here (a sparse tensor, or one inside vmap or a trace)")

    def _stream(self):
        return _raw_stream(self.device) if self.device >= 0 else None

    def _check(self, rc: int):
        if rc != 0:
            raise OpsError(self._L.phz_ops_last_error(self._h).decode())

    @staticmethod
    def _tensor(t, name: str):
        if not isinstance(t, torch.Tensor):
            raise OpsError(f"{name} has to be a torch tensor, not {type(t).__name__}")
        return t

    @staticmethod
    def _choice(table, key, what):
        try:
            return table[key]
        except (KeyError, TypeError):
            raise OpsError(f"unknown {what} {key!r}, expected one of {', '.join(table)}") from None

    # ── workspaces ──
    def reserve(self, nbytes: int):
        """Grows the current stream's workspace, as before a graph capture."""
        self._check(self._L.phz_ops_reserve(self._h, self._stream(), int(nbytes)))

    @property
    def workspace_bytes(self) -> int:
        return int(self._L.phz_ops_workspace_bytes(self._h))

    # ── the gated linear recurrence ──
    def gated_scan(self, z, x, h0=None, reset=None, form: str = "sigmoid", out=None):
        """h_t = c_t h_{t-1} + u_t over z, x [steps, worlds, width]; (h, the last
        state in float32). c = sigmoid(z), u = (1 - c) x ("sigmoid") or c = z,
        u = x ("decay"). Batch-major tensors come as transposed views. h0
        [worlds, width] float32, zeros if None; where reset [steps, worlds] is
        set an episode begins and h_{t-1} counts as 0."""
        f = self._choice(FORMS, form, "gate form")
        if out is not None:
            h, last = out
        else:
            h = torch.empty_like(self._tensor(x, "x"))
            last = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        self._run(_SCAN, f, "z x h0 reset h h_last", z, x, h0, reset, h, last)
        if out is not None:
            _written([t for t in out if t is not None])
        return h, last

    def gated_scan_backward(self, dh, z, x, h, h0=None, reset=None, dh_last=None, form: str = "sigmoid", out=None):
        """The gradients (dz, dx, dh0) of gated_scan, from those of h and of the
        last state (None: zero) and the stored h. dh0 is float32."""
        f = self._choice(FORMS, form, "gate form")
        if out is not None:
            dz, dx, dh0 = out
        else:
            dz, dx = torch.empty_like(self._tensor(z, "z")), torch.empty_like(self._tensor(x, "x"))
            dh0 = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        self._run(_SCAN_BACKWARD, f, "dh dh_last z x h h0 reset dz dx dh0", dh, dh_last, z, x, h, h0, reset, dz, dx, dh0)
        if out is not None:
            _written([t for t in out if t is not None])
        return dz, dx, dh0

    def gated_step(self, z, x, h, reset=None, form: str = "sigmoid"):
        """One step for z, x [worlds, width]: h [worlds, width] float32 is
        replaced, and returned."""
        f = self._choice(FORMS, form, "gate form")
        self._run(_STEP, f, "z x reset h", z, x, reset, h)
        _written((h,))
        return h

    # ── the linear layer ──
    @staticmethod
    def _rows(t):
        if not isinstance(t, torch.Tensor) or t.dim() <= 2:
            return t
        return t.reshape(math.prod(t.shape[:-1]), t.shape[-1])  # -1 says nothing where no element is

    def linear(self, x, w, bias=None, act: str = "none", residual=None, save_pre: bool = False, out=None):
        """y = act(x w^T + bias) + residual for x [..., n_in], w [n_out, n_in];
        with save_pre, (y, x w^T + bias). All of one type, float32 or bfloat16.
        `out` (2-D) may be the residual."""
        a = self._choice(ACTS, act, "activation")
        x2, r2 = self._rows(self._tensor(x, "x")), self._rows(residual)
        if x.dim() < 2:
            raise OpsError(f"x has {x.dim()} dimensions, expected 2 or more")
        if self._tensor(w, "w").dim() != 2:
            raise OpsError(f"w has {w.dim()} dimensions, expected 2")
        y = out if out is not None else torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device)
        pre = torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device) if save_pre else None
        self._run(_LINEAR, a, "x w bias residual pre y", x2, w, bias, r2, pre, y)
        if out is not None:
            _written((y,))
        shape = (*x.shape[:-1], w.shape[0])
        if out is None and x.dim() != 2:
            y = y.view(shape)
        return (y, pre.view(shape)) if save_pre else y

    def linear_backward(self, dy, x, w, pre=None, act: str = "none", need_dx: bool = True, need_dw: bool = True,
                        need_db: bool = True):
        """The gradients (dx, dw, db) of linear for dz = dy act'(pre); those not
        needed are None. The residual's gradient is dy itself."""
        a = self._choice(ACTS, act, "activation")
        x2, dy2, p2 = self._rows(self._tensor(x, "x")), self._rows(dy), self._rows(pre)
        if self._tensor(w, "w").dim() != 2:
            raise OpsError(f"w has {w.dim()} dimensions, expected 2")
        dx = torch.empty(x2.shape, dtype=x.dtype, device=x.device) if need_dx else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if need_dw else None
        db = torch.empty(w.shape[:1], dtype=w.dtype, device=w.device) if need_db else None
        self._run(_LINEAR_BACKWARD, a, "dy x w pre dx dw db", dy2, x2, w, p2, dx, dw, db)
        return (dx.view(x.shape) if need_dx else None), dw, db

    # ── the orthogonalised update ──
    @staticmethod
    def _muon(steps, coef, eps, lr=0.0, momentum=0.0, nesterov=True, weight_decay=0.0):
        a, b, c = coef
        return _lib.MuonCfg(a, b, c, eps, lr, momentum, weight_decay, int(steps), int(bool(nesterov)))

    def orthogonalize(self, g, steps: int = 5, coef=NEWTON_SCHULZ, eps: float = 1e-7, out=None):
        """Each [rows, cols] matrix of g after `steps` Newton-Schulz steps from
        g / (|g|_F + eps): nearly the orthogonal factor of g."""
        cfg = self._muon(steps, coef, eps)
        o = out if out is not None else torch.empty_like(self._tensor(g, "g"))
        self._run(_ORTHOGONALIZE, C.addressof(cfg), "g o", g, o)
        if out is not None:
            _written((o,))
        return o

    def muon_step(self, w, g, m, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                  weight_decay: float = 0.0, steps: int = 5, coef=NEWTON_SCHULZ, eps: float = 1e-7):
        """Muon's update of w (and the momentum m, both float32, in place) for
        the gradient g: matrices [rows, cols], or a batch of them."""
        cfg = self._muon(steps, coef, eps, lr, momentum, nesterov, weight_decay)
        self._run(_MUON, C.addressof(cfg), "w g m", w, g, m)
        _written((w, m))
