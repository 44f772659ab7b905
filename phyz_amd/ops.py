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
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib

FORMS = {"sigmoid": 0, "decay": 1}
ACTS = {"none": 0, "tanh": 1, "relu": 2, "silu": 3, "gelu": 4}
# Muon's quintic: five steps take singular values in about (0.002, 1) to within
# 0.7 to 1.2.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

_DTYPES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.uint8: 3, torch.bool: 3}
_TENSOR = struct.Struct("=q3q3qii")  # phz_tensor, 64 bytes
_PACK = _TENSOR.pack_into
_SLOTS = 10


def _current_stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# The same without the Stream object, where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


class OpsError(RuntimeError):
    pass


class Ops:
    """A handle: one GPU's operators and their workspaces (one per stream)."""

    def __init__(self, device: int = 0):
        self._L = _lib.load()
        self.device = int(device)
        h = C.c_void_p()
        if self._L.phz_ops_create(self.device, C.byref(h)) != 0:
            raise OpsError(self._L.phz_ops_last_error(None).decode())
        self._h = h
        self._buf = bytearray(_SLOTS * _TENSOR.size)
        self._keep = (C.c_char * len(self._buf)).from_buffer(self._buf)
        base = C.addressof(self._keep)
        self._at = [base + i * _TENSOR.size for i in range(_SLOTS)]

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            self._L.phz_ops_destroy(h)
            self._h = None

    # ── arguments ──
    def _put(self, slot: int, t, name: str):
        """Describes one tensor to the library; the address of its view. (The
        common ranks are written out: this is most of a small call's time.)"""
        if t is None:
            return None
        try:
            code, n = _DTYPES[t.dtype], t.dim()
            if t.get_device() == self.device:  # -1 is the host's
                if n == 2:
                    a, b = t.shape
                    s, u = t.stride()
                    _PACK(self._buf, slot << 6, t.data_ptr(), a, b, 0, s, u, 0, code, 2)
                    return self._at[slot]
                if n == 3:
                    a, b, c = t.shape
                    s, u, v = t.stride()
                    _PACK(self._buf, slot << 6, t.data_ptr(), a, b, c, s, u, v, code, 3)
                    return self._at[slot]
                if n == 1:
                    _PACK(self._buf, slot << 6, t.data_ptr(), t.shape[0], 0, 0, t.stride(0), 0, 0, code, 1)
                    return self._at[slot]
        except (AttributeError, KeyError):
            pass
        if not isinstance(t, torch.Tensor):
            raise OpsError(f"{name} has to be a torch tensor, not {type(t).__name__}")
        if t.get_device() != self.device:
            where = "a host-only handle checks CPU tensors" if self.device < 0 else f"the handle's GPU is cuda:{self.device}"
            raise OpsError(f"{name} is on {t.device}: {where}")
        if t.dtype not in _DTYPES:
            raise OpsError(f"{name} is {t.dtype}, expected float32, bfloat16 or a mask of uint8 or bool")
        raise OpsError(f"{name} has {t.dim()} dimensions, expected 1 to 3")

    def _stream(self):
        return _raw_stream(self.device) if self.device >= 0 else None

    def _check(self, rc: int):
        if rc != 0:
            raise OpsError(self._L.phz_ops_last_error(self._h).decode())

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
        az, ax = self._put(0, z, "z"), self._put(1, x, "x")
        if out is not None:
            h, last = out
        else:
            h = torch.empty_like(x)
            last = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        self._check(self._L.phz_gated_scan(self._h, self._stream(), f, az, ax, self._put(2, h0, "h0"),
                                           self._put(3, reset, "reset"), self._put(4, h, "h"),
                                           self._put(5, last, "h_last")))
        return h, last

    def gated_scan_backward(self, dh, z, x, h, h0=None, reset=None, dh_last=None, form: str = "sigmoid", out=None):
        """The gradients (dz, dx, dh0) of gated_scan, from those of h and of the
        last state (None: zero) and the stored h. dh0 is float32."""
        f = self._choice(FORMS, form, "gate form")
        az, ax = self._put(0, z, "z"), self._put(1, x, "x")
        if out is not None:
            dz, dx, dh0 = out
        else:
            dz, dx = torch.empty_like(z), torch.empty_like(x)
            dh0 = torch.empty(x.shape[1:], dtype=torch.float32, device=x.device)
        self._check(self._L.phz_gated_scan_backward(
            self._h, self._stream(), f, self._put(2, dh, "dh"), self._put(3, dh_last, "dh_last"), az, ax,
            self._put(4, h, "h"), self._put(5, h0, "h0"), self._put(6, reset, "reset"), self._put(7, dz, "dz"),
            self._put(8, dx, "dx"), self._put(9, dh0, "dh0")))
        return dz, dx, dh0

    def gated_step(self, z, x, h, reset=None, form: str = "sigmoid"):
        """One step for z, x [worlds, width]: h [worlds, width] float32 is
        replaced, and returned."""
        f = self._choice(FORMS, form, "gate form")
        self._check(self._L.phz_gated_step(self._h, self._stream(), f, self._put(0, z, "z"), self._put(1, x, "x"),
                                           self._put(2, reset, "reset"), self._put(3, h, "h")))
        return h

    # ── the linear layer ──
    @staticmethod
    def _rows(t):
        return t.reshape(-1, t.shape[-1]) if isinstance(t, torch.Tensor) and t.dim() > 2 else t

    def linear(self, x, w, bias=None, act: str = "none", residual=None, save_pre: bool = False, out=None):
        """y = act(x w^T + bias) + residual for x [..., n_in], w [n_out, n_in];
        with save_pre, (y, x w^T + bias). All of one type, float32 or bfloat16.
        `out` (2-D) may be the residual."""
        a = self._choice(ACTS, act, "activation")
        x2, r2 = self._rows(x), self._rows(residual)
        ax, aw = self._put(0, x2, "x"), self._put(1, w, "w")
        if w.dim() != 2:
            raise OpsError(f"w has {w.dim()} dimensions, expected 2")
        y = out if out is not None else torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device)
        pre = torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device) if save_pre else None
        self._check(self._L.phz_linear(self._h, self._stream(), a, ax, aw, self._put(2, bias, "bias"),
                                       self._put(3, r2, "residual"), self._put(4, pre, "pre"), self._put(5, y, "y")))
        shape = (*x.shape[:-1], w.shape[0])
        if out is None and x.dim() != 2:
            y = y.view(shape)
        return (y, pre.view(shape)) if save_pre else y

    def linear_backward(self, dy, x, w, pre=None, act: str = "none", need_dx: bool = True, need_dw: bool = True,
                        need_db: bool = True):
        """The gradients (dx, dw, db) of linear for dz = dy act'(pre); those not
        needed are None. The residual's gradient is dy itself."""
        a = self._choice(ACTS, act, "activation")
        x2, dy2, p2 = self._rows(x), self._rows(dy), self._rows(pre)
        ax, aw = self._put(0, x2, "x"), self._put(1, w, "w")
        dx = torch.empty(x2.shape, dtype=x.dtype, device=x.device) if need_dx else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if need_dw else None
        db = torch.empty(w.shape[:1], dtype=w.dtype, device=w.device) if need_db else None
        self._check(self._L.phz_linear_backward(
            self._h, self._stream(), a, self._put(2, dy2, "dy"), ax, aw, self._put(3, p2, "pre"),
            self._put(4, dx, "dx"), self._put(5, dw, "dw"), self._put(6, db, "db")))
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
        ag = self._put(0, g, "g")
        o = out if out is not None else torch.empty_like(g)
        self._check(self._L.phz_orthogonalize(self._h, self._stream(), C.byref(cfg), ag, self._put(1, o, "o")))
        return o

    def muon_step(self, w, g, m, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                  weight_decay: float = 0.0, steps: int = 5, coef=NEWTON_SCHULZ, eps: float = 1e-7):
        """Muon's update of w (and the momentum m, both float32, in place) for
        the gradient g: matrices [rows, cols], or a batch of them."""
        cfg = self._muon(steps, coef, eps, lr, momentum, nesterov, weight_decay)
        self._check(self._L.phz_muon_step(self._h, self._stream(), C.byref(cfg), self._put(0, w, "w"),
                                          self._put(1, g, "g"), self._put(2, m, "m")))
