"""Operators of sequence policies on the device, over the C ABI of
phyz_amd/csrc/phz_scan.hip, phz_linear.hip, phz_muon.hip, phz_attend.hip,
phz_rotary.hip and phz_adamw.hip.

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

The recurrence's state may be a matrix for each head instead of a vector, read
by queries and written by keys and values (linear attention with a decay), with
positions as rotations of queries and keys; and parameters of any shapes take
one AdamW step together:

    qk = ops.rotary(qkv[..., :2 * n], positions, freq, heads=2 * heads)
    o, s = ops.linear_attention(qk[..., :n], qk[..., n:], qkv[..., 2 * n:], g, reset=reset)
    o = ops.linear_attention_step(q, k, v, g, s)              # acting: s advances
    ops.adamw_step(params, grads, m, v, step)

Arguments are torch tensors on the handle's GPU; calls enqueue their work on
torch's current stream and return without waiting. Errors raise OpsError with
the library's message. There is no host fallback: the kernels run on a HIP
device or not at all. Ops(device=-1) checks arguments only (of CPU tensors)
and then raises.

Autograd records none of this: gradients come from the _backward calls. The
forward operators refuse tensors that require gradients while it is recording
(call them under torch.no_grad(), or on detached tensors), and tensors that carry
tangents of forward-mode differentiation; the _backward calls
and muon_step take them as they are. What a call writes in place or into `out`
counts as changed for graphs that saved it.
"""
from __future__ import annotations

import ctypes as C
import math
import os

import torch
from torch.autograd import forward_ad

from . import _lib

FORMS = {"sigmoid": 0, "decay": 1}
ACTS = {"none": 0, "tanh": 1, "relu": 2, "silu": 3, "gelu": 4}
# Muon's quintic: five steps take singular values in about (0.002, 1) to within
# 0.7 to 1.2.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)

PAIRS = {"half": 0, "interleaved": 1}

_DTYPES = (torch.float32, torch.float64, torch.bfloat16, torch.uint8, torch.bool, torch.int32, torch.int64)
# The entry points, in the order of phz_describe.cpp's table.
_ENTRIES = ("phz_gated_scan", "phz_gated_scan_backward", "phz_gated_step", "phz_linear", "phz_linear_backward",
            "phz_orthogonalize", "phz_muon_step", "phz_linear_attention", "phz_linear_attention_backward",
            "phz_linear_attention_step", "phz_rotary", "phz_adamw_step", "phz_adamw_values")
(_SCAN, _SCAN_BACKWARD, _STEP, _LINEAR, _LINEAR_BACKWARD, _ORTHOGONALIZE, _MUON, _ATTENTION, _ATTENTION_BACKWARD,
 _ATTENTION_STEP, _ROTARY, _ADAMW, _ADAMW_VALUES) = range(13)
# Whose results a user may expect autograd to know.
_FORWARD = {_SCAN, _STEP, _LINEAR, _ORTHOGONALIZE, _ATTENTION, _ATTENTION_STEP, _ROTARY}
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


def rotary_frequencies(size: int, base: float = 10000.0, stretch: float = 1.0, turns=None, context: int = 0) -> torch.Tensor:
    """Radians a position for the size / 2 pairs of Ops.rotary, float64 on the CPU:
    base^(-2 i / size). For contexts `stretch` times as long as those trained on,
    all are divided by it, or, given turns=(few, many) and the trained context,
    only pairs that turn at most `few` times in it; pairs that turn `many` times or
    more are kept, those between blended."""
    if size < 0 or size % 2:
        raise OpsError(f"the rotated part of a head has to be even, not {size}")
    if not (base > 0 and stretch > 0 and math.isfinite(base) and math.isfinite(stretch)):
        raise OpsError("base and stretch have to be positive and finite")
    f = base ** (-torch.arange(size // 2, dtype=torch.float64) * 2 / max(size, 1))
    if turns is None:
        return f / stretch
    few, many = turns
    if not (0 <= few < many and math.isfinite(many) and context > 0):
        raise OpsError("turns have to be (few, many), few below many, with the trained context")
    keep = ((f * context / (2 * math.pi) - few) / (many - few)).clamp(0, 1)
    return f * (keep + (1 - keep) / stretch)


class Ops:
    """A handle: one GPU's operators and their workspaces, one per stream and one
    per captured graph. A handle whose workspace a captured graph holds is kept to
    the end of the process, so that the graph outlives the last reference to it."""

    def __init__(self, device: int = 0):
        self._L = _lib.load()
        self._call, self._call_lists = _bound().call, _bound().call_lists
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
        if getattr(forward_ad, "_current_level", 0) >= 0 and op in _FORWARD:
            for name, t in zip(names.split(), tensors):
                if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                    raise OpsError(f"{name} carries a tangent, which these operators do not record: call on detached tensors")
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

    def _run_lists(self, op: int, head: int, names: str, lists, single=None):
        """One entry point of lists of tensors on the current stream."""
        names = names.split()
        for name, x in zip(names, lists):
            if not isinstance(x, (list, tuple)) and (x is not None or name == names[0]):
                raise OpsError(f"{name} has to be a list of tensors, not {type(x).__name__}")
        lists = [None if x is None else tuple(x) for x in lists]
        n = len(lists[0])
        for name, x in zip(names, lists):
            if x is not None and len(x) != n:
                raise OpsError(f"{name} has {len(x)} tensors, {names[0]} has {n}")
        rc = self._call_lists(op, self._h, _raw_stream(self.device) if self.device >= 0 else 0, self.device, head,
                              tuple(lists), single)
        if rc > 0:
            raise OpsError(self._L.phz_ops_last_error(self._h).decode())
        if rc <= -(1 << 40):
            i = -(1 << 40) - rc
            raise OpsError(f"{names[1]}[{i}] has the shape {tuple(lists[1][i].shape)}, {names[0]}[{i}] {tuple(lists[0][i].shape)}")
        if rc < 0:
            i, l = divmod(-1 - rc, 5)
            name, t = (names[5], single) if i == n else (f"{names[l]}[{i}]", lists[l][i])
            if isinstance(t, torch.Tensor) and t.get_device() == self.device and t.dtype in _DTYPES and not t.is_contiguous():
                raise OpsError(f"{name} is not contiguous")
            self._complain(name, t)

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
    def _whole(x, name: str) -> int:
        try:
            n = int(x)
            if n == x and -1 << 31 <= n < 1 << 31:
                return n
        except (TypeError, ValueError, OverflowError):
            pass
        raise OpsError(f"{name} has to be a whole number, not {x!r}")

    @staticmethod
    def _number(x, name: str) -> float:
        try:
            return float(x)
        except (TypeError, ValueError, OverflowError):
            raise OpsError(f"{name} has to be a number, not {x!r}") from None

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

    # ── linear attention with a decay for each head ──
    @staticmethod
    def _heads(q, v, g, size_k, size_v, scale):
        """(heads, the head sizes and scale as the library takes them)."""
        for t, name in ((v, "v"), (g, "g")):
            if t.dim() < 1:
                raise OpsError(f"{name} has 0 dimensions, expected {q.dim()}")
        heads = g.shape[-1]
        if heads < 1:
            raise OpsError("g has no heads")
        size_k = q.shape[-1] // heads if size_k is None else Ops._whole(size_k, "size_k")
        size_v = v.shape[-1] // heads if size_v is None else Ops._whole(size_v, "size_v")
        if not (1 <= size_k <= 128 and 1 <= size_v <= 128):
            raise OpsError(f"size_k and size_v have to be 1 to 128, not {size_k} and {size_v}")
        return heads, _lib.AttentionCfg(size_k ** -0.5 if scale is None else Ops._number(scale, "scale"), size_k, size_v)

    @staticmethod
    def _matrices(s, name: str, cfg):
        """States [worlds, heads, size_k, size_v] with one axis for each's elements."""
        if s is None:
            return None
        if not isinstance(s, torch.Tensor) or s.dim() != 4:
            raise OpsError(f"{name} has to be a tensor [worlds, heads, size_k, size_v]")
        for axis, n in ((2, cfg.size_k), (3, cfg.size_v)):
            if s.shape[axis] != n:
                raise OpsError(f"{name} has {s.shape[axis]} elements along axis {axis}, expected {n}")
        try:
            return s.view(s.shape[0], s.shape[1], s.shape[2] * s.shape[3])
        except RuntimeError:
            raise OpsError(f"{name}: each head's state has to be dense") from None

    def _rates(self, g, like):
        """g of all steps and worlds, from one of the heads alone."""
        if self._tensor(g, "g").dim() == 1 and like.dim() > 1:
            return g.expand(*like.shape[:-1], g.shape[0])
        return g

    def linear_attention(self, q, k, v, g, s0=None, reset=None, size_k=None, size_v=None, scale=None, out=None):
        """S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t for q, k
        [steps, worlds, heads * size_k] and v [steps, worlds, heads * size_v] (views
        with a dense last axis) and g [steps, worlds, heads] float32, or [heads]: (o
        like v's heads, the last state [worlds, heads, size_k, size_v] float32).
        Given size_k and size_v, q, k and v may each have fewer heads than g: each
        then serves heads / its heads of g's in a row. s0 are the states before the
        first step (None: zeros); where reset [steps, worlds] is set, or g is below
        -104, an episode begins and S_{t-1} counts as 0. scale: size_k^-0.5 if None."""
        for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g")):
            self._tensor(t, name)
        if q.dim() != 3:
            raise OpsError(f"q has {q.dim()} dimensions, expected 3")
        g = self._rates(g, q)
        heads, cfg = self._heads(q, v, g, size_k, size_v, scale)
        if out is not None:
            o, last = out
        else:
            o = torch.empty((*q.shape[:-1], heads * cfg.size_v), dtype=q.dtype, device=q.device)
            last = torch.empty((q.shape[1], heads, cfg.size_k, cfg.size_v), dtype=torch.float32, device=q.device)
        self._run(_ATTENTION, C.addressof(cfg), "q k v g s0 reset o s_last", q, k, v, g, self._matrices(s0, "s0", cfg), reset, o,
                  self._matrices(last, "s_last", cfg))
        if out is not None:
            _written([t for t in out if t is not None])
        return o, last

    def linear_attention_backward(self, do, q, k, v, g, s0=None, reset=None, ds=None, size_k=None, size_v=None, scale=None,
                                  need_dg: bool = True, out=None):
        """The gradients (dq, dk, dv, dg, ds0) of linear_attention, from those of o
        and of the last state (None: zero). dq, dk and dv are like q, k and v, summed
        over the heads that share them; dg [steps, worlds, heads] is every step's and
        world's own also where g is one of the heads alone, None if not needed; dg and
        ds0 are float32."""
        for t, name in ((do, "do"), (q, "q"), (k, "k"), (v, "v"), (g, "g")):
            self._tensor(t, name)
        if q.dim() != 3:
            raise OpsError(f"q has {q.dim()} dimensions, expected 3")
        g = self._rates(g, q)
        heads, cfg = self._heads(q, v, g, size_k, size_v, scale)
        if out is not None:
            dq, dk, dv, dg, ds0 = out
        else:
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            dg = torch.empty((*q.shape[:-1], heads), dtype=torch.float32, device=q.device) if need_dg else None
            ds0 = torch.empty((q.shape[1], heads, cfg.size_k, cfg.size_v), dtype=torch.float32, device=q.device)
        self._run(_ATTENTION_BACKWARD, C.addressof(cfg), "do ds q k v g s0 reset dq dk dv dg ds0", do, self._matrices(ds, "ds", cfg),
                  q, k, v, g, self._matrices(s0, "s0", cfg), reset, dq, dk, dv, dg, self._matrices(ds0, "ds0", cfg))
        if out is not None:
            _written([t for t in out if t is not None])
        return dq, dk, dv, dg, ds0

    def linear_attention_step(self, q, k, v, g, s, reset=None, size_k=None, size_v=None, scale=None, out=None):
        """One step for q, k, v and g without the axis of steps: o [worlds, heads *
        size_v]; the states s [worlds, heads, size_k, size_v] float32 are replaced."""
        for t, name in ((q, "q"), (k, "k"), (v, "v"), (g, "g")):
            self._tensor(t, name)
        if q.dim() != 2:
            raise OpsError(f"q has {q.dim()} dimensions, expected 2")
        g = self._rates(g, q)
        heads, cfg = self._heads(q, v, g, size_k, size_v, scale)
        o = out if out is not None else torch.empty((q.shape[0], heads * cfg.size_v), dtype=q.dtype, device=q.device)
        self._run(_ATTENTION_STEP, C.addressof(cfg), "q k v g reset s o", q, k, v, g, reset,
                  self._matrices(self._tensor(s, "s"), "s", cfg), o)
        _written((s,) if out is None else (s, o))
        return o

    # ── rotary positions ──
    def rotary(self, x, positions, freq, heads: int = 1, layout: str = "half", scale: float = 1.0, inverse: bool = False,
               out=None):
        """x [..., heads * size] with the first 2 len(freq) elements of each head
        turned by positions * freq, in pairs (i, i + len(freq)) ("half") or (2 i, 2 i
        + 1) ("interleaved"), and multiplied by scale; the others are copied. positions
        (int32 or int64) have x's axes but the last, of which there are one or two;
        freq is float64 (rotary_frequencies). inverse turns back: the gradient for x is
        rotary(dy, ..., inverse=True). `out` may be x."""
        p = self._choice(PAIRS, layout, "layout")
        cfg = _lib.RotaryCfg(self._number(scale, "scale"), self._whole(heads, "heads"), p, int(bool(inverse)))
        y = out if out is not None else torch.empty_like(self._tensor(x, "x"))
        x3, p2, y3 = x, positions, y
        if isinstance(x, torch.Tensor) and x.dim() == 2:
            x3, p2, y3 = (t[None] if isinstance(t, torch.Tensor) else t for t in (x, positions, y))
        self._run(_ROTARY, C.addressof(cfg), "x positions freq y", x3, p2, freq, y3)
        if out is not None:
            _written((y,))
        return y

    # ── AdamW ──
    @staticmethod
    def adamw_state(params, bits: int = 32):
        """(m, v, exponents, step) of adamw_step for tensors like params, before the
        first step: moments in 32 bits (exponents None), or in 8 with an exponent for
        each 256 elements."""
        params = [Ops._tensor(p, "params") for p in params]
        if bits not in (32, 8):
            raise OpsError(f"moments have 32 or 8 bits, not {bits}")
        dt = torch.float32 if bits == 32 else torch.uint8
        m, v = ([torch.zeros(p.shape, dtype=dt, device=p.device) for p in params] for _ in range(2))
        e = None if bits == 32 else [torch.zeros(2, -(-p.numel() // 256), dtype=torch.uint8, device=p.device) for p in params]
        where = params[0].device if params else torch.device("cpu")
        return m, v, e, torch.zeros(1, dtype=torch.int64, device=where)

    def adamw_step(self, w, g, m, v, step, exponents=None, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                   weight_decay: float = 0.01, seed: int = 0):
        """One AdamW step of the tensors w (float32 or bfloat16, in place) for the
        gradients g (either; of w's shapes, or vectors), with the moments m and v (in place; float32, or uint8
        with their exponents): lists of one length, of contiguous tensors of any
        shapes, best made by adamw_state. step, an int64 tensor of one element, counts
        the steps, also in replays of a captured graph. Moments of 8 bits are rounded
        by random bits that follow from seed and step."""
        try:
            b1, b2 = betas
        except (TypeError, ValueError):
            raise OpsError(f"betas have to be two numbers, not {betas!r}") from None
        try:
            seed = int(seed) & 0xffffffff
        except (TypeError, ValueError, OverflowError):
            raise OpsError(f"seed has to be a whole number, not {seed!r}") from None
        cfg = _lib.AdamWCfg(*(self._number(x, n) for x, n in ((lr, "lr"), (b1, "betas"), (b2, "betas"), (eps, "eps"),
                                                              (weight_decay, "weight_decay"))), seed)
        self._run_lists(_ADAMW, C.addressof(cfg), "w g m v exponents step", (w, g, m, v, exponents), self._tensor(step, "step"))
        _written([*w, *m, *v, *(exponents or ()), step])

    def adamw_values(self, m, v, exponents, out=None):
        """The values of 8-bit moments, lists of bfloat16 tensors, which hold them
        exactly: (m's, v's)."""
        if out is None:
            for name, x in (("m", m), ("v", v)):
                if not isinstance(x, (list, tuple)):
                    raise OpsError(f"{name} has to be a list of tensors, not {type(x).__name__}")
            out = tuple([torch.empty(self._tensor(t, "m").shape, dtype=torch.bfloat16, device=t.device) for t in x]
                        for x in (m, v))
            self._run_lists(_ADAMW_VALUES, 0, "m v exponents m_values v_values", (m, v, exponents, *out))
        else:
            self._run_lists(_ADAMW_VALUES, 0, "m v exponents m_values v_values", (m, v, exponents, *out))
            _written([t for x in out for t in x])
        return out
