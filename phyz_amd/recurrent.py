"""A policy with memory, built from the operators of phyz_amd.ops, and its
training by imitation of a rollout.

    embedding   x = tanh(obs W_e^T + b_e)
    gates       (z, u) = x W_g^T + b_g
    memory      h_t = sigmoid(z_t) h_{t-1} + (1 - sigmoid(z_t)) u_t, from 0 where an episode begins
    block       y = x + h W_o^T + b_o
    action      a = y W_a^T + b_a

or, with memory="attention", a matrix for each head instead of the vector:

    (q, k, v, z) = x W_g^T + b_g, q and k turned by the step of the episode
    S_t = sigmoid(z_t) S_{t-1} + k_t v_t^T,   h_t = S_t^T q_t / sqrt(size of a head)

Over a rollout the memory is one scan (or one linear attention); acting, it is one
step of it with the state kept on the device. Matrices take Muon's update and
biases momentum descent, or, with optimizer="adamw", all parameters one AdamW step
together, whose moments may be held in 8 bits.

    policy = RecurrentPolicy(n_in=29, width=256, n_out=8)
    loss = policy.imitate(obs, actions, reset=reset)     # [steps, worlds, ...]
    policy.begin(worlds)
    a = policy.act(obs_now, reset_now)                   # [worlds, n_out]

`python -m phyz_amd.recurrent` (--memory, --optimizer) collects a rollout of the control-loop workload's
policy on the device and fits a recurrent student to it from fewer
observations: positions without velocities, which memory has to make up for.
"""
from __future__ import annotations

import math
from typing import Dict, Optional

import torch

from .ops import Ops, OpsError, rotary_frequencies


class RecurrentPolicy:
    def __init__(self, n_in: int, width: int, n_out: int, device: int = 0, dtype=torch.float32, seed: int = 0,
                 memory: str = "gates", heads: int = 4, optimizer: str = "muon", moment_bits: int = 32):
        if memory not in ("gates", "attention") or optimizer not in ("muon", "adamw"):
            raise OpsError(f"unknown memory {memory!r} or optimizer {optimizer!r}")
        if memory == "attention" and (heads < 1 or width % (2 * heads)):
            raise OpsError(f"heads of an even size have to divide the width {width}, not {heads}")
        if memory == "attention" and width // heads > 128:
            raise OpsError(f"heads have a size of at most 128, not {width // heads}")
        if moment_bits not in (32, 8):
            raise OpsError(f"moments have 32 or 8 bits, not {moment_bits}")
        self.ops = Ops(device)
        self.n_in, self.width, self.n_out, self.dtype = n_in, width, n_out, dtype
        self.memory, self.heads, self.optimizer, self.seed = memory, heads, optimizer, seed
        self.device = torch.device("cuda", device)
        gen = torch.Generator().manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=gen) / math.sqrt(cols)).to(self.device)

        # f32 masters; products take them in `dtype`.
        gates = 2 * width if memory == "gates" else 3 * width + heads
        self.w = {"embed": matrix(width, n_in), "gate": matrix(gates, width), "out": 0.1 * matrix(width, width),
                  "act": matrix(n_out, width)}
        self.b = {k: torch.zeros(v.shape[0], device=self.device) for k, v in self.w.items()}
        # Memories of about 1 to 50 steps to begin with.
        if memory == "gates":
            self.b["gate"][:width] = torch.linspace(0.0, 4.0, width, device=self.device)
        else:
            self.b["gate"][3 * width:] = torch.linspace(0.0, 4.0, heads, device=self.device)
            self._freq = rotary_frequencies(width // heads).to(self.device)
        if optimizer == "muon":
            self._momentum = {k: torch.zeros_like(v) for k, v in {**self.w, **{"b_" + k: v for k, v in self.b.items()}}.items()}
        else:
            self._moments = self.ops.adamw_state([*self.w.values(), *self.b.values()], bits=moment_bits)
        self._state = None

    def _params(self, name: str):
        return self.w[name].to(self.dtype), self.b[name].to(self.dtype)

    # ── the memory ──
    def _positions(self, steps: int, worlds: int, reset, first):
        """Each step's place in its episode, and each world's next one."""
        t = torch.arange(steps, device=self.device)[:, None]
        start = torch.zeros(worlds, dtype=torch.int64, device=self.device) if first is None else first
        p = start + t
        if reset is not None and steps:
            at = torch.where(reset.bool(), t, -1).cummax(0).values
            p = torch.where(at >= 0, t - at, p)
        return p, (p[-1] + 1 if steps else start)

    def _remember(self, zu, h0, reset):
        """(h, what backward needs, the last state) of the gates' layer over a rollout."""
        ops, n = self.ops, self.width
        if self.memory == "gates":
            h, last = ops.gated_scan(zu[..., :n], zu[..., n:], h0=h0, reset=reset)
            return h, {"zu": zu, "h0": h0}, last
        s0, first = h0 if h0 is not None else (None, None)
        p, following = self._positions(*zu.shape[:2], reset, first)
        ops.rotary(zu[..., :2 * n], p, self._freq, heads=2 * self.heads, out=zu[..., :2 * n])
        z = zu[..., 3 * n:].float()
        g = torch.nn.functional.logsigmoid(z)
        h, last = ops.linear_attention(zu[..., :n], zu[..., n:2 * n], zu[..., 2 * n:3 * n], g, s0=s0, reset=reset)
        return h, {"zu": zu, "h0": s0, "p": p, "z": z, "g": g}, (last, following)

    def _remember_backward(self, dh, c):
        ops, n, zu = self.ops, self.width, c["zu"]
        d = torch.empty_like(zu)
        if self.memory == "gates":
            dh0 = torch.empty(zu.shape[1], n, dtype=torch.float32, device=self.device)
            ops.gated_scan_backward(dh, zu[..., :n], zu[..., n:], c["h"], h0=c["h0"], reset=c["reset"],
                                    out=(d[..., :n], d[..., n:], dh0))
            return d
        dg = torch.empty_like(c["g"])
        ops.linear_attention_backward(dh, zu[..., :n], zu[..., n:2 * n], zu[..., 2 * n:3 * n], c["g"], s0=c["h0"], reset=c["reset"],
                                      out=(d[..., :n], d[..., n:2 * n], d[..., 2 * n:3 * n], dg, None))
        ops.rotary(d[..., :2 * n], c["p"], self._freq, heads=2 * self.heads, inverse=True, out=d[..., :2 * n])
        d[..., 3 * n:] = dg * torch.sigmoid(-c["z"])
        return d

    # ── over a rollout ──
    def forward(self, obs, reset=None, h0=None):
        """Actions [steps, worlds, n_out] for obs [steps, worlds, n_in], and what
        backward needs; under "last" the memory behind the last step, as h0 takes it."""
        ops = self.ops
        obs = obs.to(self.dtype)
        w, b = self._params("embed")
        x, pre = ops.linear(obs, w, bias=b, act="tanh", save_pre=True)
        w, b = self._params("gate")
        h, kept, last = self._remember(ops.linear(x, w, bias=b), h0, reset)
        w, b = self._params("out")
        y = ops.linear(h, w, bias=b, residual=x)
        w, b = self._params("act")
        return ops.linear(y, w, bias=b), {"obs": obs, "pre": pre, "x": x, "h": h, "y": y, "reset": reset, "last": last, **kept}

    def backward(self, d_act, c) -> Dict[str, torch.Tensor]:
        """The loss's gradients for every parameter, from those for the actions."""
        ops, g = self.ops, {}
        dy, g["act"], g["b_act"] = ops.linear_backward(d_act.to(self.dtype), c["y"], self._params("act")[0])
        dh, g["out"], g["b_out"] = ops.linear_backward(dy, c["h"], self._params("out")[0])
        d_zu = self._remember_backward(dh, c)
        dx, g["gate"], g["b_gate"] = ops.linear_backward(d_zu, c["x"], self._params("gate")[0])
        dx += dy  # the residual's way
        _, g["embed"], g["b_embed"] = ops.linear_backward(dx, c["obs"], self._params("embed")[0], pre=c["pre"], act="tanh",
                                                          need_dx=False)
        return g

    def update(self, grads, lr: Optional[float] = None, bias_lr: float = 0.02, momentum: float = 0.95):
        """One step of the optimizer; lr is 0.02 for Muon and 1e-3 for AdamW if None,
        bias_lr and momentum are Muon's."""
        if self.optimizer == "adamw":
            m, v, exponents, step = self._moments
            self.ops.adamw_step([*self.w.values(), *self.b.values()], [grads[k] for k in self.w] + [grads["b_" + k] for k in self.b],
                                m, v, step, exponents=exponents, lr=1e-3 if lr is None else lr, seed=self.seed)
            return
        lr = 0.02 if lr is None else lr
        for k, w in self.w.items():
            self.ops.muon_step(w, grads[k], self._momentum[k], lr=lr, momentum=momentum)
        for k, b in self.b.items():
            m = self._momentum["b_" + k]
            m.mul_(momentum).add_(grads["b_" + k].float())
            b.sub_(m, alpha=bias_lr)

    def imitate(self, obs, actions, reset=None, lr: Optional[float] = None, bias_lr: float = 0.02) -> torch.Tensor:
        """One update towards `actions`; the mean squared error before it (a
        device tensor: nothing waits)."""
        a, c = self.forward(obs, reset)
        err = a.float() - actions
        self.update(self.backward(err * (2.0 / err.numel()), c), lr, bias_lr)
        return err.square().mean()

    # ── acting ──
    def begin(self, worlds: int):
        if self.memory == "gates":
            self._state = torch.zeros(worlds, self.width, device=self.device)
        else:
            n = self.width // self.heads
            self._state = (torch.zeros(worlds, self.heads, n, n, device=self.device),
                           torch.zeros(worlds, dtype=torch.int64, device=self.device))

    def _recall(self, zu, reset):
        """One step of the memory: h [worlds, width]; the state advances."""
        ops, n = self.ops, self.width
        if self.memory == "gates":
            ops.gated_step(zu[:, :n], zu[:, n:], self._state, reset=reset)
            return self._state.to(self.dtype)
        s, p = self._state
        if reset is not None:
            p.masked_fill_(reset.bool(), 0)
        ops.rotary(zu[:, :2 * n], p, self._freq, heads=2 * self.heads, out=zu[:, :2 * n])
        p += 1
        g = torch.nn.functional.logsigmoid(zu[:, 3 * n:].float())
        return ops.linear_attention_step(zu[:, :n], zu[:, n:2 * n], zu[:, 2 * n:3 * n], g, s, reset=reset)

    def act(self, obs, reset=None):
        """One control step: actions [worlds, n_out]; the memory advances."""
        ops = self.ops
        w, b = self._params("embed")
        x = ops.linear(obs.to(self.dtype), w, bias=b, act="tanh")
        w, b = self._params("gate")
        h = self._recall(ops.linear(x, w, bias=b), reset)
        w, b = self._params("out")
        y = ops.linear(h, w, bias=b, residual=x)
        w, b = self._params("act")
        return ops.linear(y, w, bias=b)


def collect(worlds: int, device: int = 0):
    """(observations, the teacher's mean actions' samples) of one rollout of the
    control-loop workload, on the device: [steps, worlds, 29] and [steps, worlds, 8]."""
    from . import workloads as W
    from .sim import from_control_loop
    cl = W.control_loop(hidden=64)
    sim = from_control_loop(cl, "f32", nworld=worlds, device=device)
    q, v, _, _ = cl.base.initial_state(worlds)
    sim.load_states(q, v)
    sim.rollout(0, cl.n_control, cl.control_every, False)
    obs, out = sim.readback_policy_history(0, cl.n_control)
    dev = torch.device("cuda", device)
    return (torch.as_tensor(obs, dtype=torch.float32, device=dev).contiguous(),
            torch.as_tensor(out[..., :-1], dtype=torch.float32, device=dev).contiguous())


def main(worlds: int = 512, updates: int = 150, memory: str = "gates", optimizer: str = "muon", moment_bits: int = 32):
    obs, actions = collect(worlds)
    # Without the 14 velocities (columns 13 to 26).
    seen = torch.cat([obs[..., :13], obs[..., 27:]], -1).contiguous()
    mean, std = seen.mean((0, 1)), seen.std((0, 1)) + 1e-6
    seen = (seen - mean) / std
    reset = torch.zeros(seen.shape[:2], dtype=torch.bool, device=seen.device)
    reset[0] = True
    policy = RecurrentPolicy(seen.shape[-1], 128, actions.shape[-1], memory=memory, optimizer=optimizer, moment_bits=moment_bits)
    rate = 0.02 if optimizer == "muon" else 3e-3
    print(f"{worlds} worlds x {seen.shape[0]} control steps; actions' variance {float(actions.var()):.5f}")
    for k in range(updates):
        loss = policy.imitate(seen, actions, reset=reset, lr=rate * (1 - k / updates))
        if k % 25 == 0 or k + 1 == updates:
            print(f"update {k:4d}  mean squared error {float(loss):.5f}", flush=True)
    policy.begin(worlds)
    whole, _ = policy.forward(seen, reset)
    worst = 0.0
    for t in range(seen.shape[0]):
        worst = max(worst, float((policy.act(seen[t], reset[t]) - whole[t]).abs().max()))
    print(f"acting step by step against the scan: {worst:.2e}")


if __name__ == "__main__":
    import argparse
    args = argparse.ArgumentParser(prog="python -m phyz_amd.recurrent")
    args.add_argument("--worlds", type=int, default=512)
    args.add_argument("--updates", type=int, default=150)
    args.add_argument("--memory", choices=("gates", "attention"), default="gates")
    args.add_argument("--optimizer", choices=("muon", "adamw"), default="muon")
    args.add_argument("--moment-bits", type=int, choices=(32, 8), default=32)
    main(**vars(args.parse_args()))
