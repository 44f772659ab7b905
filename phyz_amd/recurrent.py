"""A policy with memory, built from the operators of phyz_amd.ops, and its
training by imitation of a rollout.

    embedding   x = tanh(obs W_e^T + b_e)
    gates       (z, u) = x W_g^T + b_g
    memory      h_t = sigmoid(z_t) h_{t-1} + (1 - sigmoid(z_t)) u_t, from 0 where an episode begins
    block       y = x + h W_o^T + b_o
    action      a = y W_a^T + b_a

Over a rollout the memory is one scan; acting, it is one step of it with the
state kept on the device. Matrices take Muon's update, biases momentum descent.

    policy = RecurrentPolicy(n_in=29, width=256, n_out=8)
    loss = policy.imitate(obs, actions, reset=reset)     # [steps, worlds, ...]
    policy.begin(worlds)
    a = policy.act(obs_now, reset_now)                   # [worlds, n_out]

`python -m phyz_amd.recurrent` collects a rollout of the control-loop workload's
policy on the device and fits a recurrent student to it from fewer
observations: positions without velocities, which memory has to make up for.
"""
from __future__ import annotations

import math
from typing import Dict, Optional

import torch

from .ops import Ops


class RecurrentPolicy:
    def __init__(self, n_in: int, width: int, n_out: int, device: int = 0, dtype=torch.float32, seed: int = 0):
        self.ops = Ops(device)
        self.n_in, self.width, self.n_out, self.dtype = n_in, width, n_out, dtype
        self.device = torch.device("cuda", device)
        gen = torch.Generator().manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=gen) / math.sqrt(cols)).to(self.device)

        # f32 masters; products take them in `dtype`.
        self.w = {"embed": matrix(width, n_in), "gate": matrix(2 * width, width), "out": 0.1 * matrix(width, width),
                  "act": matrix(n_out, width)}
        self.b = {k: torch.zeros(v.shape[0], device=self.device) for k, v in self.w.items()}
        # Memories of about 1 to 50 steps to begin with.
        self.b["gate"][:width] = torch.linspace(0.0, 4.0, width, device=self.device)
        self._momentum = {k: torch.zeros_like(v) for k, v in {**self.w, **{"b_" + k: v for k, v in self.b.items()}}.items()}
        self._state: Optional[torch.Tensor] = None

    def _params(self, name: str):
        return self.w[name].to(self.dtype), self.b[name].to(self.dtype)

    # ── over a rollout ──
    def forward(self, obs, reset=None, h0=None):
        """Actions [steps, worlds, n_out] for obs [steps, worlds, n_in], and what
        backward needs."""
        ops, n = self.ops, self.width
        obs = obs.to(self.dtype)
        w, b = self._params("embed")
        x, pre = ops.linear(obs, w, bias=b, act="tanh", save_pre=True)
        w, b = self._params("gate")
        zu = ops.linear(x, w, bias=b)
        h, last = ops.gated_scan(zu[..., :n], zu[..., n:], h0=h0, reset=reset)
        w, b = self._params("out")
        y = ops.linear(h, w, bias=b, residual=x)
        w, b = self._params("act")
        return ops.linear(y, w, bias=b), {"obs": obs, "pre": pre, "x": x, "zu": zu, "h": h, "y": y, "h0": h0, "reset": reset,
                                          "last": last}

    def backward(self, d_act, c) -> Dict[str, torch.Tensor]:
        """The loss's gradients for every parameter, from those for the actions."""
        ops, n, g = self.ops, self.width, {}
        dy, g["act"], g["b_act"] = ops.linear_backward(d_act.to(self.dtype), c["y"], self._params("act")[0])
        dh, g["out"], g["b_out"] = ops.linear_backward(dy, c["h"], self._params("out")[0])
        d_zu = torch.empty_like(c["zu"])
        dh0 = torch.empty(c["h"].shape[1:], dtype=torch.float32, device=self.device)
        ops.gated_scan_backward(dh, c["zu"][..., :n], c["zu"][..., n:], c["h"], h0=c["h0"], reset=c["reset"],
                                out=(d_zu[..., :n], d_zu[..., n:], dh0))
        dx, g["gate"], g["b_gate"] = ops.linear_backward(d_zu, c["x"], self._params("gate")[0])
        dx += dy  # the residual's way
        _, g["embed"], g["b_embed"] = ops.linear_backward(dx, c["obs"], self._params("embed")[0], pre=c["pre"], act="tanh",
                                                          need_dx=False)
        return g

    def update(self, grads, lr: float = 0.02, bias_lr: float = 0.02, momentum: float = 0.95):
        for k, w in self.w.items():
            self.ops.muon_step(w, grads[k], self._momentum[k], lr=lr, momentum=momentum)
        for k, b in self.b.items():
            m = self._momentum["b_" + k]
            m.mul_(momentum).add_(grads["b_" + k].float())
            b.sub_(m, alpha=bias_lr)

    def imitate(self, obs, actions, reset=None, lr: float = 0.02, bias_lr: float = 0.02) -> torch.Tensor:
        """One update towards `actions`; the mean squared error before it (a
        device tensor: nothing waits)."""
        a, c = self.forward(obs, reset)
        err = a.float() - actions
        self.update(self.backward(err * (2.0 / err.numel()), c), lr, bias_lr)
        return err.square().mean()

    # ── acting ──
    def begin(self, worlds: int):
        self._state = torch.zeros(worlds, self.width, device=self.device)

    def act(self, obs, reset=None):
        """One control step: actions [worlds, n_out]; the memory advances."""
        ops, n = self.ops, self.width
        w, b = self._params("embed")
        x = ops.linear(obs.to(self.dtype), w, bias=b, act="tanh")
        w, b = self._params("gate")
        zu = ops.linear(x, w, bias=b)
        ops.gated_step(zu[:, :n], zu[:, n:], self._state, reset=reset)
        w, b = self._params("out")
        y = ops.linear(self._state.to(self.dtype), w, bias=b, residual=x)
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


def main(worlds: int = 512, updates: int = 150):
    obs, actions = collect(worlds)
    # Without the 14 velocities (columns 13 to 26).
    seen = torch.cat([obs[..., :13], obs[..., 27:]], -1).contiguous()
    mean, std = seen.mean((0, 1)), seen.std((0, 1)) + 1e-6
    seen = (seen - mean) / std
    reset = torch.zeros(seen.shape[:2], dtype=torch.bool, device=seen.device)
    reset[0] = True
    policy = RecurrentPolicy(seen.shape[-1], 128, actions.shape[-1])
    print(f"{worlds} worlds x {seen.shape[0]} control steps; actions' variance {float(actions.var()):.5f}")
    for k in range(updates):
        loss = policy.imitate(seen, actions, reset=reset, lr=0.02 * (1 - k / updates))
        if k % 25 == 0 or k + 1 == updates:
            print(f"update {k:4d}  mean squared error {float(loss):.5f}", flush=True)
    policy.begin(worlds)
    whole, _ = policy.forward(seen, reset)
    worst = 0.0
    for t in range(seen.shape[0]):
        worst = max(worst, float((policy.act(seen[t], reset[t]) - whole[t]).abs().max()))
    print(f"acting step by step against the scan: {worst:.2e}")


if __name__ == "__main__":
    main()
