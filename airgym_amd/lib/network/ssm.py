"""Memory of a policy: a selective state space layer over the steps of an episode, in front of the MLP.

    x', z = split(W_in x);  c = silu(conv(x'));  dt, B, C = split(W_x c);  y = scan(c, W_dt dt, -exp(A_log), B, C, D, gate z)
    out = x + W_out y

Trained over the horizon's sequences (forward; episodes end inside, `resets`), run one step at a time in rollouts and by the player
(step).  On the GPU the convolution and the scan are the HIP kernels (causal_conv.py, selective_scan.py); CPU tensors take their torch
forms.  The reference has no counterpart: its recurrent-state plumbing ('states', lib/agent/a2c_continuous.py:76) is never filled."""
import math

import torch
import torch.nn as nn

from airgym_amd.lib.network.causal_conv import causal_conv, causal_conv_step, causal_conv_torch
from airgym_amd.lib.network.selective_scan import selective_scan, selective_scan_step, selective_scan_torch
from airgym_amd.lib.network.splitk_linear import linear


class SelectiveMemory(nn.Module):
    """units: inner channels; states: numbers remembered per channel (1 to 32); taps: steps the convolution sees (2 to 8)."""

    def __init__(self, size, units=64, states=16, taps=4):
        super().__init__()
        self.size, self.units, self.states, self.taps = int(size), int(units), int(states), int(taps)
        if not (1 <= self.states <= 32 and 2 <= self.taps <= 8 and self.units >= 1):
            raise ValueError(f"memory: units {units}, states {states} (1 to 32), taps {taps} (2 to 8)")
        rank = self.rank = (self.units + 15) // 16
        self.in_proj = nn.Linear(self.size, 2 * self.units, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(self.units, self.taps).uniform_(-1.0, 1.0) / math.sqrt(self.taps))
        self.conv_bias = nn.Parameter(torch.zeros(self.units))
        self.x_proj = nn.Linear(self.units, rank + 2 * self.states, bias=False)
        self.dt_weight = nn.Parameter(torch.empty(self.units, rank).uniform_(-1.0, 1.0) / math.sqrt(rank))
        # steps between 0.001 and 0.1, evenly over their logarithm: softplus(dt_bias) = step
        step = torch.exp(torch.rand(self.units) * math.log(100.0) + math.log(0.001))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, self.states + 1, dtype=torch.float32)).repeat(self.units, 1))
        self.D = nn.Parameter(torch.ones(self.units))
        self.out_proj = nn.Linear(self.units, self.size, bias=False)

    def initial_state(self, rows, device=None):
        """What `rows` sequences remember before their first step: (inputs of the convolution, states of the scan)."""
        device = self.D.device if device is None else device
        return (torch.zeros(rows, self.taps - 1, self.units, device=device), torch.zeros(rows, self.units, self.states, device=device))

    def _split(self, c):
        p = linear(c.reshape(-1, self.units), self.x_proj.weight).view(*c.shape[:-1], -1)
        dt, B, C = p.split((self.rank, self.states, self.states), -1)
        return dt @ self.dt_weight.t(), B, C

    def forward(self, x, state=None, resets=None, return_state=False):
        """x [rows, steps, size]; resets [rows, steps] (bool or uint8): what is remembered is cleared before that step."""
        rows, steps, _ = x.shape
        conv, scan = (causal_conv, selective_scan) if x.is_cuda else (causal_conv_torch, selective_scan_torch)
        inner, z = linear(x.reshape(-1, self.size), self.in_proj.weight).view(rows, steps, -1).split(self.units, -1)
        before = (None, None) if state is None else state
        c, conv_state = conv(inner, self.conv_weight, self.conv_bias, initial_state=before[0], resets=resets, return_state=True)
        delta, B, C = self._split(c)
        y, scan_state = scan(c, delta, -torch.exp(self.A_log), B, C, self.D, z, self.dt_bias, initial_state=before[1], resets=resets,
                             return_state=True)
        out = x + linear(y.reshape(-1, self.units), self.out_proj.weight).view_as(x)
        return (out, (conv_state, scan_state)) if return_state else out

    @torch.no_grad()
    def step(self, x, state, resets=None):
        """x [rows, size]; state (initial_state) is moved on in place."""
        if not x.is_cuda:
            out, new = self.forward(x.unsqueeze(1), state, None if resets is None else resets.unsqueeze(1), return_state=True)
            for old, value in zip(state, new):
                old.copy_(value)
            return out.squeeze(1)
        inner, z = torch.mm(x, self.in_proj.weight.t()).split(self.units, -1)
        c = causal_conv_step(inner, state[0], self.conv_weight, self.conv_bias, resets=resets)
        delta, B, C = self._split(c)
        y = selective_scan_step(c, delta, -torch.exp(self.A_log), B, C, state[1], self.D, z, self.dt_bias, resets=resets)
        return torch.addmm(x, y, self.out_proj.weight.t())


def forget(state):
    """Clears a state (initial_state) where it lies; None: nothing to clear."""
    for t in state or ():
        t.zero_()


class RolloutMemory:
    """What the update needs of a rollout's memory, per minibatch: slicing the flattened batch (env-major, whole sequences) gives the
    state each of its sequences started from and where episodes ended inside."""

    def __init__(self, state, dones, horizon):
        self.state, self.horizon = state, horizon
        self.resets = dones.view(-1, horizon)

    def __getitem__(self, sl):
        first, last = sl.start // self.horizon, sl.stop // self.horizon
        return {"state": tuple(s[first:last] for s in self.state), "resets": self.resets[first:last]}
