"""Device-resident rollout loop with a recurrent policy.

The reference's `CoreTrainingLoop.rollout_phase` (`metta/rl/training/core.py:67-189`) copies observations host ->
device and actions device -> host every iteration.  Here observations, rewards and actions never leave HBM: the
policy reads `vecenv.observations` in place and `send` hands the action tensor's device pointer to the step
kernels (`mg_step_actions`).

`LSTMPolicy` is the mettagrid-package reference policy (`PY/policy/lstm.py:19-36`): flatten [T*3] uint8 tokens ->
Linear(128) -> Linear(128) -> LSTM(128) -> action logits / value.

`GatedRecurrentPolicy` has a gated linear recurrence for a core: the same step during the rollout, but whole segments at
once in training (`evaluate`), episodes ending inside them included.
"""

from __future__ import annotations

import time
from typing import Optional

import torch
import torch.nn as nn

from metta_amd.action_head import sample_actions
from metta_amd.recurrence import gated_recurrence, gated_recurrence_step


class LSTMPolicy(nn.Module):
    def __init__(self, num_tokens: int, num_actions: int, hidden: int = 128):
        super().__init__()
        self.enc = nn.Sequential(nn.Linear(num_tokens * 3, hidden), nn.ReLU(), nn.Linear(hidden, hidden), nn.ReLU())
        self.rnn = nn.LSTMCell(hidden, hidden)
        self.pi = nn.Linear(hidden, num_actions)
        self.v = nn.Linear(hidden, 1)
        self.hidden = hidden

    def initial_state(self, n: int, device, dtype=torch.float32):
        z = torch.zeros(n, self.hidden, device=device, dtype=dtype)
        return z, z.clone()

    def forward(self, obs_u8: torch.Tensor, state):
        x = obs_u8.reshape(obs_u8.shape[0], -1).to(self.enc[0].weight.dtype) * (1.0 / 255.0)
        h, c = self.rnn(self.enc(x), state)
        return self.pi(h), self.v(h).squeeze(-1), (h, c)


class GatedRecurrentPolicy(nn.Module):
    """`LSTMPolicy` with h[t] = a h[t-1] + (1 - a) x, a = sigmoid(gate), in place of the LSTM (metta_amd/recurrence.py).

    The state is one float32 tensor whatever the parameters' type.  Steps take the resets themselves (`takes_resets`):
    where an agent's episode has ended, its state is dropped inside the kernel."""

    takes_resets = True

    def __init__(self, num_tokens: int, num_actions: int, hidden: int = 128):
        super().__init__()
        self.enc = nn.Sequential(nn.Linear(num_tokens * 3, hidden), nn.ReLU(), nn.Linear(hidden, hidden), nn.ReLU())
        self.core = nn.Linear(hidden, 2 * hidden)  # candidates, then gates
        self.pi = nn.Linear(hidden, num_actions)
        self.v = nn.Linear(hidden, 1)
        self.hidden = hidden

    def initial_state(self, n: int, device, dtype=None):
        return (torch.zeros(n, self.hidden, device=device, dtype=torch.float32),)

    def _encode(self, obs_u8: torch.Tensor) -> torch.Tensor:
        x = obs_u8.flatten(-2).to(self.enc[0].weight.dtype) * (1.0 / 255.0)
        return self.core(self.enc(x))

    def forward(self, obs_u8: torch.Tensor, state, resets: Optional[torch.Tensor] = None):
        """One step of `[n, tokens, 3]`, without gradients."""
        with torch.no_grad():
            h, s = gated_recurrence_step(self._encode(obs_u8), None, state[0], resets)
            return self.pi(h), self.v(h).squeeze(-1), (s,)

    def evaluate(self, obs_u8: torch.Tensor, state=None, resets: Optional[torch.Tensor] = None):
        """Whole segments `[rows, steps, tokens, 3]` with gradients: (logits, values, the state after the last step)."""
        h, s = gated_recurrence(self._encode(obs_u8), None, None if state is None else state[0], resets)
        return self.pi(h), self.v(h).squeeze(-1), (s,)


def reset_state(policy, state, done: torch.Tensor):
    """The state that enters a step: zero where `done`, unless the policy does that itself."""
    if getattr(policy, "takes_resets", False):
        return state
    keep = 1 - done.to(state[0].dtype).unsqueeze(1)
    return tuple(s * keep for s in state)


class ActionControls:
    """Controls of the action head (`allowed`, `bias`, `temperature`, `repetition`, `presence`, `frequency`; see
    metta_amd/action_head.py) for a rollout, and the recent actions that the penalties look at: the last `history_length`
    of every agent, forgotten when its episode ends (an environment that is started anew wants new controls).  `rollout` and
    `rollout_phase` keep histories of their own."""

    def __init__(self, history_length: int = 0, **controls):
        if "history" in controls:
            raise ValueError("the rollout keeps the history itself: give history_length")
        self.history_length = int(history_length)
        self.controls = controls
        self._recent: dict = {}  # per slice of agents: [int32 [n, history_length], steps]

    def history(self, key, n: int, device) -> Optional[torch.Tensor]:
        """int32 [n, history_length], -1 where there is no action yet; written by `took` and `ended`."""
        if not self.history_length:
            return None
        if key not in self._recent:
            self._recent[key] = [torch.full((n, self.history_length), -1, dtype=torch.int32, device=device), 0]
        h = self._recent[key][0]
        d = torch.device(device)
        if h.shape[0] != n or h.device.type != d.type or d.index not in (None, h.device.index):
            raise ValueError(f"this history is of {h.shape[0]} agents on {h.device}, not of {n} on {device}: another environment wants new controls")
        return h

    def ended(self, key, done: torch.Tensor) -> None:
        if key in self._recent:
            self._recent[key][0].masked_fill_(done.unsqueeze(1), -1)

    def took(self, key, actions: torch.Tensor) -> None:
        if key in self._recent:
            h, steps = self._recent[key]
            h[:, steps % self.history_length] = actions  # (the order of the entries is of no account)
            self._recent[key][1] = steps + 1

    def sample(self, logits: torch.Tensor, history: Optional[torch.Tensor], generator=None):
        """(actions, log-probabilities, entropies) of one step."""
        u = torch.rand(logits.shape[:-1], device=logits.device, generator=generator)
        return sample_actions(logits, u, history=history, **self.controls)


@torch.no_grad()
def rollout(vecenv, policy, steps: int, state=None, generator=None, controls: Optional[ActionControls] = None):
    """`steps` iterations of recv -> policy -> send, all on the device.  Returns (agent_steps, seconds, state, infos).
    With `controls` the action head's kernels pick the actions, otherwise softmax and multinomial do."""
    dev = vecenv.observations.device
    n = vecenv.num_agents
    if state is None:
        state = policy.initial_state(n, dev, next(policy.parameters()).dtype)
    infos_all = []
    torch.cuda.synchronize(dev)
    t0 = time.perf_counter()
    for _ in range(steps):
        o, r, d, t, ta, infos, ids, mask = vecenv.recv()
        done = d | t
        if getattr(policy, "takes_resets", False):
            logits, value, state = policy(o, state, done)
        else:
            logits, value, state = policy(o, state)
            state = reset_state(policy, state, done)  # reset recurrent state where an episode ended
        if controls is None:
            actions = torch.multinomial(torch.softmax(logits.float(), dim=-1), 1, generator=generator).squeeze(1).to(torch.int32)
        else:
            history = controls.history(0, n, dev)
            controls.ended(0, done)
            actions, _, _ = controls.sample(logits, history, generator)
            controls.took(0, actions)
        vecenv.send(actions)
        if infos:
            infos_all.extend(infos)
    torch.cuda.synchronize(dev)
    return n * steps, time.perf_counter() - t0, state, infos_all
