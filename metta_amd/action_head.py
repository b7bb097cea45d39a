"""The action head on the device: from a policy's logits to actions, their log-probabilities and the entropy.

* `adjust_logits` -- penalties for repeated tokens, biases, temperature and masks applied to logits, with the gradient;
* `sample_actions` -- the rollout's form: adjust, pick one action per row, its log-probability and the row's entropy;
* `evaluate_actions` -- the training form: log-probability and entropy of stored actions, with the gradient;
* `pack_allowed` -- a boolean mask as bits, an eighth of its size.

The first three are HIP kernels on torch's current stream (metta_amd/csrc/action_head.hip), one launch each (two for sampling
and evaluation beyond 8192 tokens); there is no CPU path.
Log-probabilities, entropies and gradients are computed in 32 bits, or 64 where the choice of an action needed them.
They share these controls, all keyword arguments, for logits `[..., V]` of float32, bfloat16 or float16:

* `allowed`: bool `[V]` or `[..., V]`, or int32 bits `[ceil(V / 32)]` or `[..., ceil(V / 32)]` (`pack_allowed`);
* `bias`: float32 `[V]` or `[..., V]`, added before the temperature; a constant (one that requires a gradient is refused:
  a learned bias belongs to the projection that makes the logits);
* `history`: int32 `[..., L]`, recent tokens of the row; entries outside `[0, V)` (-1) are empty.  A token that stands in
  it c > 0 times has its logit divided by `repetition` if it is positive and multiplied otherwise, and then lowered by
  `frequency * c + presence`;
* `temperature`: what the result is divided by (it and `repetition`: from 1e-30 to 1e30).

    adjusted = allowed ? (penalised + bias) / temperature : -infinity

What stands at a masked token (NaN and infinities too) has no effect.  A row without an allowed token (or with -infinity
at all of them) gives action -1, log-probability 0, entropy 0 and no gradient; a row with NaN or +infinity at an allowed
token gives action -1 and NaN, and a gradient of NaN at every token that is left (allowed, and not at -infinity).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from metta_amd import native


def pack_allowed(allowed: Tensor) -> Tensor:
    """bool `[..., V]` -> int32 `[..., ceil(V / 32)]`: bit v % 32 of word v // 32 is token v's."""
    if allowed.dtype != torch.bool or allowed.dim() < 1 or allowed.size(-1) < 1:
        raise RuntimeError("allowed must be a bool tensor [..., V]")
    v = allowed.size(-1)
    bits = torch.nn.functional.pad(allowed, (0, -v % 32)).unflatten(-1, (-1, 32))
    weights = 1 << torch.arange(32, dtype=torch.int64, device=allowed.device)  # (made where they are used: also in a captured graph)
    weights = torch.where(weights > 0x7FFFFFFF, weights - (1 << 32), weights).to(torch.int32)
    return torch.where(bits, weights, 0).sum(-1, dtype=torch.int32)


def adjust_logits(
    logits: Tensor,
    *,
    allowed: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    history: Optional[Tensor] = None,
    temperature: float = 1.0,
    repetition: float = 1.0,
    presence: float = 0.0,
    frequency: float = 0.0,
) -> Tensor:
    """The adjusted logits (shape and type of `logits`, -infinity where masked), computed in 64 bits and rounded to 32 and
    to their type.  Differentiable once, in reverse mode, in `logits`."""
    return native.operators().adjust_logits(logits, allowed, bias, history, temperature, repetition, presence, frequency)


def sample_actions(
    logits: Tensor,
    uniforms: Optional[Tensor] = None,
    *,
    allowed: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    history: Optional[Tensor] = None,
    temperature: float = 1.0,
    repetition: float = 1.0,
    presence: float = 0.0,
    frequency: float = 0.0,
) -> Tuple[Tensor, Tensor, Tensor]:
    """(actions int32, log-probabilities float32, entropies float32), each of logits' shape without its last dimension.

    With `uniforms` (float32 in [0, 1), one per row, for instance `torch.rand`) the action is the first token at which the
    running sum of the probabilities exceeds the uniform, as 64-bit arithmetic finds it: the same numbers give the same
    actions whatever the shape of the batch.  (1 and more: the last token with any weight; below 0: as 0; NaN: action -1 and
    NaN.)  Without, it is the most likely token (the lowest of equals).  Carries no gradient; `evaluate_actions` does."""
    return native.operators().sample_actions(logits, uniforms, allowed, bias, history, temperature, repetition, presence, frequency)


def evaluate_actions(
    logits: Tensor,
    actions: Tensor,
    *,
    allowed: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    history: Optional[Tensor] = None,
    temperature: float = 1.0,
    repetition: float = 1.0,
    presence: float = 0.0,
    frequency: float = 0.0,
) -> Tuple[Tensor, Tensor]:
    """(log-probabilities, entropies), float32, of `actions` (int32 or int64, logits' shape without its last dimension)
    under the adjusted logits.  Differentiable once, in reverse mode, in `logits`.  An action that is masked or outside [0, V) has
    log-probability -infinity and passes no gradient of it."""
    return native.operators().evaluate_actions(logits, actions, allowed, bias, history, temperature, repetition, presence, frequency)
