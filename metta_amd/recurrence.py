"""Gated linear recurrence on the device: a recurrent core that trains over whole segments without a loop over time.

    h[t] = a[t] * (resets[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t],    a = sigmoid(gate),  h[-1] = state

element by element along the last dimension.  `gated_recurrence` runs `[rows, steps, width]` with gradients,
`gated_recurrence_step` one step of `[rows, width]` (the rollout's form).  Both are HIP kernels on torch's current stream
(`mg_gated_recurrence`, metta_amd/csrc/recurrence.hip); there is no CPU path.

Types: `x` and `gate` float32, bfloat16 or float16 (one type), `state` always float32; the state, the products along time
and the running gradient are kept in 32 bits, outputs and gradients are rounded once.  `x` and `gate` may be strided
views whose last dimension is adjacent (halves of one projection, a time-major tensor transposed); others are copied.
A padded tail is held by a gate of +infinity: the state passes such a step unchanged (with any finite x).
NaN goes as far as the formula takes it, up to the next reset.  An infinite state stays one that is not finite, infinity or
NaN (joined stretches multiply factors first, and a product that underflowed to 0 makes NaN of infinity).
"""

from __future__ import annotations

from typing import Optional, Tuple

from torch import Tensor

from metta_amd import native


def gated_recurrence(x: Tensor, gate: Optional[Tensor] = None, state: Optional[Tensor] = None, resets: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """`x`, `gate` `[rows, steps, width]` -> (h `[rows, steps, width]` of x's type, last state `[rows, width]` float32).

    Without `gate`, `x` is `[rows, steps, 2 * width]`: candidates, then gates (one projection; its gradient comes back as
    one tensor).  `state` float32 `[rows, width]` enters step 0 (None: zeros); where `resets` (bool or uint8
    `[rows, steps]`) is set, the state entering that step is zero.  Differentiable once, in reverse mode, in x, gate and state."""
    return native.operators().gated_recurrence(x, gate, state, resets)


def gated_recurrence_step(x: Tensor, gate: Optional[Tensor], state: Tensor, resets: Optional[Tensor] = None, out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One step: `x`, `gate` `[rows, width]` (gate None: `x` `[rows, 2 * width]`), `state` float32 `[rows, width]`, `resets`
    `[rows]` -> (h of x's type, new state float32).  For float32 inputs h IS the new state.

    `out_state` (contiguous float32 `[rows, width]`) receives the new state; it may be `state` itself, for a state that
    stays where it is, or a float32 `x` or `gate`, element on element.  Any other overlap with what the call reads is
    refused.  Not differentiable: a call that would need gradients is refused."""
    return native.operators().gated_recurrence_step(x, gate, state, resets, out_state)
