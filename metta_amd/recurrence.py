"""Gated linear recurrence on the device: a recurrent core that trains over whole segments without a loop over time.

    h[t] = a[t] * (resets[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t],    a = sigmoid(gate),  h[-1] = state

element by element along the last dimension.  `gated_recurrence` runs `[rows, steps, width]` with gradients,
`gated_recurrence_step` one step of `[rows, width]` (the rollout's form).  Both are HIP kernels on torch's current stream
(`mg_gated_recurrence`, metta_amd/csrc/recurrence.hip); there is no CPU path.

Types: `x` and `gate` float32, bfloat16 or float16 (one type), `state` always float32; the state, the products along time
and the running gradient are kept in 32 bits, outputs and gradients are rounded once.  `x` and `gate` may be strided
views whose last dimension is adjacent (halves of one projection, a time-major tensor transposed); others are copied.
A padded tail is held by a gate of +infinity: the state passes such a step unchanged (with any finite x).
"""

from __future__ import annotations

import ctypes as ct
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from metta_amd import native

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # MG_F32, MG_BF16, MG_F16


def _launch(name: str, device: torch.device, *args) -> None:
    L = native.load()
    stream = torch._C._cuda_getCurrentRawStream(device.index)  # current_stream(device).cuda_stream without the objects
    if device.index == torch.cuda.current_device():
        rc = getattr(L, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(L, name)(*args, stream)
    if rc:
        native.check(rc, L)


def _halves(x: Tensor, gate: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    if gate is not None:
        return x, gate
    width = x.size(-1) // 2
    return x[..., :width], x[..., width:]


def _checked(x: Tensor, gate: Optional[Tensor], state: Optional[Tensor], resets: Optional[Tensor], dims: int) -> Tuple[Tensor, Tensor]:
    """The two inputs, after the checks that all entry points share."""
    if x.dim() != dims:
        raise RuntimeError(f"x must be {dims}D")
    if gate is None:
        if x.size(-1) % 2:
            raise RuntimeError("without a gate, x holds candidates and gates side by side: its last dimension must be even")
        x, gate = _halves(x, None)
    if gate.shape != x.shape:
        raise RuntimeError("x and gate must have the same shape")
    if x.dtype not in TYPES or gate.dtype != x.dtype:
        raise RuntimeError("x and gate must both be float32, bfloat16 or float16")
    lead = x.shape[:-1]
    if state is not None:
        if state.dtype != torch.float32:
            raise RuntimeError("state must be float32")
        if state.shape != (x.size(0), x.size(-1)):
            raise RuntimeError("state must be [rows, width]")
    if resets is not None:
        if resets.dtype not in (torch.bool, torch.uint8):
            raise RuntimeError("resets must be bool or uint8")
        if resets.shape != lead:
            raise RuntimeError("resets must have x's shape without its last dimension")
    if x.size(0) * x.size(-1) > 1 << 31:
        raise RuntimeError("rows * width must not exceed 2^31")
    for t in (x, gate, state, resets):
        if t is not None and t.device != x.device:
            raise RuntimeError("All tensors must be on same device")
    if x.device.type != "cuda":
        raise RuntimeError("All tensors must be on GPU")
    return x, gate


def _adjacent(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _args(x: Tensor, gate: Tensor, state: Optional[Tensor], resets: Optional[Tensor], steps: int) -> native.MgRecurrence:
    one = x.dim() == 2  # a single step: [rows, width]
    return native.MgRecurrence(
        x.data_ptr(), gate.data_ptr(), None if state is None else state.data_ptr(), None if resets is None else resets.data_ptr(),
        x.size(0), steps, x.size(-1), x.stride(0), 0 if one else x.stride(1), gate.stride(0), 0 if one else gate.stride(1), None, 0, TYPES[x.dtype],
    )  # fmt: skip


def _workspace(args: native.MgRecurrence, device: torch.device) -> Optional[Tensor]:
    """Memory of this call's own (torch's allocator keeps it for the stream, and for a captured graph), set in `args`."""
    size = native.load().mg_gated_recurrence_workspace(ct.byref(args))
    if not size:
        return None
    w = torch.empty(size, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = w.data_ptr(), size
    return w


def _forward(x: Tensor, gate: Optional[Tensor], state: Optional[Tensor], resets: Optional[Tensor], train: bool):
    xs, gs = _halves(x, gate)
    rows, steps, width = xs.shape
    h = torch.empty(rows, steps, width, dtype=x.dtype, device=x.device)
    last = torch.empty(rows, width, dtype=torch.float32, device=x.device)
    marks = None
    if train and x.dtype != torch.float32:
        marks = torch.empty(rows, (steps - 1) // native.MARK_STEPS, width, dtype=torch.float32, device=x.device)
    args = _args(xs, gs, state, resets, steps)
    w = _workspace(args, x.device)
    _launch("mg_gated_recurrence", x.device, ct.byref(args), h.data_ptr(), last.data_ptr(), None if marks is None else marks.data_ptr())
    del w
    return h, last, marks


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, resets):
        ctx.set_materialize_grads(False)
        h, last, marks = _forward(x, gate, state, resets, True)
        # an f32 output holds the states itself, in shorter types they are kept apart
        ctx.save_for_backward(x, gate, state, resets, h if marks is None else marks)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        if dh is None and dlast is None:
            return None, None, None, None
        # (what comes back may lie elsewhere and otherwise than what was saved: a hook may have moved it)
        x, gate, state, resets, marks = ctx.saved_tensors
        x, gate = _adjacent(x), None if gate is None else _adjacent(gate)
        state, resets, marks = (None if t is None else t.contiguous() for t in (state, resets, marks))
        xs, gs = _halves(x, gate)
        rows, steps, width = xs.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dgate = None if gate is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d1, d2 = _halves(dx, dgate)
        dstate = torch.empty_like(state) if ctx.needs_input_grad[2] else None
        if dh is not None:
            dh = _adjacent(dh)
        if dlast is not None:
            dlast = dlast.contiguous()
        f32 = x.dtype == torch.float32
        grads = native.MgRecurrenceGradients(
            None if dh is None else dh.data_ptr(), None if dlast is None else dlast.data_ptr(), d1.data_ptr(), d2.data_ptr(),
            None if dstate is None else dstate.data_ptr(), *((0, 0) if dh is None else dh.stride()[:2]), *d1.stride()[:2], *d2.stride()[:2],
        )  # fmt: skip
        at = marks.data_ptr() + (4 * (native.MARK_STEPS - 1) * width if f32 else 0)
        strides = (steps * width, native.MARK_STEPS * width) if f32 else ((steps - 1) // native.MARK_STEPS * width, width)
        args = _args(xs, gs, state, resets, steps)
        w = _workspace(args, x.device)
        _launch("mg_gated_recurrence_backward", x.device, ct.byref(args), at, *strides, ct.byref(grads))
        del w
        return dx, dgate, dstate, None


def gated_recurrence(x: Tensor, gate: Optional[Tensor] = None, state: Optional[Tensor] = None, resets: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """`x`, `gate` `[rows, steps, width]` -> (h `[rows, steps, width]` of x's type, last state `[rows, width]` float32).

    Without `gate`, `x` is `[rows, steps, 2 * width]`: candidates, then gates (one projection; its gradient comes back as
    one tensor).  `state` float32 `[rows, width]` enters step 0 (None: zeros); where `resets` (bool or uint8
    `[rows, steps]`) is set, the state entering that step is zero.  Differentiable once in x, gate and state."""
    xs, gs = _checked(x, gate, state, resets, 3)
    if state is not None:
        state = state.contiguous()
    if x.size(1) == 0 or xs.numel() == 0:
        last = torch.zeros(x.size(0), xs.size(2), dtype=torch.float32, device=x.device) if state is None else state.clone()
        return torch.empty_like(xs) + gs, last  # nothing to compute; part of the graph all the same
    if resets is not None:
        resets = resets.contiguous()
    x, gate = _adjacent(x), None if gate is None else _adjacent(gate)
    if torch.is_grad_enabled() and (x.requires_grad or (gate is not None and gate.requires_grad) or (state is not None and state.requires_grad)):
        return _GatedRecurrence.apply(x, gate, state, resets)
    return _forward(x, gate, state, resets, False)[:2]


def gated_recurrence_step(x: Tensor, gate: Optional[Tensor], state: Tensor, resets: Optional[Tensor] = None, out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One step: `x`, `gate` `[rows, width]` (gate None: `x` `[rows, 2 * width]`), `state` float32 `[rows, width]`, `resets`
    `[rows]` -> (h of x's type, new state float32).  For float32 inputs h IS the new state.

    `out_state` (contiguous float32 `[rows, width]`) receives the new state; it may be `state` itself, for a state that
    stays where it is.  Not differentiable: a call that would need gradients is refused."""
    xs, gs = _checked(x, gate, state, resets, 2)
    if torch.is_grad_enabled() and (xs.requires_grad or gs.requires_grad or state.requires_grad):
        raise RuntimeError("gated_recurrence_step has no gradient: call it under torch.no_grad(), or use gated_recurrence")
    if out_state is None:
        out_state = torch.empty(state.shape, dtype=torch.float32, device=xs.device)
    elif out_state.shape != state.shape or out_state.dtype != torch.float32 or out_state.device != xs.device or not out_state.is_contiguous():
        raise RuntimeError("out_state must be contiguous float32 [rows, width] on x's device")
    elif out_state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("out_state is written in place and must not require a gradient")
    elif 0 < abs(out_state.data_ptr() - state.data_ptr()) < 4 * state.numel():
        raise RuntimeError("out_state may be state itself, but not overlap it otherwise")
    h = out_state if xs.dtype == torch.float32 else torch.empty(xs.shape, dtype=xs.dtype, device=xs.device)
    if xs.numel():
        xs, gs, state = _adjacent(xs), _adjacent(gs), state.contiguous()
        if resets is not None:
            resets = resets.contiguous()
        _launch("mg_gated_recurrence", xs.device, ct.byref(_args(xs, gs, state, resets, 1)), None if h is out_state else h.data_ptr(),
                out_state.data_ptr(), None)  # fmt: skip
    return h, out_state
