"""The action head on the device: from a policy's logits to actions, their log-probabilities and the entropy.

* `adjust_logits` -- penalties for repeated tokens, biases, temperature and masks applied to logits, with the gradient;
* `sample_actions` -- the rollout's form: adjust, pick one action per row, its log-probability and the row's entropy;
* `evaluate_actions` -- the training form: log-probability and entropy of stored actions, with the gradient;
* `pack_allowed` -- a boolean mask as bits, an eighth of its size.

The first three are single HIP kernels on torch's current stream (metta_amd/csrc/action_head.hip); there is no CPU path.
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
token gives action -1 and NaN.
"""

from __future__ import annotations

import ctypes as ct
import math
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from metta_amd import native
from metta_amd.recurrence import TYPES, _launch


def pack_allowed(allowed: Tensor) -> Tensor:
    """bool `[..., V]` -> int32 `[..., ceil(V / 32)]`: bit v % 32 of word v // 32 is token v's."""
    if allowed.dtype != torch.bool or allowed.dim() < 1 or allowed.size(-1) < 1:
        raise RuntimeError("allowed must be a bool tensor [..., V]")
    v = allowed.size(-1)
    bits = torch.nn.functional.pad(allowed, (0, -v % 32)).unflatten(-1, (-1, 32))
    weights = 1 << torch.arange(32, dtype=torch.int64, device=allowed.device)  # (made where they are used: also in a captured graph)
    weights = torch.where(weights > 0x7FFFFFFF, weights - (1 << 32), weights).to(torch.int32)
    return torch.where(bits, weights, 0).sum(-1, dtype=torch.int32)


class _Head:
    """Checked arguments of one call; keeps what the C structure points at alive."""

    __slots__ = ("logits", "bias", "allowed", "history", "args", "lead")

    def __init__(self, logits, allowed, bias, history, temperature, repetition, presence, frequency, gradient=True):
        if logits.dim() < 1 or logits.size(-1) < 1:
            raise RuntimeError("logits must be [..., V] with at least one token")
        if logits.dtype not in TYPES:
            raise RuntimeError("logits must be float32, bfloat16 or float16")
        lead, v = logits.shape[:-1], logits.size(-1)
        if v >= 1 << 31:
            raise RuntimeError("logits must have fewer than 2^31 tokens")
        device = logits.device
        for name, x in (("temperature", temperature), ("repetition", repetition)):
            if not 1e-30 <= x <= 1e30:
                raise RuntimeError(f"{name} must be from 1e-30 to 1e30")
        if not (math.isfinite(presence) and math.isfinite(frequency)):
            raise RuntimeError("presence and frequency must be finite")
        for t in (allowed, bias, history):
            if t is not None and t.device != device:
                raise RuntimeError("All tensors must be on same device")
        kind = width = 0
        if allowed is not None:
            if allowed.dtype == torch.bool:
                kind, width = native.ALLOWED_BOOL, v
            elif allowed.dtype == torch.int32:
                kind, width = native.ALLOWED_BITS, (v + 31) // 32
            else:
                raise RuntimeError("allowed must be bool, or int32 bits (pack_allowed)")
        if bias is not None:
            if bias.dtype != torch.float32:
                raise RuntimeError("bias must be float32")
            if gradient and bias.requires_grad and torch.is_grad_enabled():
                raise RuntimeError("bias is a constant: it must not require a gradient")
        if history is not None:
            if history.dtype != torch.int32:
                raise RuntimeError("history must be int32")
            if history.shape[:-1] != lead or history.dim() < 1:
                raise RuntimeError("history must be [..., L] with the logits' leading dimensions")
            if history.size(-1) > 1 << 30:
                raise RuntimeError("history must have at most 2^30 entries")
            if history.size(-1) == 0 or (repetition == 1.0 and presence == 0.0 and frequency == 0.0):
                history = None
        elif repetition != 1.0 or presence != 0.0 or frequency != 0.0:
            raise RuntimeError("penalties need a history")
        allowed, allowed_row = self._control("allowed", allowed, lead, width)
        bias, bias_row = self._control("bias", bias, lead, v)
        if device.type != "cuda":
            raise RuntimeError("All tensors must be on GPU")
        logits = self._rows(logits)
        history = None if history is None else self._rows(history)
        self.logits, self.bias, self.allowed, self.history, self.lead = logits, bias, allowed, history, lead
        self.args = native.MgLogits(
            logits.data_ptr(), None if bias is None else bias.data_ptr(), None if allowed is None else allowed.data_ptr(),
            None if history is None else history.data_ptr(), logits.size(0), logits.stride(0), bias_row, allowed_row,
            0 if history is None else history.stride(0), temperature, repetition, presence, frequency, None, 0, v,
            0 if history is None else history.size(1), kind, TYPES[logits.dtype],
        )  # fmt: skip

    @staticmethod
    def _rows(t: Tensor) -> Tensor:
        """[..., V] as [rows, V] with adjacent columns, a view where the strides allow it."""
        t = t.detach()
        if t.dim() != 2:
            t = t.reshape(-1, t.size(-1)) if t.dim() > 1 else t.unsqueeze(0)
        return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()

    def _control(self, name: str, t: Optional[Tensor], lead, width: int) -> Tuple[Optional[Tensor], int]:
        """A control and its row stride: 0 where one row serves all."""
        if t is None:
            return None, 0
        if t.dim() < 1 or t.size(-1) != width or (t.dim() > 1 and t.shape[:-1] != lead):
            raise RuntimeError(f"{name} must be [{width}] or [..., {width}] with the logits' leading dimensions")
        if t.dim() == 1:
            return t.detach().contiguous(), 0
        t = self._rows(t)
        return t, t.stride(0)


def _workspace(args: native.MgLogits, device: torch.device) -> Optional[Tensor]:
    """Memory of this call's own (torch's allocator keeps it for the stream, and for a captured graph), set in `args`."""
    size = native.load().mg_logits_workspace(ct.byref(args)) if args.width > native.STATS_WIDTH else 0
    if not size:
        return None
    w = torch.empty(size, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = w.data_ptr(), size
    return w


def _per_row(name: str, t: Tensor, dtypes, lead, device) -> Tensor:
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}")
    if t.shape != lead:
        raise RuntimeError(f"{name} must have the logits' shape without its last dimension")
    if t.device != device:
        raise RuntimeError("All tensors must be on same device")
    return t.detach().contiguous()


def _adjust(shape, head: _Head) -> Tensor:
    out = torch.empty(shape, dtype=head.logits.dtype, device=head.logits.device)
    if out.numel():
        _launch("mg_adjust_logits", out.device, ct.byref(head.args), out.data_ptr())
    return out


def _evaluate(head: _Head, actions: Tensor, train: bool):
    device = head.logits.device
    logp = torch.empty(head.lead, dtype=torch.float32, device=device)
    entropy = torch.empty_like(logp)
    wide = train and head.args.width > native.STATS_WIDTH
    stats = torch.empty(*head.lead, 2, dtype=torch.float64, device=device) if wide else None
    if logp.numel():
        w = _workspace(head.args, device)
        _launch("mg_evaluate_actions", device, ct.byref(head.args), actions.data_ptr(), logp.data_ptr(), entropy.data_ptr(),
                None if stats is None else stats.data_ptr())  # fmt: skip
        del w
    return logp, entropy, stats


def _save(ctx, head: _Head, shape, *more) -> None:
    # through save_for_backward, so that a tensor changed in between is noticed
    ctx.save_for_backward(head.logits, head.bias, head.allowed, head.history, *more)
    ctx.args, ctx.shape = head.args, shape


def _saved(ctx):
    """The arguments, pointing at what was saved (which a hook may have moved: it may lie elsewhere and otherwise), and the
    rest of what was saved."""
    logits, bias, allowed, history, *more = ctx.saved_tensors
    a = native.MgLogits.from_buffer_copy(ctx.args)
    kept = []
    for name, t in (("logits", logits), ("bias", bias), ("allowed", allowed), ("history", history)):
        if t is None:
            continue
        if t.stride(-1) != 1 and t.size(-1) != 1:
            t = t.contiguous()
        kept.append(t)
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_row", t.stride(0) if t.dim() == 2 else 0)
    return a, kept, more


class _AdjustLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, head):
        _save(ctx, head, logits.shape)
        return _adjust(logits.shape, head)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        d = torch.empty(ctx.shape, dtype=dout.dtype, device=dout.device)
        if d.numel():
            args, kept, _ = _saved(ctx)
            dout = dout.contiguous()
            _launch("mg_adjust_logits_backward", d.device, ct.byref(args), dout.data_ptr(), d.data_ptr())
        return d, None


class _EvaluateActions(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, head, actions):
        ctx.set_materialize_grads(False)
        logp, entropy, stats = _evaluate(head, actions, True)
        _save(ctx, head, logits.shape, actions, entropy, stats)
        return logp, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy):
        if dlogp is None and dentropy is None:
            return None, None, None
        args, kept, (actions, entropy, stats) = _saved(ctx)
        d = torch.empty(ctx.shape, dtype=kept[0].dtype, device=kept[0].device)
        if d.numel():
            dlogp, dentropy, actions, entropy, stats = (None if t is None else t.contiguous() for t in (dlogp, dentropy, actions, entropy, stats))
            _launch("mg_evaluate_actions_backward", d.device, ct.byref(args), actions.data_ptr(), entropy.data_ptr(),
                    None if stats is None else stats.data_ptr(), None if dlogp is None else dlogp.data_ptr(),
                    None if dentropy is None else dentropy.data_ptr(), d.data_ptr())  # fmt: skip
        return d, None, None


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
    """The adjusted logits (shape and type of `logits`, -infinity where masked), computed in 64 bits and rounded once.
    Differentiable once in `logits`."""
    head = _Head(logits, allowed, bias, history, temperature, repetition, presence, frequency)
    if logits.requires_grad and torch.is_grad_enabled():
        return _AdjustLogits.apply(logits, head)
    return _adjust(logits.shape, head)


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
    actions whatever the shape of the batch.  Without, it is the most likely token (the lowest of equals).  Carries no
    gradient; `evaluate_actions` does."""
    head = _Head(logits, allowed, bias, history, temperature, repetition, presence, frequency, gradient=False)
    if uniforms is not None:
        uniforms = _per_row("uniforms", uniforms, (torch.float32,), head.lead, logits.device)
    actions = torch.empty(head.lead, dtype=torch.int32, device=logits.device)
    logp = torch.empty(head.lead, dtype=torch.float32, device=logits.device)
    entropy = torch.empty_like(logp)
    if actions.numel():
        w = _workspace(head.args, logits.device)
        _launch("mg_sample_actions", logits.device, ct.byref(head.args), None if uniforms is None else uniforms.data_ptr(), actions.data_ptr(),
                logp.data_ptr(), entropy.data_ptr())  # fmt: skip
        del w
    return actions, logp, entropy


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
    under the adjusted logits.  Differentiable once in `logits`.  An action that is masked or outside [0, V) has
    log-probability -infinity and passes no gradient of it."""
    head = _Head(logits, allowed, bias, history, temperature, repetition, presence, frequency)
    actions = _per_row("actions", actions, (torch.int32, torch.int64), head.lead, logits.device)
    if actions.dtype == torch.int64:  # kept outside [0, V) where it is outside
        actions = actions.clamp(-1, 2**31 - 1).to(torch.int32)
    if logits.requires_grad and torch.is_grad_enabled():
        return _EvaluateActions.apply(logits, head, actions)
    return _evaluate(head, actions, False)[:2]
