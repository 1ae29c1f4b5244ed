"""Log probabilities of given actions under softmax(logits / temperature), with the entropy and the
best alternatives: ``VanillaActorNetwork.get_action_prob`` (actor_networks.py:155-176) in logarithms, for
any number of actions, from the logits (``pa_action_log_probs``, log_probs.hip)."""
from __future__ import annotations

from functools import lru_cache
from typing import Any, NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ... import _native as N
from ..common.token_ops import FLOATS, INDICES, _address, dtype_code, no_tangents, on_one_gpu, scratch_of


class ActionLogProbs(NamedTuple):
    log_prob: Tensor                    # (...) float32
    entropy: Tensor                     # (...) float32, in nats
    top_actions: Optional[Tensor]       # (..., top) int64, -1 where fewer actions are available
    top_log_probs: Optional[Tensor]     # (..., top) float32
    row_stats: Tensor                   # (..., 3) what action_log_probs_grad reads of the softmax


def action_log_probs(logits: Tensor, actions: Tensor, unavailable_actions_mask: Optional[Tensor] = None,
                     temperature: float = 1.0, top: int = 0) -> ActionLogProbs:
    """For logits (..., A) and integer actions (...): log pi(action), the entropy of pi and, for ``top`` > 0,
    the ``top`` (at most 64) most probable actions with their log probabilities, in falling order with equal
    logits by index.  pi = softmax(logits / temperature) over the available actions, for temperatures up to
    2^121; the mask ((..., A) or (A,), bool, True = unavailable) takes actions out, as does a logit of -inf.

    A row without an available action has log_prob -inf, entropy 0, alternatives -1.  Action -1 stands for
    "none taken" (padding): log_prob 0.  Any other action outside [0, A) gives NaN.  log_prob and entropy are
    differentiable with respect to the logits (backwards; logits with a forward-mode tangent are refused); the
    alternatives are not."""
    no_tangents("action_log_probs", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _ActionLogProbs.apply(logits, actions, unavailable_actions_mask, temperature, top)
        return ActionLogProbs(*out)
    return _log_probs(logits, actions, unavailable_actions_mask, temperature, top)


@lru_cache(maxsize=4096)
def _scratch_bytes(rows: int, width: int, code: int, top: int) -> int:
    return N.lib().pa_action_log_probs_scratch(rows, width, code, top)


def _inputs(op: str, logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float) -> Tuple:
    """Checks what both directions share; returns the head of the C arguments and what it points to."""
    shape = logits.shape
    if not shape or shape[:-1] != actions.shape:
        raise ValueError(f"{op}: logits have shape {tuple(logits.shape)}, actions {tuple(actions.shape)}, "
                         "not (..., A) and (...)")
    if not 0.0 < temperature <= 2.0 ** 121:
        raise ValueError(f"{op}: temperature {temperature} (up to 2^121)")
    code, action_code = dtype_code(op, "logits", logits, FLOATS), dtype_code(op, "actions", actions, INDICES)
    width, rows = shape[-1], actions.numel()
    if width >= 2 ** 31:
        raise NotImplementedError(f"{op}: {width} actions (up to 2^31 - 1)")
    flat = logits if len(shape) == 2 else logits.reshape(rows, width)
    if flat.stride(1) != 1 and width > 1:
        flat = flat.contiguous()
    actions = actions.contiguous()
    mask_ld = 0
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or (mask.shape != shape and mask.shape != shape[-1:]):
            raise ValueError(f"{op}: unavailable_actions_mask is {mask.dtype} {tuple(mask.shape)}, "
                             f"not bool {tuple(shape)} or {(width,)}")
        if mask.dim() == 1 and len(shape) != 1:
            mask = mask.contiguous()
        else:
            mask = mask if len(shape) == 2 else mask.reshape(rows, width)
            if mask.stride(1) != 1 and width > 1:
                mask = mask.contiguous()
            mask_ld = mask.stride(0)
    device = logits.device
    on_one_gpu(op, device, actions, mask)
    head = (device.index, code, action_code, width, rows, flat.data_ptr(), flat.stride(0), actions.data_ptr(),
            _address(mask), mask_ld, temperature)
    return head, (flat, actions, mask)


def _log_probs(logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float, top: int
               ) -> ActionLogProbs:
    if not 0 <= top <= 64:
        raise NotImplementedError(f"action_log_probs: top {top} (0 to 64)")
    head, alive = _inputs("action_log_probs", logits, actions, mask, temperature)
    device, shape = logits.device, actions.shape
    f32 = torch.float32
    log_prob = torch.empty(shape, dtype=f32, device=device)
    entropy = torch.empty(shape, dtype=f32, device=device)
    stats = torch.empty(*shape, 3, dtype=f32, device=device)
    top_actions = top_log_probs = None
    if top:
        top_actions = torch.empty(*shape, top, dtype=torch.int64, device=device)
        top_log_probs = torch.empty(*shape, top, dtype=f32, device=device)
    scratch = scratch_of(_scratch_bytes(head[4], head[3], head[1], top), device)
    args = N.LOG_PROBS_ARGS.pack(*head, top, log_prob.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                                 _address(top_actions), _address(top_log_probs), _address(scratch), 0, 0, 0)
    N.check(N.lib().pa_action_log_probs(args, N.stream_ptr(device)))
    del alive
    return ActionLogProbs(log_prob, entropy, top_actions, top_log_probs, stats)


def action_log_probs_grad(out: ActionLogProbs, logits: Tensor, actions: Tensor,
                          d_log_prob: Optional[Tensor] = None, d_entropy: Optional[Tensor] = None,
                          unavailable_actions_mask: Optional[Tensor] = None, temperature: float = 1.0) -> Tensor:
    """The logits' gradient, in their type, of ``action_log_probs`` called with the same arguments, for the
    float32 gradients of log_prob and of the entropy (None: zero)."""
    op = "action_log_probs_grad"
    no_tangents(op, logits, d_log_prob, d_entropy)
    head, alive = _inputs(op, logits, actions, unavailable_actions_mask, temperature)
    device, shape, stats = logits.device, actions.shape, out.row_stats
    on_one_gpu(op, device, stats, d_log_prob, d_entropy)
    if stats.shape != (*shape, 3) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"{op}: out.row_stats is not what action_log_probs returns for these logits")
    for name, t in (("d_log_prob", d_log_prob), ("d_entropy", d_entropy)):
        if t is not None and (t.shape != shape or t.dtype != torch.float32):
            raise ValueError(f"{op}: {name} is {t.dtype} {tuple(t.shape)}, not float32 {tuple(shape)}")
    d_log_prob = None if d_log_prob is None else d_log_prob.contiguous()
    d_entropy = None if d_entropy is None else d_entropy.contiguous()
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    args = N.LOG_PROBS_ARGS.pack(*head, 0, 0, 0, stats.data_ptr(), 0, 0, 0, _address(d_log_prob), _address(d_entropy),
                                 d_logits.data_ptr())
    N.check(N.lib().pa_action_log_probs_grad(args, N.stream_ptr(device)))
    del alive
    return d_logits


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float, top: int
                ) -> Tuple:
        out = _log_probs(logits, actions, mask, temperature, top)
        ctx.save_for_backward(logits, actions, mask, out.row_stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (out.top_actions, out.top_log_probs, out.row_stats) if t is not None])
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, d_log_prob: Optional[Tensor], d_entropy: Optional[Tensor], *_: Any) -> Tuple:
        logits, actions, mask, stats = ctx.saved_tensors
        if d_log_prob is None and d_entropy is None:
            return None, None, None, None, None
        out = ActionLogProbs(stats, stats, None, None, stats)      # the gradient reads the statistics alone
        return (action_log_probs_grad(out, logits, actions, d_log_prob, d_entropy, mask, ctx.temperature),
                None, None, None, None)
