"""Log probabilities of given actions under softmax(logits / temperature), with the entropy and the
best alternatives: ``VanillaActorNetwork.get_action_prob`` (actor_networks.py:155-176) in logarithms, for
any number of actions, from the logits (``pa_action_log_probs``, log_probs.hip)."""
from __future__ import annotations

from ctypes import byref
from typing import Any, NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ... import _native as N
from ..common.token_ops import FLOATS, INDICES, dtype_code, on_one_gpu, scratch_of, wants_grad


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
    logits by index.  pi = softmax(logits / temperature) over the available actions; the mask ((..., A) or
    (A,), bool, True = unavailable) takes actions out, as does a logit of -inf.

    A row without an available action has log_prob -inf, entropy 0, alternatives -1.  Action -1 stands for
    "none taken" (padding): log_prob 0.  Any other action outside [0, A) gives NaN.  log_prob and entropy are
    differentiable with respect to the logits; the alternatives are not."""
    if wants_grad(logits):
        out = _ActionLogProbs.apply(logits, actions, unavailable_actions_mask, temperature, top)
        return ActionLogProbs(*out)
    return _log_probs(logits, actions, unavailable_actions_mask, temperature, top)


def _args(op: str, logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float) -> Tuple:
    device = logits.device
    if logits.dim() < 1 or logits.shape[:-1] != actions.shape:
        raise ValueError(f"{op}: logits have shape {tuple(logits.shape)}, actions {tuple(actions.shape)}, "
                         "not (..., A) and (...)")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"{op}: temperature {temperature}")
    a = N.LogProbsArgs()
    a.dtype = dtype_code(op, "logits", logits, FLOATS)
    a.action_dtype = dtype_code(op, "actions", actions, INDICES)
    width = logits.shape[-1]
    rows = actions.numel()
    flat = logits if logits.dim() == 2 else logits.reshape(rows, width)
    if flat.stride(1) != 1 and width > 1:
        flat = flat.contiguous()
    actions = actions.contiguous()
    a.A, a.rows, a.temperature = width, rows, temperature
    a.logits, a.ld, a.actions = flat.data_ptr(), flat.stride(0), actions.data_ptr()
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8) or (mask.shape != logits.shape and mask.shape != (width,)):
            raise ValueError(f"{op}: unavailable_actions_mask is {mask.dtype} {tuple(mask.shape)}, "
                             f"not bool {tuple(logits.shape)} or {(width,)}")
        if mask.dim() == 1 and logits.dim() != 1:
            mask = mask.contiguous()
        else:
            mask = mask.reshape(rows, width)
            if mask.stride(1) != 1 and width > 1:
                mask = mask.contiguous()
            a.ldm = mask.stride(0)
        a.mask = mask.data_ptr()
    on_one_gpu(op, device, actions, mask)
    a.device = device.index
    return a, (flat, actions, mask)


def _log_probs(logits: Tensor, actions: Tensor, mask: Optional[Tensor], temperature: float, top: int
               ) -> ActionLogProbs:
    if not 0 <= top <= 64:
        raise NotImplementedError(f"action_log_probs: top {top} (0 to 64)")
    a, alive = _args("action_log_probs", logits, actions, mask, temperature)
    device, shape = logits.device, actions.shape
    a.top = top
    log_prob = torch.empty(shape, dtype=torch.float32, device=device)
    entropy = torch.empty(shape, dtype=torch.float32, device=device)
    stats = torch.empty(*shape, 3, dtype=torch.float32, device=device)
    top_actions = top_log_probs = None
    if top:
        top_actions = torch.empty(*shape, top, dtype=torch.int64, device=device)
        top_log_probs = torch.empty(*shape, top, dtype=torch.float32, device=device)
        a.top_actions, a.top_log_probs = top_actions.data_ptr(), top_log_probs.data_ptr()
    lib = N.lib()
    scratch = scratch_of(lib.pa_action_log_probs_scratch(a.rows, a.A, a.dtype, top), device)
    a.log_prob, a.entropy, a.stats = log_prob.data_ptr(), entropy.data_ptr(), stats.data_ptr()
    a.scratch = N.ptr(scratch)
    N.check(lib.pa_action_log_probs(byref(a), N.stream_ptr(device)))
    del alive
    return ActionLogProbs(log_prob, entropy, top_actions, top_log_probs, stats)


def action_log_probs_grad(out: ActionLogProbs, logits: Tensor, actions: Tensor,
                          d_log_prob: Optional[Tensor] = None, d_entropy: Optional[Tensor] = None,
                          unavailable_actions_mask: Optional[Tensor] = None, temperature: float = 1.0) -> Tensor:
    """The logits' gradient, in their type, of ``action_log_probs`` called with the same arguments, for the
    float32 gradients of log_prob and of the entropy (None: zero)."""
    op = "action_log_probs_grad"
    a, alive = _args(op, logits, actions, unavailable_actions_mask, temperature)
    device, shape = logits.device, actions.shape
    stats = out.row_stats
    on_one_gpu(op, device, stats, d_log_prob, d_entropy)
    if stats.shape != (*shape, 3) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"{op}: out.row_stats is not what action_log_probs returns for these logits")
    grads = []
    for name, t in (("d_log_prob", d_log_prob), ("d_entropy", d_entropy)):
        if t is not None:
            if t.shape != shape or t.dtype != torch.float32:
                raise ValueError(f"{op}: {name} is {t.dtype} {tuple(t.shape)}, not float32 {tuple(shape)}")
            t = t.contiguous()
        grads.append(t)
    d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    a.stats = stats.data_ptr()
    a.d_log_prob, a.d_entropy, a.d_logits = N.ptr(grads[0]), N.ptr(grads[1]), d_logits.data_ptr()
    N.check(N.lib().pa_action_log_probs_grad(byref(a), N.stream_ptr(device)))
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
