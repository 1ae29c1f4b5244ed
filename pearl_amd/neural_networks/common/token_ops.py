"""Differentiable operators for policies over tokens and histories, each one HIP launch sequence of
libpearl_amd (embed.hip, recurrence.hip):

* ``embed_tokens`` — rows of a table by token: ``OneHotActionTensorRepresentationModule`` followed by a
  dense layer, without the one-hot matrix;
* ``gated_recurrence`` — a gated linear recurrence over a history, with episode starts inside it;
  ``gated_recurrence_step`` is its single step for acting.

Parameters and results are torch tensors in HBM (float32, bfloat16 or float16); work runs on the
current stream of the tensors' device, which need not be the current device.  The functions record
a backward pass when gradients are asked for; ``embed_tokens_grad`` and ``gated_recurrence_grad`` are
the same kernels for learners that run their backward pass explicitly."""
from __future__ import annotations

from ctypes import byref
from typing import Any, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ... import _native as N

FLOATS = {torch.float32: N.PA_F32, torch.bfloat16: N.PA_BF16, torch.float16: N.PA_F16}
INDICES = {torch.int64: N.PA_I64, torch.int32: N.PA_I32}


def on_one_gpu(op: str, device: torch.device, *others: Optional[Tensor]) -> None:
    """After the other checks: the tensors lie on one GPU."""
    if device.type != "cuda":
        raise N.NativeError(f"{op}: tensors on {device}; the operator is a HIP kernel for gfx950, "
                            "there is no CPU fallback")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{op}: tensors on {t.device} and on {device}")


def dtype_code(op: str, name: str, t: Tensor, table: dict) -> int:
    code = table.get(t.dtype)
    if code is None:
        raise TypeError(f"{op}: {name} is {t.dtype}, not one of "
                        f"{', '.join(str(k).replace('torch.', '') for k in table)}")
    return code


def scratch_of(nbytes: int, device: torch.device) -> Optional[Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def wants_grad(*tensors: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------- embedding
def embed_tokens(weight: Tensor, tokens: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * weight[tokens]``, rounded once: (vocab, dim) and integer tokens of any shape give
    ``tokens.shape + (dim,)`` in the weight's type.

    Token -1 stands for "none": a row of zeros that takes no part in the gradient.  Any other token
    outside the table gives a row of NaN; nothing is read for it.  The weight's gradient is dense,
    summed in float32 in the order of the tokens and the same bits for the same inputs."""
    if wants_grad(weight):
        return _EmbedTokens.apply(weight, tokens, scale)
    return _embed(weight, tokens, scale)


def _embed(weight: Tensor, tokens: Tensor, scale: float) -> Tensor:
    if weight.dim() != 2:
        raise ValueError(f"embed_tokens: weight has {weight.dim()} dimensions, not (vocab, dim)")
    code = dtype_code("embed_tokens", "weight", weight, FLOATS)
    index = dtype_code("embed_tokens", "tokens", tokens, INDICES)
    on_one_gpu("embed_tokens", weight.device, tokens)
    vocab, dim = weight.shape
    if weight.stride(1) != 1 or weight.stride(0) < dim:
        weight = weight.contiguous()
    tokens = tokens.contiguous()
    out = torch.empty(*tokens.shape, dim, dtype=weight.dtype, device=weight.device)
    N.check(N.lib().pa_embed_tokens(weight.data_ptr(), code, max(weight.stride(0), dim), vocab, dim,
                                    tokens.data_ptr(), index, tokens.numel(), scale, out.data_ptr(),
                                    weight.device.index, N.stream_ptr(weight.device)))
    return out


def embed_tokens_grad(d_out: Tensor, tokens: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """The gradient of ``embed_tokens`` with respect to its (vocab, dim) weight, in ``d_out``'s type."""
    code = dtype_code("embed_tokens_grad", "d_out", d_out, FLOATS)
    index = dtype_code("embed_tokens_grad", "tokens", tokens, INDICES)
    if d_out.dim() < 1 or d_out.shape[:-1] != tokens.shape:
        raise ValueError(f"embed_tokens_grad: d_out has shape {tuple(d_out.shape)}, the tokens "
                         f"{tuple(tokens.shape)}")
    on_one_gpu("embed_tokens_grad", d_out.device, tokens)
    n, dim = tokens.numel(), d_out.shape[-1]
    rows = d_out if d_out.dim() == 2 else d_out.reshape(n, dim)
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    tokens = tokens.contiguous()
    lib = N.lib()
    d_weight = torch.empty(vocab, dim, dtype=d_out.dtype, device=d_out.device)
    scratch = scratch_of(lib.pa_embed_tokens_grad_scratch(n, dim, code), d_out.device)
    N.check(lib.pa_embed_tokens_grad(rows.data_ptr(), code, rows.stride(0), tokens.data_ptr(), index, n, scale,
                                     vocab, dim, d_weight.data_ptr(), N.ptr(scratch), d_out.device.index,
                                     N.stream_ptr(d_out.device)))
    return d_weight


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, weight: Tensor, tokens: Tensor, scale: float) -> Tensor:
        out = _embed(weight, tokens, scale)
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, d_out: Tensor) -> Tuple[Tensor, None, None]:
        tokens, = ctx.saved_tensors
        return embed_tokens_grad(d_out, tokens, ctx.vocab, ctx.scale), None, None


# ---------------------------------------------------------------------------- recurrence
def gated_recurrence(x: Tensor, gate: Tensor, initial_state: Optional[Tensor] = None,
                     resets: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                     gate_logits: bool = True, reverse: bool = False, keep: bool = False) -> Tuple:
    """The states of a gated linear recurrence over (batch, time, channels) and the last of them::

        gate_logits=True:   h_t = a_t h_{t-1} + (1 - a_t) x_t,   a_t = sigmoid(gate_t)
        gate_logits=False:  h_t = gate_t h_{t-1} + x_t

    ``gate`` has x's shape and its type, or float32 (decays close to one need it).  The state is float32
    throughout: ``initial_state`` (batch, channels; zeros if None) and the returned last state are
    float32, h is rounded to x's type.  ``resets`` (batch, time; bool) marks steps that begin an episode
    and ignore the state before them; ``lengths`` (batch) ends histories early: behind the end h is
    zero, whatever x and gate hold there.  ``reverse`` runs from the last step to the first, as advantage
    sums do (a reset there marks the last step of an episode).

    Returns ``(h, last_state)``.  With ``keep=True`` no backward pass is recorded and a third result is
    what ``gated_recurrence_grad`` needs of the forward pass."""
    if not keep and wants_grad(x, gate, initial_state):
        return _GatedRecurrence.apply(x, gate, initial_state, resets, lengths, gate_logits, reverse)
    h, last, kept = _recurrence(x, gate, initial_state, resets, lengths, gate_logits, reverse, keep)
    return (h, last, kept) if keep else (h, last)


def _rows(t: Tensor) -> Tensor:
    """(batch, time, channels) with adjacent channels, and steps less than the kernels' 2^23 bytes apart."""
    near = t.stride(1) * t.element_size() < 2 ** 23 or t.shape[1] == 1
    return t if near and (t.stride(2) == 1 or t.shape[2] == 1) else t.contiguous()


def _strides(t: Tensor) -> Tuple[int, int]:
    return t.stride(0), t.stride(1) if t.shape[1] > 1 else 0      # a single step's stride means nothing


def _recurrence_args(op: str, x: Tensor, gate: Tensor, initial_state: Optional[Tensor], resets: Optional[Tensor],
                     lengths: Optional[Tensor], gate_logits: bool, reverse: bool, a: N.RecurrenceArgs) -> Tuple:
    """Checks the arguments that both directions share and fills them in; returns what must stay alive."""
    device = x.device
    if x.dim() != 3 or gate.shape != x.shape:
        raise ValueError(f"{op}: x has shape {tuple(x.shape)} and gate {tuple(gate.shape)}, "
                         "not twice (batch, time, channels)")
    a.dtype = dtype_code(op, "x", x, FLOATS)
    a.gate_dtype = dtype_code(op, "gate", gate, FLOATS)
    if gate.dtype != x.dtype and gate.dtype != torch.float32:
        raise TypeError(f"{op}: gate is {gate.dtype}, x is {x.dtype}: the gate has x's type or float32")
    b, t, d = x.shape
    x, gate = _rows(x), _rows(gate)
    a.gate_logits, a.reverse = bool(gate_logits), bool(reverse)
    a.B, a.T, a.D = b, t, d
    a.x, a.gate = x.data_ptr(), gate.data_ptr()
    a.x_b, a.x_t = _strides(x)
    a.gate_b, a.gate_t = _strides(gate)
    if initial_state is not None:
        if initial_state.shape != (b, d) or initial_state.dtype != torch.float32:
            raise ValueError(f"{op}: initial_state is {initial_state.dtype} {tuple(initial_state.shape)}, "
                             f"not float32 {(b, d)}")
        initial_state = initial_state.contiguous()
        a.h0 = initial_state.data_ptr()
    if resets is not None:
        if resets.shape != (b, t) or resets.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"{op}: resets is {resets.dtype} {tuple(resets.shape)}, not bool {(b, t)}")
        a.resets = resets.data_ptr()
        if resets.stride(1) >= 2 ** 23:
            resets = resets.contiguous()
        a.resets_b, a.resets_t = _strides(resets)
    if lengths is not None:
        if lengths.shape != (b,) or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{op}: lengths is {lengths.dtype} {tuple(lengths.shape)}, not int32 or int64 {(b,)}")
        # clamped before the cast, so that no length wraps around
        on_one_gpu(op, device, lengths)
        lengths = (lengths.clamp(0, t).to(torch.int32) if lengths.dtype == torch.int64 else lengths).contiguous()
        a.lengths = lengths.data_ptr()
    on_one_gpu(op, device, gate, initial_state, resets)
    a.device = device.index
    return x, gate, initial_state, resets, lengths


def _recurrence(x: Tensor, gate: Tensor, initial_state: Optional[Tensor], resets: Optional[Tensor],
                lengths: Optional[Tensor], gate_logits: bool, reverse: bool, keep: bool) -> Tuple:
    a = N.RecurrenceArgs()
    alive = _recurrence_args("gated_recurrence", x, gate, initial_state, resets, lengths, gate_logits, reverse, a)
    b, t, d = x.shape
    device = x.device
    h = torch.empty(b, t, d, dtype=x.dtype, device=device)
    if b * t * d == 0:      # no step: the state passes through
        last = torch.zeros(b, d, device=device) if initial_state is None else initial_state.detach().clone()
        return h, last, torch.empty(0, device=device)
    lib = N.lib()
    last = torch.empty(b, d, dtype=torch.float32, device=device)
    a.h, a.last = h.data_ptr(), last.data_ptr()
    kept = None
    if keep:
        kept = torch.empty(lib.pa_gated_recurrence_carries(b, t, d), dtype=torch.float32, device=device)
        a.carries = kept.data_ptr()
    scratch = scratch_of(lib.pa_gated_recurrence_scratch(b, t, d), device)
    a.scratch = N.ptr(scratch)
    N.check(lib.pa_gated_recurrence(byref(a), N.stream_ptr(device)))
    del alive
    return h, last, kept


def gated_recurrence_grad(x: Tensor, gate: Tensor, kept: Tensor, d_h: Optional[Tensor] = None,
                          d_last: Optional[Tensor] = None, resets: Optional[Tensor] = None,
                          lengths: Optional[Tensor] = None, gate_logits: bool = True, reverse: bool = False,
                          ) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients ``(d_x, d_gate, d_initial_state)`` of ``gated_recurrence`` called with ``keep=True`` on the
    same x, gate, resets, lengths and flags, for the gradients of h and of the last state (None: zero)."""
    op = "gated_recurrence_grad"
    if d_h is not None and (d_h.shape != x.shape or d_h.dtype != x.dtype):
        raise ValueError(f"{op}: d_h is {d_h.dtype} {tuple(d_h.shape)}, not {x.dtype} {tuple(x.shape)}")
    if d_last is not None and (d_last.shape != x.shape[:1] + x.shape[-1:] or d_last.dtype != torch.float32):
        raise ValueError(f"{op}: d_last is {d_last.dtype} {tuple(d_last.shape)}, not float32 (batch, channels)")
    a = N.RecurrenceArgs()
    alive = _recurrence_args(op, x, gate, None, resets, lengths, gate_logits, reverse, a)
    b, t, d = x.shape
    device = x.device
    on_one_gpu(op, device, d_h, d_last, kept)
    if d_h is not None:
        d_h = _rows(d_h)
        a.d_h = d_h.data_ptr()
        a.d_h_b, a.d_h_t = _strides(d_h)
    if d_last is not None:
        d_last = d_last.contiguous()
        a.d_last = d_last.data_ptr()
    d_x = torch.empty(b, t, d, dtype=x.dtype, device=device)
    d_gate = torch.empty(b, t, d, dtype=gate.dtype, device=device)
    if b * t * d == 0:
        d_h0 = torch.zeros(b, d, device=device) if d_last is None else d_last.clone()
        return d_x, d_gate, d_h0
    lib = N.lib()
    if kept.dtype != torch.float32 or not kept.is_contiguous() or \
            kept.numel() != lib.pa_gated_recurrence_carries(b, t, d):
        raise ValueError(f"{op}: kept is not what gated_recurrence(..., keep=True) returns for this shape")
    d_h0 = torch.empty(b, d, dtype=torch.float32, device=device)
    scratch = scratch_of(lib.pa_gated_recurrence_scratch(b, t, d), device)
    a.carries, a.scratch = kept.data_ptr(), N.ptr(scratch)
    a.d_x, a.d_gate, a.d_h0 = d_x.data_ptr(), d_gate.data_ptr(), d_h0.data_ptr()
    N.check(lib.pa_gated_recurrence_grad(byref(a), N.stream_ptr(device)))
    del alive
    return d_x, d_gate, d_h0


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, gate: Tensor, initial_state: Optional[Tensor], resets: Optional[Tensor],
                lengths: Optional[Tensor], gate_logits: bool, reverse: bool) -> Tuple[Tensor, Tensor]:
        h, last, kept = _recurrence(x, gate, initial_state, resets, lengths, gate_logits, reverse, True)
        ctx.save_for_backward(x, gate, kept, resets, lengths)
        ctx.flags = bool(gate_logits), bool(reverse)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, d_h: Optional[Tensor], d_last: Optional[Tensor]) -> Tuple:
        x, gate, kept, resets, lengths = ctx.saved_tensors
        if d_h is None and d_last is None:
            return (None,) * 7
        logits, reverse = ctx.flags
        d_x, d_gate, d_h0 = gated_recurrence_grad(x, gate, kept, d_h, d_last, resets, lengths, logits, reverse)
        want_x, want_gate, want_h0 = ctx.needs_input_grad[:3]
        return (d_x if want_x else None, d_gate if want_gate else None, d_h0 if want_h0 else None,
                None, None, None, None)


def gated_recurrence_step(x: Tensor, gate: Tensor, state: Optional[Tensor] = None,
                          resets: Optional[Tensor] = None, gate_logits: bool = True,
                          out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One step of ``gated_recurrence`` for acting: x and gate (batch, channels), state float32 (batch,
    channels) or None for zeros, resets (batch).  Returns ``(h, new_state)``; ``out_state`` receives the new
    state and may be ``state`` itself.  Records no backward pass and refuses inputs that ask for one."""
    op = "gated_recurrence_step"
    if wants_grad(x, gate, state):
        raise RuntimeError(f"{op} records no backward pass: call it under torch.no_grad(), or gated_recurrence")
    if x.dim() != 2 or gate.shape != x.shape:
        raise ValueError(f"{op}: x has shape {tuple(x.shape)} and gate {tuple(gate.shape)}, "
                         "not twice (batch, channels)")
    if resets is not None and resets.shape != x.shape[:1]:
        raise ValueError(f"{op}: resets has shape {tuple(resets.shape)}, not {tuple(x.shape[:1])}")
    a = N.RecurrenceArgs()
    alive = _recurrence_args(op, x.unsqueeze(1), gate.unsqueeze(1), state,
                             None if resets is None else resets.unsqueeze(1), None, gate_logits, False, a)
    b, d = x.shape
    if out_state is None:
        out_state = torch.empty(b, d, dtype=torch.float32, device=x.device)
    else:
        on_one_gpu(op, x.device, out_state)
        if out_state.shape != (b, d) or out_state.dtype != torch.float32 or not out_state.is_contiguous():
            raise ValueError(f"{op}: out_state is not a contiguous float32 tensor of shape {(b, d)}")
    h = torch.empty(b, d, dtype=x.dtype, device=x.device)
    if b * d:
        a.h, a.last = h.data_ptr(), out_state.data_ptr()
        N.check(N.lib().pa_gated_recurrence(byref(a), N.stream_ptr(x.device)))
    del alive
    return h, out_state
