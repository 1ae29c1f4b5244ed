"""Differentiable operators for policies over tokens and histories, each one HIP launch sequence of
libpearl_amd (embed.hip, recurrence.hip):

* ``embed_tokens`` — rows of a table by token: ``OneHotActionTensorRepresentationModule`` followed by a
  dense layer, without the one-hot matrix;
* ``gated_recurrence`` — a gated linear recurrence over a history, with episode starts inside it;
  ``gated_recurrence_step`` is its single step for acting.

Parameters and results are torch tensors in HBM (float32, bfloat16 or float16); work runs on the
current stream of the tensors' device, which need not be the current device.  The functions record
a backward pass when gradients are asked for; ``embed_tokens_grad`` and ``gated_recurrence_grad`` are
the same kernels for learners that run their backward pass explicitly.  None has a forward-mode derivative:
inputs with a tangent are refused."""
from __future__ import annotations

from functools import lru_cache
from typing import Any, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

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


def no_tangents(op: str, *inputs: Optional[Tensor]) -> None:
    """The kernels would drop the tangents of dual tensors without a word."""
    if forward_ad._current_level < 0:       # no dual tensors anywhere: the usual case, at no cost
        return
    for t in inputs:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{op} has no forward-mode derivative")


def dtype_code(op: str, name: str, t: Tensor, table: dict) -> int:
    code = table.get(t.dtype)
    if code is None:
        raise TypeError(f"{op}: {name} is {t.dtype}, not one of "
                        f"{', '.join(str(k).replace('torch.', '') for k in table)}")
    return code


def scratch_of(nbytes: int, device: torch.device) -> Optional[Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _address(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------- embedding
def embed_tokens(weight: Tensor, tokens: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * weight[tokens]``, rounded once: (vocab, dim) and integer tokens of any shape give
    ``tokens.shape + (dim,)`` in the weight's type.

    Token -1 stands for "none": a row of zeros that takes no part in the gradient.  Any other token
    outside the table gives a row of NaN; nothing is read for it.  The weight's gradient is dense,
    summed in float32 in the order of the tokens and the same bits for the same inputs."""
    no_tangents("embed_tokens", weight)
    if weight.requires_grad and torch.is_grad_enabled():
        return _EmbedTokens.apply(weight, tokens, scale)
    return _embed(weight, tokens, scale)


def _embed(weight: Tensor, tokens: Tensor, scale: float) -> Tensor:
    if weight.dim() != 2:
        raise ValueError(f"embed_tokens: weight has {weight.dim()} dimensions, not (vocab, dim)")
    code = dtype_code("embed_tokens", "weight", weight, FLOATS)
    index = dtype_code("embed_tokens", "tokens", tokens, INDICES)
    vocab, dim = weight.shape
    if dim > 2 ** 30:       # before the C entry, which takes 32 bits
        raise NotImplementedError(f"embed_tokens: dim {dim} (up to 2^30)")
    on_one_gpu("embed_tokens", weight.device, tokens)
    if weight.stride(1) != 1 or weight.stride(0) < dim:
        weight = weight.contiguous()
    tokens = tokens.contiguous()
    out = torch.empty(*tokens.shape, dim, dtype=weight.dtype, device=weight.device)
    N.check(N.lib().pa_embed_tokens(weight.data_ptr(), code, max(weight.stride(0), dim), vocab, dim,
                                    tokens.data_ptr(), index, tokens.numel(), scale, out.data_ptr(),
                                    weight.device.index, N.stream_ptr(weight.device)))
    return out


def embed_tokens_grad(d_out: Tensor, tokens: Tensor, vocab: int, scale: float = 1.0) -> Tensor:
    """The gradient of ``embed_tokens`` with respect to its (vocab, dim) weight, in ``d_out``'s type.  Up to 2^26
    tokens, 2^26 rows, 2^25 columns and 2^46 tokens times rows: the time grows with that product (0.06 ms at 2^33, 5.5 at 2^40)."""
    no_tangents("embed_tokens_grad", d_out)
    code = dtype_code("embed_tokens_grad", "d_out", d_out, FLOATS)
    index = dtype_code("embed_tokens_grad", "tokens", tokens, INDICES)
    if d_out.dim() < 1 or d_out.shape[:-1] != tokens.shape:
        raise ValueError(f"embed_tokens_grad: d_out has shape {tuple(d_out.shape)}, the tokens "
                         f"{tuple(tokens.shape)}")
    n, dim = tokens.numel(), d_out.shape[-1]
    if dim > 2 ** 25:
        raise NotImplementedError(f"embed_tokens_grad: dim {dim} (up to 2^25)")
    on_one_gpu("embed_tokens_grad", d_out.device, tokens)
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

    ``gate`` has x's shape and its type, or float32 (decays close to one need it); decays may be above one.
    The state is float32 throughout: ``initial_state`` (batch, channels; zeros if None) and the returned last
    state are float32, h is rounded to x's type.  ``resets`` (batch, time; bool) marks steps that begin an episode
    and ignore the state before them; ``lengths`` (batch) ends histories early: behind the end h is
    zero, whatever x and gate hold there.  ``reverse`` runs from the last step to the first, as advantage
    sums do (a reset there marks the last step of an episode).

    Returns ``(h, last_state)``.  With ``keep=True`` no backward pass is recorded and a third result is
    what ``gated_recurrence_grad`` needs of the forward pass."""
    no_tangents("gated_recurrence", x, gate, initial_state)
    if not keep and torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (
            initial_state is not None and initial_state.requires_grad)):
        return _GatedRecurrence.apply(x, gate, initial_state, resets, lengths, gate_logits, reverse)
    h, last, kept = _recurrence(x, gate, initial_state, resets, lengths, gate_logits, reverse, keep)
    return (h, last, kept) if keep else (h, last)


def _rows(t: Tensor) -> Tensor:
    """(batch, time, channels) with adjacent channels, and steps less than the kernels' 2^23 bytes apart."""
    near = t.stride(1) * t.element_size() < 2 ** 23 or t.shape[1] == 1
    return t if near and (t.stride(2) == 1 or t.shape[2] == 1) else t.contiguous()


def _strides(t: Tensor) -> Tuple[int, int]:
    return t.stride(0), t.stride(1) if t.shape[1] > 1 else 0      # a single step's stride means nothing


@lru_cache(maxsize=4096)
def _recurrence_sizes(b: int, t: int, d: int) -> Tuple[int, int]:
    """Scratch bytes of a call and floats kept for its gradient."""
    lib = N.lib()
    return lib.pa_gated_recurrence_scratch(b, t, d), lib.pa_gated_recurrence_carries(b, t, d)


def _inputs(op: str, x: Tensor, gate: Tensor, resets: Optional[Tensor], lengths: Optional[Tensor]) -> Tuple:
    """Checks what both directions share; returns it as the kernels take it, with the dtypes' codes."""
    if x.dim() != 3 or gate.shape != x.shape:
        raise ValueError(f"{op}: x has shape {tuple(x.shape)} and gate {tuple(gate.shape)}, "
                         "not twice (batch, time, channels)")
    code, gate_code = dtype_code(op, "x", x, FLOATS), dtype_code(op, "gate", gate, FLOATS)
    if gate_code != code and gate_code != N.PA_F32:
        raise TypeError(f"{op}: gate is {gate.dtype}, x is {x.dtype}: the gate has x's type or float32")
    b, t, d = x.shape
    _check_channels(op, d)
    if resets is not None:
        if resets.shape != (b, t) or resets.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"{op}: resets is {resets.dtype} {tuple(resets.shape)}, not bool {(b, t)}")
        if resets.stride(1) >= 2 ** 23:
            resets = resets.contiguous()
    if lengths is not None:
        if lengths.shape != (b,) or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{op}: lengths is {lengths.dtype} {tuple(lengths.shape)}, not int32 or int64 {(b,)}")
        on_one_gpu(op, x.device, lengths)
        # clamped before the cast, so that no length wraps around
        lengths = (lengths.clamp(0, t).to(torch.int32) if lengths.dtype == torch.int64 else lengths).contiguous()
    return code, gate_code, _rows(x), _rows(gate), resets, lengths


def _check_channels(op: str, d: int) -> None:
    if d >= 2 ** 21:        # rows of float32 gates 2^23 bytes long
        raise NotImplementedError(f"{op}: {d} channels (fewer than 2^21)")


def _check_state(op: str, name: str, state: Tensor, shape: Tuple[int, int]) -> Tensor:
    if state.shape != shape or state.dtype != torch.float32:
        raise ValueError(f"{op}: {name} is {state.dtype} {tuple(state.shape)}, not float32 {shape}")
    return state.contiguous()


def _recurrence(x: Tensor, gate: Tensor, initial_state: Optional[Tensor], resets: Optional[Tensor],
                lengths: Optional[Tensor], gate_logits: bool, reverse: bool, keep: bool) -> Tuple:
    op = "gated_recurrence"
    code, gate_code, xs, gs, resets, lengths = _inputs(op, x, gate, resets, lengths)
    b, t, d = x.shape
    if initial_state is not None:
        initial_state = _check_state(op, "initial_state", initial_state, (b, d))
    device = x.device
    on_one_gpu(op, device, gate, initial_state, resets)
    h = torch.empty(b, t, d, dtype=x.dtype, device=device)
    if b * t * d == 0:      # no step: the state passes through
        last = torch.zeros(b, d, device=device) if initial_state is None else initial_state.detach().clone()
        return h, last, torch.empty(0, device=device)
    scratch_bytes, carries = _recurrence_sizes(b, t, d)
    last = torch.empty(b, d, dtype=torch.float32, device=device)
    kept = torch.empty(carries, dtype=torch.float32, device=device) if keep else None
    scratch = scratch_of(scratch_bytes, device)
    args = N.RECURRENCE_ARGS.pack(
        device.index, code, gate_code, bool(gate_logits), bool(reverse), d, b, t,
        xs.data_ptr(), *_strides(xs), gs.data_ptr(), *_strides(gs), _address(initial_state),
        _address(resets), *((0, 0) if resets is None else _strides(resets)), _address(lengths),
        h.data_ptr(), last.data_ptr(), _address(kept), _address(scratch), 0, 0, 0, 0, 0, 0, 0)
    N.check(N.lib().pa_gated_recurrence(args, N.stream_ptr(device)))
    return h, last, kept


def gated_recurrence_grad(x: Tensor, gate: Tensor, kept: Tensor, d_h: Optional[Tensor] = None,
                          d_last: Optional[Tensor] = None, resets: Optional[Tensor] = None,
                          lengths: Optional[Tensor] = None, gate_logits: bool = True, reverse: bool = False,
                          ) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients ``(d_x, d_gate, d_initial_state)`` of ``gated_recurrence`` called with ``keep=True`` on the
    same x, gate, resets, lengths and flags, for the gradients of h and of the last state (None: zero)."""
    op = "gated_recurrence_grad"
    no_tangents(op, x, gate, d_h, d_last)
    code, gate_code, xs, gs, resets, lengths = _inputs(op, x, gate, resets, lengths)
    b, t, d = x.shape
    if d_h is not None:
        if d_h.shape != x.shape or d_h.dtype != x.dtype:
            raise ValueError(f"{op}: d_h is {d_h.dtype} {tuple(d_h.shape)}, not {x.dtype} {tuple(x.shape)}")
        d_h = _rows(d_h)
    if d_last is not None:
        d_last = _check_state(op, "d_last", d_last, (b, d))
    device = x.device
    on_one_gpu(op, device, gate, resets, d_h, d_last, kept)
    d_x = torch.empty(b, t, d, dtype=x.dtype, device=device)
    d_gate = torch.empty(b, t, d, dtype=gate.dtype, device=device)
    if b * t * d == 0:
        d_h0 = torch.zeros(b, d, device=device) if d_last is None else d_last.clone()
        return d_x, d_gate, d_h0
    scratch_bytes, carries = _recurrence_sizes(b, t, d)
    if kept.dtype != torch.float32 or not kept.is_contiguous() or kept.numel() != carries:
        raise ValueError(f"{op}: kept is not what gated_recurrence(..., keep=True) returns for this shape")
    d_h0 = torch.empty(b, d, dtype=torch.float32, device=device)
    scratch = scratch_of(scratch_bytes, device)
    args = N.RECURRENCE_ARGS.pack(
        device.index, code, gate_code, bool(gate_logits), bool(reverse), d, b, t,
        xs.data_ptr(), *_strides(xs), gs.data_ptr(), *_strides(gs), 0,
        _address(resets), *((0, 0) if resets is None else _strides(resets)), _address(lengths),
        0, 0, kept.data_ptr(), _address(scratch), _address(d_h), *((0, 0) if d_h is None else _strides(d_h)),
        _address(d_last), d_x.data_ptr(), d_gate.data_ptr(), d_h0.data_ptr())
    N.check(N.lib().pa_gated_recurrence_grad(args, N.stream_ptr(device)))
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
    state and may be ``state`` itself; one that overlaps an input in another way is refused.  Records no backward pass and refuses inputs that ask for one."""
    op = "gated_recurrence_step"
    no_tangents(op, x, gate, state)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (
            state is not None and state.requires_grad) or (out_state is not None and out_state.requires_grad)):
        raise RuntimeError(f"{op} records no backward pass: call it under torch.no_grad(), or gated_recurrence")
    shape = x.shape
    if len(shape) != 2 or gate.shape != shape:
        raise ValueError(f"{op}: x has shape {tuple(x.shape)} and gate {tuple(gate.shape)}, "
                         "not twice (batch, channels)")
    code, gate_code = dtype_code(op, "x", x, FLOATS), dtype_code(op, "gate", gate, FLOATS)
    if gate_code != code and gate_code != N.PA_F32:
        raise TypeError(f"{op}: gate is {gate.dtype}, x is {x.dtype}: the gate has x's type or float32")
    b, d = shape
    _check_channels(op, d)
    if state is not None:
        state = _check_state(op, "state", state, shape)
    if resets is not None and (resets.shape != shape[:1] or resets.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"{op}: resets is {resets.dtype} {tuple(resets.shape)}, not bool {(b,)}")
    if out_state is not None and (out_state.shape != shape or out_state.dtype != torch.float32
                                  or not out_state.is_contiguous()):
        raise ValueError(f"{op}: out_state is not a contiguous float32 tensor of shape {(b, d)}")
    device = x.device
    on_one_gpu(op, device, gate, state, resets, out_state)
    if x.stride(1) != 1 and d > 1:
        x = x.contiguous()
    if gate.stride(1) != 1 and d > 1:
        gate = gate.contiguous()
    h = torch.empty(b, d, dtype=x.dtype, device=device)
    if out_state is None:
        out_state = torch.empty(b, d, dtype=torch.float32, device=device)
    elif not out_state.is_inference():      # such tensors have no versions
        increment_version(out_state)        # or a backward pass that kept the old state would read the new one
    if b * d:
        args = N.RECURRENCE_ARGS.pack(
            device.index, code, gate_code, bool(gate_logits), False, d, b, 1,
            x.data_ptr(), x.stride(0), 0, gate.data_ptr(), gate.stride(0), 0, _address(state),
            _address(resets), 0 if resets is None else resets.stride(0), 0, 0,
            h.data_ptr(), out_state.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0)
        N.check(N.lib().pa_gated_recurrence(args, N.stream_ptr(device)))
    return h, out_state
