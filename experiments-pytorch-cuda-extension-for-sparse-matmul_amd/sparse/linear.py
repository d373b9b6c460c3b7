"""``packed_linear_attention`` and ``linear_attention_step``: linear attention with a decay for each key head.

The reference has no such call.  A sequence's past is one ``D x D`` matrix a key head, in float32, whatever its length:

    S_t = exp(log_decay) S_(t-1) + k_t v_t^T,      o_t = scale q_t S_t

Prompts and training batches are packed along the tokens as ``packed_attention`` takes them and are walked in chunks; a
decode step updates the matrices in place.  Offsets and slots stay on the device, so no call waits for it.
"""
from typing import Any, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import kernel as _k
from .cache import refuse_gradients
from .packed import _DTYPES, MOST_ROWS, check_heads, check_index, forward_mode, rows_of, strides_of

MOST_SEQUENCES = 65535


def _pointer(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def check_decay(log_decay: Any, key_heads: int, device: torch.device) -> None:
    if not (isinstance(log_decay, torch.Tensor) and log_decay.dtype == torch.float32 and tuple(log_decay.shape) == (key_heads,)
            and log_decay.is_contiguous()):
        raise ValueError(f"log_decay must be a contiguous float32 tensor [{key_heads}], one value a key head")
    if log_decay.device != device:
        raise ValueError("log_decay must live on the GPU of the operands")
    refuse_gradients("log_decay", log_decay)


def check_states(states: Any, shape: Tuple[int, ...], device: torch.device, what: str = "states") -> None:
    if not (isinstance(states, torch.Tensor) and states.dtype == torch.float32 and tuple(states.shape) == shape):
        got = f"{states.dtype} {tuple(states.shape)}" if isinstance(states, torch.Tensor) else type(states).__name__
        raise ValueError(f"{what} must be float32 {list(shape)}, got {got}")
    if states.device != device:
        raise ValueError(f"{what} must live on the GPU of the operands")


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and at a multiple of 16 bytes, as states are read."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, log_decay, offsets, states):
    check_heads(q, k, v, 3)
    check_index(offsets, "offsets", q.device, 1)
    if offsets.numel() < 1:
        raise ValueError("offsets needs one entry more than there are sequences")
    check_decay(log_decay, k.size(1), q.device)
    if q.size(0) > MOST_ROWS or offsets.numel() - 1 > MOST_SEQUENCES:
        raise ValueError(f"{q.size(0)} tokens in {offsets.numel() - 1} sequences are too many")
    if states is not None:
        check_states(states, state_shape(k, offsets), q.device)


def state_shape(k: torch.Tensor, offsets: torch.Tensor) -> Tuple[int, ...]:
    return (offsets.numel() - 1, k.size(1), k.size(2), k.size(2))


def _between(k: torch.Tensor, tokens: int, segment: int) -> Tuple[torch.Tensor, int]:
    """Room for the states between the segments of long sequences."""
    need = _k.lib.bsa_linear_attention_states_bytes(tokens, k.size(1), k.size(2), segment)
    return torch.empty(need // 4, dtype=torch.float32, device=k.device), need


def run_forward(q, k, v, log_decay, offsets, scale, states, return_states):
    """Result, final states (or None), what the backward pass needs besides."""
    _check(q, k, v, log_decay, offsets, states)
    tokens, heads, dim = q.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    last = torch.empty(state_shape(k, offsets), dtype=torch.float32, device=q.device) if return_states else None
    if tokens == 0 or offsets.numel() == 1:
        if last is not None:
            last.zero_() if states is None else last.copy_(states)
        return out.zero_(), last, torch.empty(0, dtype=torch.float32, device=q.device)
    q, k, v, states = rows_of(q), rows_of(k), rows_of(v), _dense(states)
    segment = _k.lib.bsa_linear_attention_segment(tokens, offsets.numel() - 1, k.size(1), dim)
    between, need = _between(k, tokens, segment)
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_linear_attention_forward(
            _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), log_decay.data_ptr(), offsets.data_ptr(),
            _pointer(states), _pointer(last), between.data_ptr() if need else None, need, segment, tokens, offsets.numel() - 1, heads,
            k.size(1), dim, strides_of(q, k, v), float(scale), _k.current_stream()))
    return out, last, between


def run_backward(q, k, v, states, log_decay, offsets, between, dout, dlast, scale, with_states):
    """Gradients of q, k, v and, ``with_states``, of the first states.  What autograd kept may come back as hooks made it."""
    _check(q, k, v, log_decay, offsets, states)
    tokens, heads, dim = q.shape
    if dout is None:
        dout = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if dout.shape != q.shape or dout.dtype != q.dtype or dout.device != q.device:
        raise ValueError(f"the gradient of {q.dtype} {tuple(q.shape)} on {q.device} came back as {dout.dtype} {tuple(dout.shape)} on {dout.device}")
    if dlast is not None:
        check_states(dlast, state_shape(k, offsets), q.device, "the gradient of the states")
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty(k.shape, dtype=k.dtype, device=k.device) for _ in range(2))
    dfirst = torch.empty(state_shape(k, offsets), dtype=torch.float32, device=q.device) if with_states else None
    if tokens == 0 or offsets.numel() == 1:
        if dfirst is not None:
            dfirst.zero_() if dlast is None else dfirst.copy_(dlast)
        return dq.zero_(), dk.zero_(), dv.zero_(), dfirst
    segment = _k.lib.bsa_linear_attention_segment(tokens, offsets.numel() - 1, k.size(1), dim)
    behind, need = _between(k, tokens, segment)
    if between.dtype != torch.float32 or between.numel() != behind.numel() or between.device != q.device or not between.is_contiguous():
        raise ValueError("the saved states came back as others")
    q, k, v, dout = rows_of(q), rows_of(k), rows_of(v), rows_of(dout)
    states, dlast = _dense(states), _dense(dlast)
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_linear_attention_backward(
            _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), log_decay.data_ptr(), offsets.data_ptr(),
            _pointer(states), between.data_ptr() if need else None, _pointer(dlast), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            _pointer(dfirst), behind.data_ptr() if need else None, need, segment, tokens, offsets.numel() - 1, heads, k.size(1), dim,
            strides_of(q, k, v, dout), float(scale), _k.current_stream()))
    return dq, dk, dv, dfirst


class PackedLinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q, k, v, states, log_decay, offsets, scale, return_states):
        out, last, between = run_forward(q, k, v, log_decay, offsets, scale, states, return_states)
        ctx.save_for_backward(q, k, v, states, log_decay, offsets, between)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_states else out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dout: Optional[torch.Tensor], dlast: Optional[torch.Tensor] = None):
        q, k, v, states, log_decay, offsets, between = ctx.saved_tensors
        dq, dk, dv, dfirst = run_backward(q, k, v, states, log_decay, offsets, between, dout, dlast, ctx.scale,
                                          states is not None and ctx.needs_input_grad[3])
        return dq, dk, dv, dfirst, None, None, None, None


def packed_linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, offsets: torch.Tensor,
                            scale: float = 1.0, states: Optional[torch.Tensor] = None,
                            return_states: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Linear attention inside every sequence of a packed batch: ``S_t = exp(log_decay) S_(t-1) + k_t v_t^T``, ``o_t = scale q_t S_t``.

    ``q [tokens, heads, D]``, ``k``, ``v [tokens, key heads, D]``, float16 or bfloat16, ``D`` 64 or 128; query head ``h`` reads key head
    ``h // (heads // key heads)``.  ``log_decay``, float32 ``[key heads]``, 0 or less: logarithm of what a state keeps from token to
    token (``-inf``: nothing).  ``offsets``, int32 on the GPU: sequence ``b`` is the tokens ``offsets[b]`` to ``offsets[b + 1] - 1``;
    ascending, empty sequences allowed.  ``states``, float32 ``[sequences, key heads, D, D]``: what each sequence begins with, zero
    without; with ``return_states`` the call gives ``(o, final states)``, an empty sequence's being those it began with.  Tokens
    outside every sequence (the padding of a batch) are not read; their results and gradients are zero.  Operands may be slices of a
    larger tensor; they are copied only where a row does not start at a multiple of 16 bytes.  Differentiable once in ``q``, ``k``, ``v``
    and ``states``, with the same bits in every call (in bfloat16 ``return_states`` changes ``o`` within its rounding); ``log_decay`` has no
    gradient and is refused if autograd follows it."""
    found = _k.host_calls.linear_attention(q, k, v, log_decay, offsets, scale, states, return_states)
    if found is not None:
        return found
    return general(q, k, v, log_decay, offsets, scale, states, return_states)


def general(q, k, v, log_decay, offsets, scale, states, return_states):
    """The call without the native side, which leaves to it whatever it does not take."""
    leaves = [t for t in (q, k, v, states) if isinstance(t, torch.Tensor)]
    if (torch.is_grad_enabled() and any(t.requires_grad for t in leaves)) or any(forward_mode(t) for t in leaves):
        return PackedLinearAttention.apply(q, k, v, states, log_decay, offsets, scale, bool(return_states))
    out, last, _ = run_forward(q, k, v, log_decay, offsets, scale, states, return_states)
    return (out, last) if return_states else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, states: torch.Tensor,
                          slots: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """One token of every sequence: ``states[slots[b]]`` takes it in, in place, and its result is returned.

    ``q [batch, heads, D]``, ``k``, ``v [batch, key heads, D]``, ``log_decay [key heads]`` as for ``packed_linear_attention``, whose final
    states go on here.  ``states``, float32 ``[places, key heads, D, D]``, contiguous; ``slots``, int32 on the GPU, ``[batch]``: the place of
    each sequence.  A sequence whose slot is negative or behind the states (an idle row of the batch) gets zeros and changes nothing;
    no two rows of a call may have the same slot.  Not differentiable: operands that autograd follows are refused."""
    out = _k.host_calls.linear_step(q, k, v, log_decay, states, slots, scale)
    if out is not None:
        return out
    check_heads(q, k, v, 3)
    refuse_gradients("linear_attention_step", q, k, v, *([states] if isinstance(states, torch.Tensor) else []))
    check_decay(log_decay, k.size(1), q.device)
    batch, heads, dim = q.shape
    check_states(states, (states.size(0) if isinstance(states, torch.Tensor) and states.dim() else 0, k.size(1), dim, dim), q.device)
    if not states.is_contiguous() or states.data_ptr() % 16:
        raise ValueError("states are updated in place: they must be contiguous and start at a multiple of 16 bytes")
    check_index(slots, "slots", q.device, 1)
    if slots.numel() != batch or batch > MOST_SEQUENCES:
        raise ValueError(f"{batch} sequences and {slots.numel()} slots")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    q, k, v = rows_of(q.detach()), rows_of(k.detach()), rows_of(v.detach())
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_linear_attention_step(
            _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), log_decay.data_ptr(), states.data_ptr() or None,
            slots.data_ptr(), batch, states.size(0), heads, k.size(1), dim, strides_of(q, k, v), float(scale), _k.current_stream()))
    if not states.is_inference():
        torch.autograd.graph.increment_version(states)       # a graph that kept them is told that they changed
    return out
