"""``packed_attention``: attention over sequences of different lengths packed along the tokens, with autograd.

The reference has no such call: its operators take rectangular batches.  The forward is one launch; the backward is two
that rebuild the probabilities from the saved row statistics, one walking the queries (dq), one the keys (dk, dv, summed
over the query heads that share a key head).  Offsets stay on the device, so no call waits for it.
"""
import ctypes
from typing import Any, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import kernel as _k

_DTYPES = {torch.float16: _k.BSA_F16, torch.bfloat16: _k.BSA_BF16}
HEAD_DIMS = (64, 128)
MOST_ROWS = 1 << 30                             # of a call


def rows_of(t: torch.Tensor, copy: bool = False) -> torch.Tensor:
    """``t`` as the kernels can read it in place: rows of contiguous values, every row at a multiple of 16 bytes."""
    if t.stride(-1) != 1 or t.data_ptr() & 15 or any((s & 7 or s > 1 << 24) and n > 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
        copy = True
    return t.clone(memory_format=torch.contiguous_format) if copy else t


def strides_of(*operands: torch.Tensor):
    """Strides of all but the last dimension, one operand after the other; of a dimension of one element 0."""
    values = [s if n > 1 else 0 for t in operands for s, n in zip(t.stride()[:-1], t.shape[:-1])]
    return (ctypes.c_int64 * len(values))(*values)


def check_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dims: int) -> None:
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise TypeError(f"q, k, v must all be float16 or all bfloat16, got {name}: {t.dtype}")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if not t.is_cuda or t.device != q.device:
            raise ValueError("q, k, v must live on the same GPU")
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if q.size(-1) not in HEAD_DIMS:
        raise ValueError(f"head dim must be 64 or 128, got {q.size(-1)}")
    if k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.size(-1) != k.size(-1):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if k.size(-2) < 1 or q.size(-2) < 1 or q.size(-2) % k.size(-2):
        raise ValueError(f"{q.size(-2)} query heads cannot share {k.size(-2)} key heads evenly")


def check_index(t: Any, name: str, device: torch.device, dims: int) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == dims and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dims}-D int32 tensor")
    if t.device != device:
        raise ValueError(f"{name} must live on the GPU of the operands")


def _forward(q, k, v, offsets, scale, causal, for_backward):
    check_heads(q, k, v, 3)
    check_index(offsets, "offsets", q.device, 1)
    if offsets.numel() < 1:
        raise ValueError("offsets needs one entry more than there are sequences")
    tokens, heads, dim = q.shape
    if tokens > MOST_ROWS or offsets.numel() > 1 << 24:
        raise ValueError(f"{tokens} tokens in {offsets.numel() - 1} sequences are too many")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rest = torch.empty_like(out) if for_backward else None
    lse = torch.empty((heads, tokens), dtype=torch.float32, device=q.device) if for_backward else None
    if tokens == 0:
        return out, rest, lse
    if offsets.numel() == 1:                    # no sequence: no token is in one
        return out.zero_(), rest, lse
    q, k, v = rows_of(q), rows_of(k), rows_of(v)
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_packed_attention_forward(
            _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            rest.data_ptr() if for_backward else None, lse.data_ptr() if for_backward else None, offsets.data_ptr(), tokens,
            offsets.numel() - 1, heads, k.size(1), dim, strides_of(q, k, v), float(scale), int(bool(causal)), _k.current_stream()))
    return out, rest, lse


def _check_saved(q, k, v, dout, out, rest, lse, offsets):
    """What autograd kept may come back as hooks on saved tensors made it."""
    check_heads(q, k, v, 3)
    for t, name, shape, dtype in ((dout, "gradient", q.shape, q.dtype), (out, "saved result", q.shape, q.dtype), (rest, "saved rest", q.shape, q.dtype),
                                  (lse, "saved statistics", (q.size(1), q.size(0)), torch.float32)):
        if t.shape != torch.Size(shape) or t.dtype != dtype or t.device != q.device:
            raise ValueError(f"the {name} of {q.dtype} {tuple(q.shape)} on {q.device} came back as {t.dtype} {tuple(t.shape)} on {t.device}")
    check_index(offsets, "offsets", q.device, 1)
    if offsets.numel() < 1:
        raise ValueError("offsets needs one entry more than there are sequences")


def run_backward(q, k, v, dout, out, rest, lse, offsets, scale, causal, with_dkdv):
    _check_saved(q, k, v, dout, out, rest, lse, offsets)
    tokens, heads, dim = q.shape
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty(k.shape, dtype=k.dtype, device=k.device) for _ in range(2)) if with_dkdv else (None, None)
    if tokens == 0 or offsets.numel() == 1:
        return tuple(t if t is None else t.zero_() for t in (dq, dk, dv))
    q, k, v, dout = rows_of(q), rows_of(k), rows_of(v), rows_of(dout)
    out, rest = (rows_of(t, copy=not t.is_contiguous()) for t in (out, rest))
    lse = lse.contiguous()
    delta = torch.empty_like(lse)
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_packed_attention_backward(
            _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), out.data_ptr(), rest.data_ptr(), lse.data_ptr(),
            delta.data_ptr(), dq.data_ptr(), dk.data_ptr() if with_dkdv else None, dv.data_ptr() if with_dkdv else None,
            offsets.data_ptr(), tokens, offsets.numel() - 1, heads, k.size(1), dim, strides_of(q, k, v, dout), float(scale),
            int(bool(causal)), _k.current_stream()))
    return dq, dk, dv


class PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, scale: float,
                causal: bool) -> torch.Tensor:
        out, rest, lse = _forward(q, k, v, offsets, scale, causal, True)
        ctx.save_for_backward(q, k, v, out, rest, lse, offsets)
        ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dout: torch.Tensor) -> Tuple[Optional[torch.Tensor], ...]:
        q, k, v, out, rest, lse, offsets = ctx.saved_tensors
        grads = run_backward(q, k, v, dout, out, rest, lse, offsets, ctx.scale, ctx.causal, any(ctx.needs_input_grad[1:3]))
        return grads + (None, None, None)


def forward_mode(t):
    return torch.autograd.forward_ad.unpack_dual(t).tangent is not None


def general(q, k, v, offsets, scale, causal):
    """The call without the native side, which hands over whatever it does not take."""
    tracked = torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v))
    if tracked or any(isinstance(t, torch.Tensor) and forward_mode(t) for t in (q, k, v)):
        return PackedAttention.apply(q, k, v, offsets, scale, causal)
    return _forward(q, k, v, offsets, scale, causal, False)[0]


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, scale: float = 1.0,
                     causal: bool = True) -> torch.Tensor:
    """``softmax(scale * q @ k^T) @ v`` inside every sequence of a packed batch.

    ``q [tokens, heads, D]``, ``k``, ``v [tokens, key heads, D]``, float16 or bfloat16, ``D`` 64 or 128; query head ``h`` reads key
    head ``h // (heads // key heads)``.  ``offsets``, int32 on the GPU: sequence ``b`` is the tokens ``offsets[b]`` to
    ``offsets[b + 1] - 1``; ascending, empty sequences allowed.  With ``causal`` a token sees its sequence up to itself.
    Tokens outside every sequence (the padding of a batch) are not read; their results and gradients are zero.  Operands may be
    slices of a larger tensor (a fused projection); they are copied only where a row does not start at a multiple of 16 bytes.
    Differentiable once in ``q``, ``k`` and ``v``, with the same bits in every call."""
    return _k.host_calls.packed_attention(q, k, v, offsets, scale, causal)
