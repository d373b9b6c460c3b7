"""``KeyValueCache`` and ``cached_attention``: keys and values kept in pages from one call to the next, and the attention of
new tokens over them.

The reference keeps nothing between calls.  A page holds 32, 64, 128 or 256 tokens of every key head, head after head, in
16 bits or quantised to int8 or e4m3 with one scale per token and head.  Which pages belong to a sequence, and how many
tokens it has, is the caller's: a page table and lengths, both int32 tensors on the GPU, so that a step can be captured into a graph
and replayed while sequences grow.
"""
from typing import Optional, Tuple

import torch

from . import kernel as _k
from .packed import HEAD_DIMS, MOST_ROWS, check_heads, check_index, forward_mode, rows_of, strides_of

PAGES = (32, 64, 128, 256)
MOST_DRAFTS = 1024
_ROWS = {torch.float32: _k.BSA_F32, torch.float16: _k.BSA_F16, torch.bfloat16: _k.BSA_BF16}
_QUANTISED = {torch.int8: _k.BSA_I8, torch.float8_e4m3fn: _k.BSA_E4M3}
_HELD = {torch.float16: _k.BSA_F16, torch.bfloat16: _k.BSA_BF16, **_QUANTISED}


def refuse_gradients(what: str, *operands: torch.Tensor) -> None:
    """A result without history would cut a loss off from them without a word."""
    if (torch.is_grad_enabled() and any(t.requires_grad for t in operands)) or any(forward_mode(t) for t in operands):
        raise RuntimeError(f"{what} is not differentiable: call it under torch.no_grad() or detach its operands")


class KeyValueCache:
    """``pages`` pages of ``page`` tokens for ``heads`` key heads: ``keys``, ``values`` ``[pages, heads, page, head_dim]`` of
    ``dtype`` (int8, float8_e4m3fn, float16 or bfloat16) and, for the 8-bit types, ``key_scales``, ``value_scales``
    ``[pages, heads, page]`` in float32 (else ``None``).  A token's place is its slot, ``page number * page + place``.  The
    tensors may be written to, not replaced."""

    def __init__(self, pages: int, heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn, page: int = 64, device=None):
        if dtype not in _HELD:
            raise TypeError(f"a cache holds int8, float8_e4m3fn, float16 or bfloat16, got {dtype}")
        if page not in PAGES:
            raise ValueError(f"page must be 32, 64, 128 or 256 tokens, got {page}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head dim must be 64 or 128, got {head_dim}")
        if not (1 <= heads <= 65535 and pages >= 1 and pages * page < 2 ** 31):
            raise ValueError(f"a cache of {pages} pages of {page} tokens for {heads} heads cannot be addressed")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("a cache lives on the GPU")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.heads, self.head_dim, self.dtype, self.page, self.device = pages, heads, head_dim, dtype, page, device
        shape = (pages, heads, page)
        held = [torch.empty(shape + (head_dim,), dtype=dtype, device=device) for _ in range(2)]
        held += [torch.empty(shape, dtype=torch.float32, device=device) if dtype in _QUANTISED else None for _ in range(2)]
        self._held, self._native = tuple(held), _k.host_calls.new_cache(*held)

    keys = property(lambda self: self._held[0])
    values = property(lambda self: self._held[1])
    key_scales = property(lambda self: self._held[2])
    value_scales = property(lambda self: self._held[3])

    def __getstate__(self):
        state = {name: value for name, value in self.__dict__.items() if name != "_native"}
        # as bytes: pickle has no float8 storage
        state["_held"] = tuple(t.view(torch.uint8) for t in self._held[:2]) + self._held[2:]
        return state

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._held = tuple(t.view(self.dtype) for t in self._held[:2]) + self._held[2:]
        self.device = self.keys.device
        if self.device.type != "cuda":              # loaded elsewhere: its calls would hand host addresses to kernels
            raise ValueError("a cache lives on the GPU")
        self._native = _k.host_calls.new_cache(*self._held)

    def _tensors(self):
        scales = (self.key_scales, self.value_scales)
        return (self.keys.data_ptr(), self.values.data_ptr(), *(None if t is None else t.data_ptr() for t in scales))

    def _sizes(self, tokens):
        return tokens, self.heads, self.head_dim, self.pages, self.page

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Stores ``k``, ``v`` ``[tokens, heads, head_dim]`` at ``slots`` (int32 on the GPU, ``[tokens]``), quantised if the cache is:
        the scale is the row's largest magnitude over 127 or 448, values are rounded to the nearest, ties to even.  Rows
        with a negative slot (refused drafts, padding) or one behind the cache are left out; no two rows of a call may have the same
        slot.  A row with an infinity or a NaN is kept as NaN.  Not differentiable: operands that
        autograd follows are refused."""
        if _k.host_calls.cache_write(self._native, k, v, slots):
            return
        for t, name in ((k, "k"), (v, "v")):
            if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != k.dtype:
                raise TypeError(f"k and v must both be float16 or both bfloat16, got {name}: {t.dtype}")
            if t.dim() != 3 or t.size(1) != self.heads or t.size(2) != self.head_dim or t.size(0) != k.size(0):
                raise ValueError(f"{name} must be [tokens, {self.heads}, {self.head_dim}], got {tuple(t.shape)}")
            if t.device != self.device:
                raise ValueError(f"{name} must live on the cache's GPU")
        if self.dtype not in _QUANTISED and k.dtype != self.dtype:
            raise TypeError(f"a cache of {self.dtype} takes rows of that type, got {k.dtype}")
        refuse_gradients("KeyValueCache.write", k, v)
        check_index(slots, "slots", self.device, 1)
        if slots.numel() != k.size(0) or k.size(0) > MOST_ROWS:
            raise ValueError(f"{k.size(0)} rows and {slots.numel()} slots")
        k, v = rows_of(k.detach()), rows_of(v.detach())
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_cache_write(_ROWS[k.dtype], _HELD[self.dtype], k.data_ptr(), v.data_ptr(), slots.data_ptr(),
                                            *self._tensors(), *self._sizes(k.size(0)), strides_of(k, v), _k.current_stream()))

    def read(self, slots: torch.Tensor, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values at ``slots``, ``[tokens, heads, head_dim]`` each, in float32, float16 or bfloat16; zeros for a slot that is
        negative or behind the cache."""
        rows = _k.host_calls.cache_read(self._native, slots, dtype)
        if rows is not None:
            return rows
        if dtype not in _ROWS:
            raise TypeError(f"rows are read as float32, float16 or bfloat16, got {dtype}")
        check_index(slots, "slots", self.device, 1)
        if slots.numel() > MOST_ROWS:
            raise ValueError(f"{slots.numel()} slots are too many")
        shape = (slots.numel(), self.heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_cache_read(_ROWS[dtype], _HELD[self.dtype], *self._tensors(), slots.data_ptr(), k.data_ptr(),
                                           v.data_ptr(), *self._sizes(slots.numel()), _k.current_stream()))
        return k, v

    def copy(self, sources: torch.Tensor, targets: torch.Tensor, origin: Optional["KeyValueCache"] = None) -> None:
        """Copies whole pages as they are, values and scales: page ``sources[i]`` of ``origin`` (this cache without one) to page
        ``targets[i]`` of this one (int32 on the GPU).  ``origin`` has the same type, heads, head dim and page on the same GPU, and any number of
        pages.  Pairs with a number outside either cache (-1) are left out.  No page may be the target of two pairs, nor, in one cache, the
        target of one and the source of another."""
        origin = self if origin is None else origin
        if not isinstance(origin, KeyValueCache):
            raise TypeError(f"origin must be a KeyValueCache, got {type(origin).__name__}")
        if _k.host_calls.cache_copy(self._native, origin._native, sources, targets):
            return
        for name in ("dtype", "heads", "head_dim", "page", "device"):
            if getattr(origin, name) != getattr(self, name):
                raise ValueError(f"pages of a cache with {name} {getattr(origin, name)} do not fit one with {getattr(self, name)}")
        check_index(sources, "sources", self.device, 1)
        check_index(targets, "targets", self.device, 1)
        if sources.numel() != targets.numel() or sources.numel() > 1 << 24:
            raise ValueError(f"{sources.numel()} sources and {targets.numel()} targets")
        if sources.numel() == 0:
            return
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_cache_copy(_HELD[self.dtype], *origin._tensors(), origin.pages, *self._tensors(), self.pages, sources.data_ptr(),
                                           targets.data_ptr(), sources.numel(), self.heads, self.head_dim, self.page, _k.current_stream()))


def cached_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KeyValueCache, pages: torch.Tensor,
                     lengths: torch.Tensor, tree: Optional[torch.Tensor] = None, scale: float = 1.0) -> torch.Tensor:
    """Attention of ``n`` new tokens of every sequence over what ``cache`` holds of it and over one another.

    ``q [batch, n, heads, D]`` and the new tokens' own ``k``, ``v [batch, n, key heads, D]`` (not yet in the cache; those that are
    kept go there by ``cache.write``).  ``pages [batch, width]`` lists the page numbers of every sequence, ``lengths [batch]`` says how
    many tokens it has in them, both int32 on the GPU.  ``tree``, bool ``[n, n]`` or ``[batch, n, n]``: whether new token ``i`` sees new
    token ``j`` (itself too, where it should); without it they are a chain, ``j <= i``.  ``n = 1`` is a decode step.  Every new token sees
    the whole cached part of its sequence; one that sees nothing gets zeros.  At most 1024 new tokens a sequence.  Not
    differentiable: operands that autograd follows are refused."""
    if not isinstance(cache, KeyValueCache):
        raise TypeError(f"cache must be a KeyValueCache, got {type(cache).__name__}")
    out = _k.host_calls.cached_attention(q, k, v, cache._native, pages, lengths, tree, scale)
    if out is not None:
        return out
    check_heads(q, k, v, 4)
    refuse_gradients("cached_attention", q, k, v)
    batch, drafts, heads, dim = q.shape
    if (cache.heads, cache.head_dim) != (k.size(2), dim) or cache.device != q.device:
        raise ValueError(f"k {tuple(k.shape)} on {k.device} does not fit a cache of {cache.heads} heads of {cache.head_dim} on {cache.device}")
    if cache.dtype not in _QUANTISED and q.dtype != cache.dtype:
        raise TypeError(f"a cache of {cache.dtype} is attended to in that type, got {q.dtype}")
    check_index(pages, "pages", q.device, 2)
    check_index(lengths, "lengths", q.device, 1)
    if pages.size(0) != batch or lengths.numel() != batch or pages.numel() > MOST_ROWS:
        raise ValueError(f"{batch} sequences, pages {tuple(pages.shape)} and lengths {tuple(lengths.shape)}")
    if drafts > MOST_DRAFTS:
        raise ValueError(f"at most {MOST_DRAFTS} new tokens a sequence, got {drafts}")
    if tree is not None:
        if not isinstance(tree, torch.Tensor) or tree.dtype != torch.bool or tree.device != q.device or tuple(tree.shape) not in ((drafts, drafts), (batch, drafts, drafts)):
            raise ValueError(f"tree must be bool [{drafts}, {drafts}] or [{batch}, {drafts}, {drafts}] on the GPU of the operands")
        tree = tree.contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    q, k, v = rows_of(q.detach()), rows_of(k.detach()), rows_of(v.detach())
    sizes = (batch, drafts, heads, k.size(2), dim)
    need = _k.lib.bsa_cached_attention_workspace_bytes(*sizes, pages.size(1), cache.page)
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    with _k.on_device(q.device):
        _k.check(_k.lib.bsa_cached_attention(
            _ROWS[q.dtype], _HELD[cache.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *cache._tensors(),
            pages.data_ptr(), lengths.data_ptr(), None if tree is None else tree.data_ptr(), int(tree is not None and tree.dim() == 2),
            *sizes, cache.pages, cache.page, pages.size(1), strides_of(q, k, v), float(scale),
            workspace.data_ptr() if need else None, need, _k.current_stream()))
    return out
