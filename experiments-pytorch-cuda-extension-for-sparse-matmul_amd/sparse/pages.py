"""``PageTable``: which pages of a cache each sequence has, kept on the GPU.

The reference keeps nothing between calls.  The table, the lengths and the count of each page's users are int32 tensors that
``cached_attention`` takes as they are; sequences grow, are continued by others, end and move together without the host
knowing their lengths, so that these calls can be captured into a graph with the attention they serve.  One table serves all layers of a
model: every layer has a ``KeyValueCache`` of its own with the same pages.
"""
import operator
from typing import Tuple

import torch

from . import kernel as _k
from .cache import PAGES
from .packed import MOST_ROWS, check_index

MOST_SEQUENCES = 4096


class PageTable:
    """Pages of ``page`` tokens, ``pages`` of them, for up to ``sequences`` sequences of at most ``width`` pages: ``table [sequences, width]``
    (-1 behind the last page of each), ``lengths [sequences]`` in tokens, ``uses [pages]``: how many sequences have a page, and
    ``missing [1]``: how many requests for pages could not be met so far.  A whole page may belong to several sequences, a last page
    that is not full belongs to one.  The lowest free pages are taken first.  The tensors may be written to, not replaced (whoever lowers a
    length by whole pages frees them too, in ``uses`` and in the row); the calls for a table are to be ordered, on one stream or by
    events."""

    def __init__(self, pages: int, page: int, sequences: int, width: int, device=None):
        if page not in PAGES:
            raise ValueError(f"page must be 32, 64, 128 or 256 tokens, got {page}")
        if not (pages >= 1 and pages * page < 2 ** 31):
            raise ValueError(f"{pages} pages of {page} tokens cannot be addressed")
        if not (1 <= sequences <= MOST_SEQUENCES and width >= 1 and width * page <= 2 ** 30 and sequences * width < 2 ** 31):
            raise ValueError(f"a table of {sequences} sequences (at most {MOST_SEQUENCES}) of {width} pages of {page} tokens is too large")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("a table lives on the GPU")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.page, self.sequences, self.width, self.device = pages, page, sequences, width, device
        self._tensors = (torch.full((sequences, width), -1, dtype=torch.int32, device=device),
                         *(torch.zeros(n, dtype=torch.int32, device=device) for n in (sequences, pages, 1)))
        self._native = _k.host_calls.new_page_table(*self._tensors, page)

    table = property(lambda self: self._tensors[0])
    lengths = property(lambda self: self._tensors[1])
    uses = property(lambda self: self._tensors[2])
    missing = property(lambda self: self._tensors[3])

    def __getstate__(self):
        return {name: value for name, value in self.__dict__.items() if name != "_native"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.device = self.table.device
        if self.device.type != "cuda":              # loaded elsewhere: its calls would hand host addresses to kernels
            raise ValueError("a table lives on the GPU")
        self._native = _k.host_calls.new_page_table(*self._tensors, self.page)

    def _pointers(self, count):
        return [t.data_ptr() for t in self._tensors[:count]]

    def _sizes(self):
        return self.sequences, self.width, self.pages, self.page

    def _int32(self, *shape):
        return torch.empty(shape, dtype=torch.int32, device=self.device)

    def _entries(self, t, name):
        check_index(t, name, self.device, 1)
        if t.numel() > MOST_SEQUENCES:
            raise ValueError(f"at most {MOST_SEQUENCES} entries, got {t.numel()}")

    def append(self, offsets: torch.Tensor, tokens: int) -> torch.Tensor:
        """Room for ``tokens`` new tokens, packed along the tokens: those from ``offsets[b]`` to ``offsets[b + 1] - 1`` go behind what
        sequence ``b`` has (int32 on the GPU, ``[sequences + 1]``, ascending).  Returns their slots, int32 ``[tokens]``, for
        ``KeyValueCache.write``.  A sequence whose tokens would need more pages than are free, after those in front of it, or than its row
        has stays as it is, is counted in ``missing``, and its tokens have slot -1, as those outside every sequence have."""
        slots = _k.host_calls.pages_append(self._native, offsets, tokens)
        if slots is not None:
            return slots
        check_index(offsets, "offsets", self.device, 1)
        if offsets.numel() != self.sequences + 1:
            raise ValueError(f"offsets of {self.sequences} sequences have {self.sequences + 1} entries, got {offsets.numel()}")
        tokens = operator.index(tokens)
        if not 0 <= tokens <= MOST_ROWS:
            raise ValueError(f"{tokens} tokens")
        slots, scratch = self._int32(tokens), self._int32(self.sequences)
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_pages_append(*self._pointers(4), offsets.data_ptr(), slots.data_ptr() or None, tokens, *self._sizes(),
                                             scratch.data_ptr(), _k.current_stream()))
        return slots

    def free(self, which: torch.Tensor) -> None:
        """The sequences numbered in ``which`` (int32 on the GPU) end: their length is 0, their pages have one user less.  Numbers that are
        no sequence's (-1, say) are left out."""
        if _k.host_calls.pages_free(self._native, which):
            return
        self._entries(which, "which")
        if which.numel() == 0:
            return
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_pages_free(*self._pointers(3), which.data_ptr(), which.numel(), *self._sizes(), _k.current_stream()))

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Sequence ``children[i]`` becomes what ``parents[i]`` was before the call, for all ``i`` at once (int32 on the GPU): a beam that goes
        on as another, several answers to one prompt.  What the children had is freed; whole pages are shared.  Returns ``(sources,
        targets)`` for ``KeyValueCache.copy``, to be called for the cache of every layer before the next ``append``: the last pages that are not
        full, -1 where none is to be copied (the first heir of a parent that is itself replaced keeps its page).  A child whose page was
        not to be had is left empty and counted in ``missing``.  Of several entries for a child the first counts; an entry with a number that
        is no sequence's is left out."""
        moves = _k.host_calls.pages_fork(self._native, parents, children)
        if moves is not None:
            return moves
        self._entries(parents, "parents")
        self._entries(children, "children")
        count = parents.numel()
        if children.numel() != count:
            raise ValueError(f"{count} parents and {children.numel()} children")
        sources, targets = self._int32(count), self._int32(count)
        if count == 0:
            return sources, targets
        need = _k.lib.bsa_pages_fork_scratch_bytes(count, self.width)
        scratch = torch.empty(need, dtype=torch.uint8, device=self.device)
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_pages_fork(*self._pointers(4), parents.data_ptr(), children.data_ptr(), sources.data_ptr(), targets.data_ptr(),
                                           count, *self._sizes(), scratch.data_ptr(), need, _k.current_stream()))
        return sources, targets

    def compact(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The used pages become the lowest ones: those that lie too high move, in their order, to the free ones below.  Returns ``(sources,
        targets)`` for ``KeyValueCache.copy``, int32 ``[pages // 2]``, filled up with -1, to be called for the cache of every layer."""
        moves = _k.host_calls.pages_compact(self._native)
        if moves is not None:
            return moves
        sources, targets, scratch = self._int32(self.pages // 2), self._int32(self.pages // 2), self._int32(self.pages + 1)
        with _k.on_device(self.device):
            _k.check(_k.lib.bsa_pages_compact(*self._pointers(3), sources.data_ptr() or None, targets.data_ptr() or None, *self._sizes(),
                                              scratch.data_ptr(), _k.current_stream()))
        return sources, targets
