from . import _native
from .layout import SparseLayout
from .matmul import matmul
from .softmax import softmax
from .attention import attention
from .packed import packed_attention
from .cache import KeyValueCache, cached_attention
from .linear import linear_attention_step, packed_linear_attention
from .pages import PageTable

__all__ = ["SparseLayout", "matmul", "softmax", "attention", "packed_attention", "KeyValueCache", "cached_attention",
           "packed_linear_attention", "linear_attention_step", "PageTable"]
