from . import _native
from .layout import SparseLayout
from .matmul import matmul
from .softmax import softmax
from .attention import attention
from .packed import packed_attention
from .cache import KeyValueCache, cached_attention

__all__ = ["SparseLayout", "matmul", "softmax", "attention", "packed_attention", "KeyValueCache", "cached_attention"]
