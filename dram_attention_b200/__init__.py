"""B200-native implementation of the generate stage of DRAM Attention.

Exports the same names as the reference package (dram_attention/__init__.py:3-13), and the operators for several
sequences in one paged cache (`PagedKVCache`, `Rotary`)."""

__version__ = "0.1.0"

from .dram_attention import DRAMAttention
from .lru_cache import CacheOutput, LRUCache
from .max_ip import max_inner_product, max_ip_ref
from .paged_cache import PagedKVCache
from .rotary import Rotary, rotary_frequencies

__all__ = (
    "CacheOutput",
    "DRAMAttention",
    "LRUCache",
    "PagedKVCache",
    "Rotary",
    "max_inner_product",
    "max_ip_ref",
    "rotary_frequencies",
)
