from .manager import CacheError, CacheManager, OutOfPages, PagePool
from .shared import SharedPrefix

__all__ = ["CacheError", "CacheManager", "OutOfPages", "PagePool", "SharedPrefix"]
