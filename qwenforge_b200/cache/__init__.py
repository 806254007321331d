from .allocators import CacheFull, CacheMisuse, PageAllocator, SlotAllocator
from .cache import (PAGE_TOKENS, BundleNeed, BundleSite, KvGroup, KvNeed, KvSite, SequenceCache, StateGroup, StateNeed, StateSite, round_up,
                    tokens_for_continuations)

__all__ = [
    "CacheFull", "CacheMisuse", "PageAllocator", "SlotAllocator", "PAGE_TOKENS", "BundleNeed", "BundleSite", "KvGroup", "KvNeed", "KvSite",
    "SequenceCache", "StateGroup", "StateNeed", "StateSite", "round_up",
    "tokens_for_continuations",
]
