from .cache import CacheLayout, SequenceCache
from .slots import FreeList, PagePool, SlotList
from .spec import CacheFull, KVSpec, PAGE_TOKENS, SideBySideSpec, StateSpec, StoreSizes
from .stores import KVLayerView, Kv4LayerView, KVStore, Kv4Store, SideBySideStore, StateLayerView, StateStore, pages_for

__all__ = ["CacheLayout", "SequenceCache", "FreeList", "PagePool", "SlotList", "CacheFull",
           "KVSpec", "PAGE_TOKENS", "StateSpec", "StoreSizes", "KVLayerView", "Kv4LayerView", "KVStore", "Kv4Store", "StateLayerView",
           "StateStore", "pages_for", "SideBySideSpec", "SideBySideStore"]
