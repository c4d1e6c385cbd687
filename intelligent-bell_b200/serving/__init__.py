"""Cache sink, multi-layer injector over the restore pipeline, and decoding behind a shared prefix."""

from .kv_injector import KVInjector, MultiLayerKVInjector, SpecDynamicCache
from .shared_prefix import SharedPrefixCache

__all__ = ["KVInjector", "MultiLayerKVInjector", "SharedPrefixCache", "SpecDynamicCache"]
