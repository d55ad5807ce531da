from .cache import CacheSpec, CacheState, FullLayerCache, Int4LayerCache, KsaLayerCache
from .engine import KsaInferenceEngine

__all__ = ["CacheSpec", "CacheState", "FullLayerCache", "Int4LayerCache", "KsaLayerCache", "KsaInferenceEngine"]
