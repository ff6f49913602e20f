"""Generation and scoring with a compressed model (counterpart of ``ssalaad.inference``)."""
from .generate import generate, generate_no_cache
from .paged import beam_search, cache_for_model, generate_paged, score

__all__ = ["generate", "generate_no_cache", "generate_paged", "beam_search", "score", "cache_for_model"]
