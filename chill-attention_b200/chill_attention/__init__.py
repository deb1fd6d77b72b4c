"""chill_attention for NVIDIA B200 (sm_100a): masked flash attention with the API of
alexdremov/chill-attention (same export list as its chill_attention/__init__.py:1-13), the operators that serve a
model from a paged cache (cache.py), rotary positions (rotary.py) and beam search (beams.py)."""
from .chill import (
    _chill_reference_naive,
    chill_attention,
    register_chill_mask,
)
from ._cabi import is_deterministic, set_deterministic
from .beams import ChillBeams, chill_beam_select
from .cache import (
    ChillCopies,
    ChillPages,
    ChillStep,
    chill_attention_cached,
    chill_cache_append,
    chill_cache_commit,
    chill_cache_copy,
    chill_pages_compact,
    chill_pages_fork,
    chill_pages_reserve,
    chill_pages_trim,
)
from .mask import (
    CausalChillMask,
    ChillMask,
    ChunkwiseChillMask,
    FullChillMask,
    PrefixLMChillMask,
    SlidingWindowChillMask,
)
from .rotary import ChillRotary, chill_rotate, chill_rotate_append

__all__ = [
    "chill_attention", "register_chill_mask", "_chill_reference_naive", "ChillMask", "FullChillMask",
    "CausalChillMask", "SlidingWindowChillMask", "ChunkwiseChillMask", "PrefixLMChillMask",
    "set_deterministic", "is_deterministic",
    "ChillPages", "ChillStep", "chill_pages_reserve", "chill_pages_trim", "chill_cache_append", "chill_cache_commit",
    "chill_attention_cached",
    "ChillCopies", "chill_pages_fork", "chill_pages_compact", "chill_cache_copy",
    "ChillRotary", "chill_rotate", "chill_rotate_append", "ChillBeams", "chill_beam_select",
]
