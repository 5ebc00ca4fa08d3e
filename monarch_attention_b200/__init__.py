"""B200 (sm_100a) MonarchAttention forward library behind the reference's module API."""
from .host_pipeline import monarch_attention_b200_host
from .kv_cache import CachedAttention, PagedKV, append_kv_b200, cached_attention_b200
from .kv_sequences import AcceptedDrafts, accept_drafts_b200, fork_sequences_b200
from .monarch_attention import MonarchAttention, PadType, monarch_attention_b200, register_impl
from .rotary import RotaryPositions, rotary_b200

__all__ = ["AcceptedDrafts", "CachedAttention", "MonarchAttention", "PadType", "PagedKV", "RotaryPositions", "accept_drafts_b200", "append_kv_b200",
           "cached_attention_b200", "fork_sequences_b200", "monarch_attention_b200", "monarch_attention_b200_host", "register_impl", "rotary_b200"]
