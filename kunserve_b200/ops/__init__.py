from ._native import native, available, check_error, NativeUnavailable
from .cache import (DecodePlan, PagedKV, PrefixGroup, SharedPrefixPlan, compact_cache, select_evictions,
                    shared_prefix_attention, weighted_decode_attention)
from .rotary import Rotary, rotary_append, rotary_apply, rotary_frequencies
