from ._native import native, available, check_error, NativeUnavailable
from .cache import (DecodePlan, PagedKV, PrefixGroup, SharedPrefixPlan, compact_cache, select_evictions,
                    shared_prefix_attention, weighted_decode_attention)
from .int8 import (Int8Weight, add_rms_norm_int8, dequantize_int8, int8_linear, quantize_int8,
                   silu_mul_int8)
from .rotary import Rotary, rotary_append, rotary_apply, rotary_frequencies
