"""moba_hip: MI355X-native (gfx950) MoBA sparse block attention.

Importing the package registers the ``opt_hip`` (GQA/MQA/MHA) and
``opt_merge_hip`` (MHA contract) prefill entries in :mod:`moba_hip.api`,
mirroring src/moba_opt/__init__.py:3-7, and exports the decode caches.
"""
from . import baseline_adapter  # noqa: F401
from . import grouped_attention  # noqa: F401  (registers opt_hip, opt_merge_hip)
from .api import available_impls, register, run_impl  # noqa: F401
from .grouped_attention import opt_hip, opt_hip_mha  # noqa: F401
from .merge import merge_forward  # noqa: F401
from .kv_cache import ContiguousKVCache, DecodeResult, PagedKVCache  # noqa: F401
from .prepared_decode import PreparedDecode  # noqa: F401
from .prepared_shared import PreparedSharedDecode  # noqa: F401
from .quantized import QuantizedPages, quantized_append, quantized_attention, quantized_read  # noqa: F401
from .quantized_cache import PreparedQuantizedDecode, QuantizedKVCache  # noqa: F401
from .rotary import RotaryTable, append_rotary  # noqa: F401
from .shared_prefix import SharedPrefixPlan, shared_prefix_attention  # noqa: F401
