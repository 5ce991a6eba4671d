"""Custom ops.  The reference keeps the group-quantization ops out of this namespace to avoid a
compile on import (popxl_addons/ops/__init__.py:2); nothing is compiled on import here (the HIP
library is prebuilt and loaded on first use), so the public names are available from `popxl_addons.ops`
as well as from their modules.  `rotary_pos_embed` and `low_rank_adapters` name a module and the function in
it: here they are the modules, which are called as the functions."""
from .group_quantize_decompress import (  # noqa: F401
    group_quantize_compress,
    group_quantize_compress_numpy,
    group_quantize_decompress,
    group_quantize_decompress_numpy,
)
from .kv_cache_gq import KVCacheGQ, kv_cache_append, kv_cache_attention, kv_cache_gather  # noqa: F401
from .low_rank_adapters import AdapterPlan, LowRankAdapters, low_rank_adapters_grad  # noqa: F401
from .rotary_pos_embed import RotaryPosEmbed, rotary_frequencies  # noqa: F401
