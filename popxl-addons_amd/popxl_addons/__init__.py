"""MI355X-native group-quantization path of popxl-addons.

The 4-bit group-quantization decompress path, at the reference's import paths: the op wrappers under
`popxl_addons.ops.group_quantize_decompress` and the `LinearGQ` layer under `popxl_addons.layers.linear_gq`; and
the operators that a decoder needs beside it, under `popxl_addons.ops`: `rotary_pos_embed`, `kv_cache_gq`,
`low_rank_adapters`.  Importing this package loads
neither torch nor the HIP library; both are loaded on first use of a device op.
"""
__version__ = "0.1.0"
