from .kv_cache_gq import *
