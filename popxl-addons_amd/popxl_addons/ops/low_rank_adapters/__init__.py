from .low_rank_adapters import *
