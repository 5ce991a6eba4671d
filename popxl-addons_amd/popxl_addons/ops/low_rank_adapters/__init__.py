from popxl_addons.utils import callable_module

from .low_rank_adapters import *

callable_module(__name__, low_rank_adapters)
del callable_module
