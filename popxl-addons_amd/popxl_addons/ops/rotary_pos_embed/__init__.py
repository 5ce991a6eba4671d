from popxl_addons.utils import callable_module

from .rotary_pos_embed import *

callable_module(__name__, rotary_pos_embed)
del callable_module
