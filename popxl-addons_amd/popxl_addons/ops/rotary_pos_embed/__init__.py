from .rotary_pos_embed import *
