from .dcnv4_func import DCNv4Function
from .flash_deform_attn_func import FlashDeformAttnFunction
from .layer_norm_func import AddLayerNormFunction, LayerNormFunction, LayerNormResidualFunction

__all__ = ["DCNv4Function", "FlashDeformAttnFunction", "AddLayerNormFunction", "LayerNormFunction",
           "LayerNormResidualFunction"]
