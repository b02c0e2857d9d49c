from .add_layer_norm_func import AddLayerNormFunction, add_layer_norm
from .center_feature_func import CenterFeatureBlendFunction
from .dcnv4_func import DCNv4Function
from .depthwise_conv_func import DepthwiseConvNHWCFunction
from .flash_deform_attn_func import FlashDeformAttnFunction, FlashDeformAttnSplitFunction
from .layer_norm_func import LayerNormResidualFunction, layer_norm_residual
from .query_attention_func import QueryAttentionFunction, query_attention

__all__ = ["AddLayerNormFunction", "CenterFeatureBlendFunction", "DCNv4Function", "DepthwiseConvNHWCFunction", "FlashDeformAttnFunction", "FlashDeformAttnSplitFunction", "LayerNormResidualFunction",
           "QueryAttentionFunction", "add_layer_norm", "layer_norm_residual", "query_attention"]
