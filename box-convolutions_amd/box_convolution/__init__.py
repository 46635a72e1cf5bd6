"""Box convolution for AMD MI355X (gfx950): ``from box_convolution import BoxConv2d``."""
from .box_convolution_module import BoxConv2d
from .operators import (Float8Blocks, GroupNormAct, PointwiseConv2d, PointwiseConv2dFloat8, ResidualNorm, group_norm_act, linear_act,
                        linear_act_float8, quantize_blocks, residual_norm)

__all__ = ["BoxConv2d", "Float8Blocks", "GroupNormAct", "PointwiseConv2d", "PointwiseConv2dFloat8", "ResidualNorm", "group_norm_act", "linear_act",
           "linear_act_float8", "quantize_blocks", "residual_norm"]
