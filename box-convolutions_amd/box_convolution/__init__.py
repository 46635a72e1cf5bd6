"""Box convolution for AMD MI355X (gfx950): ``from box_convolution import BoxConv2d``."""
from .box_convolution_module import BoxConv2d
from .operators import GroupNormAct, PointwiseConv2d, group_norm_act, linear_act

__all__ = ["BoxConv2d", "GroupNormAct", "PointwiseConv2d", "group_norm_act", "linear_act"]
