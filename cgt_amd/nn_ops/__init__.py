"""The image-processing ops of the CNN hot path (reference cgt/nn_ops/) and the ops of a transformer layer."""
from . import attention, conv_col, conv_same, cross_channel_lrn, dropout, im2col, layer_norm, max_pool_2d  # noqa: F401
