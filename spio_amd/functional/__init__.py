"""Functional interface: the `spio::conv2d_gw8` custom operators, norms over channels_last tensors, the 8-bit form,
and the operators of token-mixing layers."""

from .conv2d_gw8_function import (
    conv2d_gw8,
    conv2d_gw8_backward_op,
    fused_backward_kernel,
    reset_fused_backward_choices,
)
from .layernorm_2d_function import layernorm_2d, layernorm_2d_backward, layernorm_2d_gradients
from .group_norm_2d_function import group_norm_2d, group_norm_2d_gradients
from .activation_8bit_function import Packed8bit, activation_8bit, activation_8bit_gradient, pack_8bit, unpack_8bit
from .conv2d_gw8_8bit_function import conv2d_gw8_8bit, conv2d_gw8_8bit_gradients
from .causal_conv1d_function import causal_conv1d, causal_conv1d_gradients, causal_conv1d_step
from .selective_scan_function import selective_scan, selective_scan_gradients, selective_scan_step
from .head_norm_rotary_function import head_norm_rotary, head_norm_rotary_gradients, rotary, rotary_frequencies
from .. import native as _native_path

_native_path.adopt(conv2d_gw8, "conv2d_gw8")
_native_path.adopt(layernorm_2d, "layernorm_2d")
_native_path.configure(conv2d_gw8_backward_op, layernorm_2d_gradients)
_native_path.configure_kept(group_norm_2d_gradients, activation_8bit_gradient, conv2d_gw8_8bit_gradients)
_native_path.configure_tokens(causal_conv1d_gradients, selective_scan_gradients, head_norm_rotary_gradients)
