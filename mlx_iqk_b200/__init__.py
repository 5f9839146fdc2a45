"""B200-native IQ_K routed-expert hot path (drop-in for mlx-iqk's IqkSwitchLinear).

Hand-written sm_100a CUDA kernels behind a C ABI (``include/iqk_b200.h``,
``libiqk_b200.so``), reached from this thin PyTorch layer. Nothing here falls
back to the CPU: a missing library raises.
"""

from . import format  # noqa: F401
from .format import IqkFormatError
from .kernels import IqkKernelError, IqkRuntimeError
from .nn import DECODE_MAT_LIMIT, IqkSwitchLinear, grid_table, member_table, value_table
from .glu import GraphedSwitchGLU, IqkSwitchGLU
from .mx import (MxSwitchGLU, mx_aligned_scales, mx_dequantize, mx_linear, mx_quantize,
                 mx_switch_linear)
from .router import balance_loss, route, route_balanced

__all__ = ["DECODE_MAT_LIMIT", "IqkFormatError", "IqkKernelError", "IqkRuntimeError",
           "GraphedSwitchGLU", "IqkSwitchGLU", "IqkSwitchLinear", "MxSwitchGLU", "balance_loss",
           "format", "grid_table", "member_table", "mx_aligned_scales", "mx_dequantize",
           "mx_linear", "mx_quantize", "mx_switch_linear", "route", "route_balanced",
           "value_table"]
