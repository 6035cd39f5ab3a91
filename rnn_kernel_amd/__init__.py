"""MI355X (gfx950) fp32 GRU training path: hand-written HIP kernels behind a
C ABI (librnn_kernel_amd.so), with an nn.GRU-compatible PyTorch front end."""
from .conv import CausalConvFunction, causal_conv, causal_conv_step
from .delta import GatedDeltaFunction, gated_delta_rule, gated_delta_step
from .delta_layer import GatedDelta
from .gru import (
    GRU,
    GRUFunction,
    MAX_HIDDEN_SIZE,
    RecurrenceAbortedError,
    check_recurrences,
    from_torch_gru,
    gru_forward_inference,
    is_available,
    is_supported_gru,
    set_strict,
)
from .linear import Linear, LinearFunction, linear
from .loss import LinearCrossEntropy, LinearCrossEntropyFunction, linear_cross_entropy
from .norm import LayerNorm, LayerNormFunction, layer_norm
from .scan import SelectiveScanFunction, selective_scan, selective_step
from .scan_layer import SelectiveScan
from .train import AdamW, HeadFunction, LinearHead, MSELossFunction, mse_loss

__all__ = [
    "SelectiveScan",
    "LinearCrossEntropy",
    "LinearCrossEntropyFunction",
    "linear_cross_entropy",
    "SelectiveScanFunction",
    "selective_scan",
    "selective_step",
    "LayerNorm",
    "LayerNormFunction",
    "layer_norm",
    "CausalConvFunction",
    "causal_conv",
    "causal_conv_step",
    "Linear",
    "LinearFunction",
    "linear",
    "GatedDelta",
    "GatedDeltaFunction",
    "gated_delta_rule",
    "gated_delta_step",
    "AdamW",
    "HeadFunction",
    "LinearHead",
    "MSELossFunction",
    "mse_loss",
    "GRU",
    "GRUFunction",
    "MAX_HIDDEN_SIZE",
    "RecurrenceAbortedError",
    "check_recurrences",
    "from_torch_gru",
    "gru_forward_inference",
    "is_available",
    "is_supported_gru",
    "set_strict",
]
