"""Layer primitives the MoE path needs: the parameter-owning base class, the
gated-activation registry, the RMSNorm or LayerNorm that precedes the MoE block and the
8-bit rows the former can leave."""

from .activation import GATED_ACTIVATIONS, activation_code
from .base import BaseOP
from .norm import LayerNorm, RMSNorm
from reframework_amd.mx import Mxfp8Rows, quantize_mxfp8

__all__ = ["BaseOP", "GATED_ACTIVATIONS", "activation_code", "RMSNorm", "LayerNorm", "Mxfp8Rows",
           "quantize_mxfp8"]
