"""Layer primitives the MoE path needs: the parameter-owning base class, the
gated-activation registry, the RMSNorm that precedes the MoE block and the 8-bit
rows it can leave."""

from .activation import GATED_ACTIVATIONS, activation_code
from .base import BaseOP
from .norm import RMSNorm
from reframework_amd.mx import Mxfp8Rows, quantize_mxfp8

__all__ = ["BaseOP", "GATED_ACTIVATIONS", "activation_code", "RMSNorm", "Mxfp8Rows",
           "quantize_mxfp8"]
