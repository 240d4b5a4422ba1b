"""Quantized modules of the v2 path."""
from .base import (BaseQuantizationMixin, QuantizationMixin, QuantizedConv2d, QuantizedConvTranspose2d, QuantizedLinear,
                   QuantizedReLU)
from .fused import FusedLayerNorm, FusedLinear, QuantizedFusedLayerNorm, QuantizedFusedLinear

__all__ = ['BaseQuantizationMixin', 'QuantizationMixin', 'QuantizedLinear', 'QuantizedConv2d',
           'QuantizedConvTranspose2d', 'QuantizedReLU', 'FusedLayerNorm', 'FusedLinear', 'QuantizedFusedLayerNorm',
           'QuantizedFusedLinear']
