"""Layer norm and linear layers whose whole forward -- and whose backward -- is one call into the HIP kernels, as
functions, as modules and as quantized modules.

FusedLinear is a linear layer, its activation and the addition of a residual as one module: one pass over the output, with
one output quantizer behind it.  With ReLU that is what a configuration with the supergroup [Gemm, Relu] (the reference's
default_config.json) has for the two modules.  With another activation or a residual it is fewer quantizers than
separate modules get: nothing is quantized between the product, the activation and the sum.  A model whose target
quantizes there keeps separate modules.  FusedLayerNorm is nn.LayerNorm on one pass over the input.  Both train: gradients of
input, weight, bias and residual.

float32 and bfloat16 tensors on the GPU; sums and statistics are float32; differentiable once.  In bfloat16 the gradient behind an
activation is rounded on its way into the gradients of input and weight, as between two torch layers.  Under torch.autocast
the functions follow torch's own: linear() computes in the autocast type, layer_norm() in float32.  torch.jit.trace records
them as aimet_amd::linear and aimet_amd::layer_norm; make_fx, torch.export and functorch's transforms are refused.
"""
from typing import Optional, Sequence

import torch
from torch import nn

from ... import ops
from ..._lib import native as _native
from .base import QuantizationMixin

ACTIVATIONS = tuple(ops.ACTIVATIONS)


def layer_norm(input: torch.Tensor, normalized_shape: Sequence[int], weight: Optional[torch.Tensor] = None,  # pylint: disable=redefined-builtin
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """torch.nn.functional.layer_norm on the HIP kernels: normalizes over the trailing `normalized_shape`, then scales
    and shifts.  `weight` and `bias` have that shape and the input's type."""
    return _native.layer_norm(input, normalized_shape, weight, bias, eps)


def linear(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,  # pylint: disable=redefined-builtin
           activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(input weight^T + bias) + residual.  input [..., in], weight [out, in], bias [out], residual of the
    output's shape [..., out]; all of one type.  activation: "none", "relu", "silu", "gelu" (exact) or "gelu_tanh"."""
    code = ops.ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)} is expected")
    return _native.linear(input, weight, bias, code, residual)


class FusedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm computed by layer_norm()."""

    def forward(self, input):  # pylint: disable=redefined-builtin
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)

    @classmethod
    def from_layer_norm(cls, module: nn.LayerNorm) -> "FusedLayerNorm":
        """The same layer norm, sharing its parameters."""
        fused = cls.__new__(cls)
        fused.__dict__ = module.__dict__.copy()
        fused._parameters = module._parameters.copy()
        fused._buffers, fused._modules = module._buffers.copy(), module._modules.copy()
        return fused


class FusedLinear(nn.Module):
    """nn.Linear, an activation and, where forward() is given one, the addition of a residual, computed by linear().

    Deliberately not an nn.Linear: AdaRound and sequential MSE compare outputs of F.linear(), which this module's output
    is not once it has an activation.  Configurations address it as "Gemm"."""

    _quantsim_op_type = "Gemm"

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", device=None,
                 dtype=None):
        super().__init__()
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)} is expected")
        linear_ = nn.Linear(in_features, out_features, bias, device, dtype)     # its initial values
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        self.weight = linear_.weight
        self.register_parameter("bias", linear_.bias)

    def forward(self, input, residual=None):  # pylint: disable=redefined-builtin
        return linear(input, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, " \
               f"activation={self.activation}"

    @classmethod
    def from_linear(cls, module: nn.Linear, activation: str = "none") -> "FusedLinear":
        """The same product followed by `activation`, sharing the weight and the bias."""
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)} is expected")
        fused = cls.__new__(cls)
        nn.Module.__init__(fused)
        fused.in_features, fused.out_features, fused.activation = module.in_features, module.out_features, activation
        fused.weight = module.weight
        fused.register_parameter("bias", module.bias)
        fused.train(module.training)
        return fused


QuantizedFusedLayerNorm = QuantizationMixin.wrap(FusedLayerNorm)
QuantizedFusedLinear = QuantizationMixin.wrap(FusedLinear)
