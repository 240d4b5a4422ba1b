"""Layer norm and linear layers whose whole forward -- and whose backward -- is one call into the HIP kernels, as
functions, as modules and as quantized modules.

A quantized transformer block places one quantizer behind a supergroup ([Gemm, Relu] and the like in the reference's
default_config.json) but runs its members as separate torch modules.  FusedLinear is such a group as one module: product,
bias, activation and residual in one pass over the output, with one output quantizer behind it.  FusedLayerNorm is
nn.LayerNorm on one pass over the input.  Both train: gradients of input, weight, bias and residual.

float32 and bfloat16 tensors on the GPU; sums and statistics are float32.  Under torch.autocast the functions follow
torch's own: linear() computes in the autocast type, layer_norm() in float32.
"""
from typing import Optional, Sequence

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from ... import ops
from .base import QuantizationMixin

ACTIVATIONS = tuple(ops.ACTIVATIONS)


class _LayerNormFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, width, eps):  # pylint: disable=arguments-differ
        x = x.contiguous()
        y, stats = ops.layer_norm_fwd(x, width, weight, bias, eps, want_stats=True)
        ctx.width = width
        ctx.shapes = (None if weight is None else weight.shape, None if bias is None else bias.shape)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):  # pylint: disable=arguments-differ
        x, weight, stats = ctx.saved_tensors
        want_dx, want_dw, want_db = ctx.needs_input_grad[:3]
        dx, dw, db = ops.layer_norm_bwd(x, grad, ctx.width, weight, stats, want_dx, want_dw, want_db)
        w_shape, b_shape = ctx.shapes
        return dx, (dw.view(w_shape) if want_dw else None), (db.view(b_shape) if want_db else None), None, None


class _LinearFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):  # pylint: disable=arguments-differ
        x, weight = x.contiguous(), weight.contiguous()
        wants = any(ctx.needs_input_grad[:3])
        y, saved = ops.linear_fwd(x, weight, bias, activation, residual, want_saved=wants)
        ctx.activation = activation
        if wants:
            ctx.save_for_backward(x, weight, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):  # pylint: disable=arguments-differ
        want_dx, want_dw, want_db, want_dr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_dx or want_dw or want_db:
            x, weight, saved = ctx.saved_tensors
            dx, dw, db = ops.linear_bwd(grad, saved, x, weight, ctx.activation, want_dx, want_dw, want_db)
        return dx, dw, db, (grad if want_dr else None), None


def _differentiates(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _cast(dtype, *tensors):
    return [t if t is None or t.dtype is dtype or not t.is_floating_point() else t.to(dtype) for t in tensors]


def layer_norm(input: torch.Tensor, normalized_shape: Sequence[int], weight: Optional[torch.Tensor] = None,  # pylint: disable=redefined-builtin
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """torch.nn.functional.layer_norm on the HIP kernels: normalizes over the trailing `normalized_shape`, then scales
    and shifts.  `weight` and `bias` have that shape and the input's type."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not shape or tuple(input.shape[-len(shape):]) != shape:
        raise RuntimeError(f"normalized_shape {shape} is not the end of the input's shape {tuple(input.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != shape:
            raise RuntimeError(f"{name} has shape {tuple(t.shape)}, {shape} is expected")
    if torch.is_autocast_enabled("cuda"):
        input, weight, bias = _cast(torch.float32, input, weight, bias)
    width = 1
    for d in shape:
        width *= d
    if _differentiates(input, weight, bias):
        return _LayerNormFunc.apply(input, weight, bias, width, eps)
    return ops.layer_norm_fwd(input, width, weight, bias, eps)[0]


def linear(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,  # pylint: disable=redefined-builtin
           activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """activation(input weight^T + bias) + residual.  input [..., in], weight [out, in], bias [out], residual of the
    output's shape [..., out]; all of one type.  activation: "none", "relu", "silu", "gelu" (exact) or "gelu_tanh"."""
    if activation not in ops.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)} is expected")
    if torch.is_autocast_enabled("cuda"):
        input, weight, bias, residual = _cast(torch.get_autocast_dtype("cuda"), input, weight, bias, residual)
    if _differentiates(input, weight, bias, residual):
        return _LinearFunc.apply(input, weight, bias, residual, activation)
    return ops.linear_fwd(input, weight, bias, activation, residual)[0]


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
