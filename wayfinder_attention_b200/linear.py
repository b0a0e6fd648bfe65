"""Linear layer with bias, activation and residual in the product's epilogue (``wf_linear``).

The decoder's projections and FFN (``routing_attention/models/transformer.py:26-72``) run
``nn.Linear``, the activation and the residual add as separate layers; ``fused_linear``
is one pass over the product, and differentiable in every input.
"""

from __future__ import annotations

import torch

from . import _lib

ACTIVATIONS = {"none": 0, "gelu": 1, "relu": 2, "silu": 3}


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
                 residual: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one kernel; products and sums in fp32, one rounding.

    x: (..., d_in); weight: (d_out, d_in); bias: (d_out,) or None; residual: the output's
    shape (..., d_out) or None; all CUDA tensors of one type (bfloat16, float16 or
    float32).  activation: "none", "gelu" (the erf form), "relu" or "silu".
    Differentiable in x, weight, bias and residual, every gradient in x's type.  The backward
    reads the pre-activations as kept in fp16 (fp32 for fp32), which adds 6% to the error of
    gelu's and silu's fp16 gradients; from 2^30 multiplications on, their own gradient of a
    16-bit gelu or silu is rounded to the type before the products, which leaves x's and the
    weight's gradients with 1.4 times the error of their rounding.
    relu's slope goes by the sign of the pre-activation as its sum came out: one within the
    sum's own rounding of 0 (2^-22 of its terms' size) may fall on either side.
    fp32 inputs are multiplied to fp32 accuracy on the tensor cores, as three bf16 pieces each: an
    infinite or NaN input makes its outputs NaN or infinite, not always the same of the two.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}; expected one of {', '.join(ACTIVATIONS)}")
    if not x.is_cuda:  # refused, after the checks that come before
        return _lib.torch_ops().fused_linear(x, weight, bias, residual, act, 0, status is not None)
    dev = x.device
    y = _lib.torch_ops().fused_linear(x, weight, bias, residual, act, _lib.status_arg(dev, status), status is not None)
    _lib.status_after(dev, status)
    return y


def runs_as(module: torch.nn.Module, kind: type) -> bool:
    """Whether calling ``module`` is ``kind``'s own forward and nothing else: no subclass, hook or replaced forward."""
    return type(module) is kind and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                                         or module._backward_pre_hooks or "forward" in module.__dict__)


def project(layer: torch.nn.Module, x: torch.Tensor, fused: bool, activation: str = "none",
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """A linear layer of a model with what follows it: through ``fused_linear``, or as PyTorch layers.

    A layer that is not a plain ``nn.Linear`` (an adapter in its place, a hook on it) is called.
    Under autocast the product is taken in its type, as ``nn.Linear``'s is, and the residual
    is added in the wider of the two.
    """
    if fused and runs_as(layer, torch.nn.Linear):
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            bias = None if layer.bias is None else layer.bias.to(dtype)
            y = fused_linear(x.to(dtype), layer.weight.to(dtype), bias, activation=activation)
            return y if residual is None else residual + y
        return fused_linear(x, layer.weight, layer.bias, activation=activation, residual=residual)
    y = layer(x)
    if activation == "gelu":
        y = torch.nn.functional.gelu(y)
    return y if residual is None else residual + y
