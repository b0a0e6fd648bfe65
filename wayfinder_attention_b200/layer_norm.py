"""Layer norm over the last axis, with its backward (``wf_layer_norm``).

What the decoder's ``nn.LayerNorm`` computes (``routing_attention/models/transformer.py:26-72``):
one pass over the rows each way, statistics in fp32, and the weight's and bias's
gradients reduced in a fixed order.
"""

from __future__ import annotations

import torch

from . import _lib


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, rounded once.

    x: (..., d) CUDA tensor of bfloat16, float16 or float32; weight and bias: (d,), both of
    x's type or both float32, or None.  Differentiable in x, weight and bias.
    """
    return _lib.torch_ops().layer_norm(x, weight, bias, eps)
