"""Token embedding with scaling and positions, with its tables' gradients (``wf_token_embedding``).

What the decoder's two ``nn.Embedding`` and their sum compute
(``routing_attention/models/transformer.py:76-312``), in one pass; the gradients are sums
over the sorted tokens, the same bits each time.
"""

from __future__ import annotations

import operator

import torch

from . import _lib


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                    position_weight: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                    padding_index: int | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * weight[tokens] + position_weight[positions]``, rounded once: (..., d) for tokens (...).

    tokens: int64 or int32; weight: (vocab, d) and position_weight: (places, d) or None, CUDA
    tensors of one type (bfloat16, float16 or float32).  positions: int64 or int32, of the
    tokens' shape or of its last axis; None counts 0, 1, ... along the last axis.
    Differentiable in weight and position_weight: the gradients are dense, summed in fp32 in a
    fixed order and rounded once.  ``weight``'s row ``padding_index`` gets none.  A token or
    position outside its table makes its row NaN, adds nothing to a gradient of the table it is
    outside of, and sets the status word's bit 0.
    """
    padding = -1 if padding_index is None else operator.index(padding_index)
    if padding_index is not None and padding < 0:
        raise ValueError(f"padding_index must be >= 0, got {padding_index}")
    if not weight.is_cuda:  # refused, after the checks that come before
        return _lib.torch_ops().token_embedding(tokens, weight, scale, position_weight, positions, padding, 0,
                                                status is not None)
    dev = weight.device
    y = _lib.torch_ops().token_embedding(tokens, weight, scale, position_weight, positions, padding,
                                         _lib.status_arg(dev, status), status is not None)
    _lib.status_after(dev, status)
    return y
