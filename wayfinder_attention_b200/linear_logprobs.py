"""Log probabilities of given tokens from hidden states and a head's weight (``wf_linear_token_logprobs``).

``token_logprobs`` of the head's logits without the logits: a piece of the vocabulary at a
time, the product's accumulator goes into running sums, so that scoring and training over a
large vocabulary hold nothing of the size (tokens, vocabulary).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class LinearLogprobs(NamedTuple):
    logprob: torch.Tensor  # (...) float32
    entropy: torch.Tensor  # (...) float32


def linear_token_logprobs(x: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor,
                          bias: torch.Tensor | None = None, ignore_index: int = -100,
                          status: torch.Tensor | None = None) -> LinearLogprobs:
    """Log probability of ``tokens`` under ``softmax(x @ weight.T + bias)`` and that distribution's entropy, in float32.

    x: (..., d); weight: (vocab, d); bias: (vocab,) or None; CUDA tensors of one type (bfloat16,
    float16 or float32); tokens: (...) int64 or int32.  The logits are fp32 and not rounded.
    A token equal to ``ignore_index`` gets log probability 0 and no gradient from it; any other
    token outside the vocabulary gets NaN, NaN gradients, and sets the status word's bit 0.
    A bias of -inf bans its token; a row whose tokens are all banned has log probability -inf,
    entropy 0 and no gradient.  A NaN or +inf among its logits makes a row NaN.
    Differentiable in x, weight and bias through logprob and entropy.  The backward makes the
    logits again.  Their gradients are taken to x's type before the two products (two pieces of
    it up to 64 rows or 2^30 multiplications, one above, which leaves x's and weight's gradients
    with 1.4 times the error of their rounding; float32 in three bf16 pieces).  In float16 a row whose
    gradient is 2^-24 of the largest row's, or less, loses digits of x in weight's gradient.  The workspace holds them
    for a piece of the vocabulary: at most 512 MB, or 2048 columns; in float16 as much again for
    the piece's rows of weight's gradient.  What the tensor cores cannot read as it lies is laid out in
    the workspace besides, forward and backward: float32 x and weight whole, in 6 bytes an element (3.2 GB for
    a weight of (131072, 4096)), and 16-bit ones whose rows do not start on 16 bytes, in 2.
    """
    if not x.is_cuda:  # refused, after the checks that come before
        return LinearLogprobs(*_lib.torch_ops().linear_token_logprobs(x, weight, tokens, bias, ignore_index, 0,
                                                                      status is not None))
    dev = x.device
    r = _lib.torch_ops().linear_token_logprobs(x, weight, tokens, bias, ignore_index, _lib.status_arg(dev, status),
                                               status is not None)
    _lib.status_after(dev, status)
    return LinearLogprobs(*r)
