"""Log probabilities of given tokens, with entropy and top alternatives (``wf_token_logprobs``).

What scoring an answer and training on it take from the logits: one pass over each row
gives the token's log probability (its negative mean is the cross entropy of the
reference's training loss), the entropy of the distribution and its most likely tokens.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor  # (...) float32
    entropy: torch.Tensor  # (...) float32
    top_logprobs: torch.Tensor  # (..., top_n) float32, descending
    top_tokens: torch.Tensor  # (..., top_n) int64


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0, ignore_index: int = -100,
                   status: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probability of ``tokens`` under ``logits``, entropies and the ``top_n`` likeliest tokens, in float32.

    logits: (..., vocab) CUDA tensor of bfloat16, float16 or float32; tokens: (...) int64
    or int32.  A token equal to ``ignore_index`` gets log probability 0 and no gradient
    from it; any other token outside the vocabulary gets NaN and sets the status word's
    bit 0.  A logit of -inf bans its token; a row of nothing else has log probability
    -inf, entropy 0 and no gradient.  Equal logits rank by the lower index, NaN first.
    top_n is at most 32.  Differentiable in logits through logprob and entropy.
    """
    if not logits.is_cuda:  # refused, after the checks that come before
        return TokenLogprobs(*_lib.torch_ops().token_logprobs(logits, tokens, top_n, ignore_index, 0,
                                                              status is not None))
    dev = logits.device
    r = _lib.torch_ops().token_logprobs(logits, tokens, top_n, ignore_index, _lib.status_arg(dev, status),
                                        status is not None)
    _lib.status_after(dev, status)
    return TokenLogprobs(*r)
