"""Log probabilities of given tokens, with entropy and top alternatives (``wf_token_logprobs``).

What scoring an answer and training on it take from the logits: one pass over each row
gives the token's log probability (its negative mean is the cross entropy of the
reference's training loss), the entropy of the distribution and its most likely tokens.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib


MAX_TOP_TOKENS = 32  # wf_max_top_tokens()


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor  # (...) float32
    entropy: torch.Tensor  # (...) float32
    top_logprobs: torch.Tensor  # (..., top_n) float32, descending
    top_tokens: torch.Tensor  # (..., top_n) int64


def _launch(logits, tokens, top_n, ignore_index, lead, keep_stats, status):
    dev = logits.device
    rows, vocab = logits.shape
    logprob = torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    stats = torch.empty(2, rows, dtype=torch.float32, device=dev) if keep_stats else None
    top_logprobs = torch.empty((*lead, top_n), dtype=torch.float32, device=dev)
    top_tokens = torch.empty((*lead, top_n), dtype=torch.int64, device=dev)
    st = _lib.status_arg(dev, status)
    with _lib.on_device(dev):
        rc = _lib.load_library().wf_token_logprobs(
            logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, vocab, logits.stride(0), tokens.data_ptr(),
            ignore_index, top_n, logprob.data_ptr(), entropy.data_ptr(), None if stats is None else stats.data_ptr(),
            top_logprobs.data_ptr(), top_tokens.data_ptr(), st, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    _lib.status_after(dev, status)
    return logprob, entropy, stats, top_logprobs, top_tokens


class _TokenLogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_n, ignore_index, lead):
        x = _lib.rows_of(logits)
        logprob, entropy, stats, top_logprobs, top_tokens = _launch(x, tokens, top_n, ignore_index, lead, True, None)
        ctx.save_for_backward(x, tokens, stats, entropy)
        ctx.ignore_index, ctx.shape = ignore_index, logits.shape
        ctx.mark_non_differentiable(top_logprobs, top_tokens)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogprob, dentropy, _top_logprobs, _top_tokens):
        if dlogprob is None and dentropy is None:
            return None, None, None, None, None
        x, tokens, stats, entropy = ctx.saved_tensors
        rows, vocab = x.shape
        dev = x.device
        dlogprob = None if dlogprob is None else dlogprob.contiguous()
        dentropy = None if dentropy is None else dentropy.contiguous()
        dx = x.new_empty(ctx.shape)
        with _lib.on_device(dev):
            rc = _lib.load_library().wf_token_logprobs_backward(
                x.data_ptr(), _lib.dtype_code(x.dtype), rows, vocab, x.stride(0), tokens.data_ptr(), ctx.ignore_index,
                stats.data_ptr(), entropy.data_ptr(), None if dlogprob is None else dlogprob.data_ptr(),
                None if dentropy is None else dentropy.data_ptr(), dx.data_ptr(), _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc)
        return dx, None, None, None, None


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
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"expected logits (..., vocab) with vocab >= 1, got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not match logits {tuple(logits.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
    most = min(logits.shape[-1], MAX_TOP_TOKENS)
    if not 0 <= top_n <= most:
        raise ValueError(f"top_n must be in [0, {most}] here, got {top_n}")
    _lib.require_cuda(logits, tokens)
    lead = tokens.shape
    flat = tokens if tokens.dtype == torch.int64 else tokens.to(torch.int64)
    flat = flat if flat.is_contiguous() else flat.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        if status is not None:
            raise ValueError("status is not supported on the differentiable path")
        return TokenLogprobs(*_TokenLogprobsFunction.apply(logits, flat, top_n, ignore_index, lead))
    logprob, entropy, _, top_logprobs, top_tokens = _launch(_lib.rows_of(logits), flat, top_n, ignore_index, lead,
                                                            False, status)
    return TokenLogprobs(logprob, entropy, top_logprobs, top_tokens)
