"""Calls under inference_mode, and calls outside it after a first one inside."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_first_call_in_inference_mode(cuda_device, monkeypatch):
    from wayfinder_attention_b200 import _lib, causal_topk, check_status, fused_linear, layer_norm, token_logprobs

    monkeypatch.setattr(_lib, "_status", {})  # as in a new process
    x, w = torch.randn(1, 256, 32, device=cuda_device), torch.randn(8, 32, device=cuda_device)
    t = torch.zeros(1, 256, dtype=torch.int64, device=cuda_device)

    def calls():
        return causal_topk(x, x, 16), fused_linear(x, w, activation="gelu"), layer_norm(x), token_logprobs(x, t).logprob

    with torch.inference_mode():
        inside = calls()
    check_status()
    for _ in range(2 * _lib.READBACK_CALLS):
        outside = calls()
    check_status()
    assert all(torch.equal(a, b) for a, b in zip(inside, outside))
    with torch.inference_mode():
        calls()
        check_status()
        bad = token_logprobs(x, t + 99).logprob
        assert torch.isnan(bad).all()
        with pytest.raises(RuntimeError, match="out of range"):
            check_status()
    wg = w.clone().requires_grad_()
    fused_linear(x, wg, activation="silu").sum().backward()
    assert torch.isfinite(wg.grad).all()
    check_status()
