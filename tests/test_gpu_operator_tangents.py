"""Forward-mode derivatives are refused, not lost, also where no input asks for a gradient."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def test_dual_inputs_are_refused(cuda_device):
    from wayfinder_attention_b200 import fused_linear, layer_norm, token_logprobs

    x, w = torch.randn(4, 16, device=cuda_device), torch.randn(8, 16, device=cuda_device)
    t = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        dw = fwad.make_dual(w, torch.ones_like(w))
        for call in (lambda: fused_linear(d, w), lambda: fused_linear(x, dw), lambda: layer_norm(d),
                     lambda: layer_norm(x, dw[0]), lambda: token_logprobs(d, t),
                     lambda: fused_linear(x, w, residual=fwad.make_dual(torch.ones(4, 8, device=cuda_device),
                                                                        torch.ones(4, 8, device=cuda_device)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # inputs without tangents run
        assert fused_linear(x, w).shape == (4, 8)
