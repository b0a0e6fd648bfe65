"""How exact linear_token_logprobs is past the sizes whose dz is in two pieces, next to fused_linear and token_logprobs.

Both round the gradients of the logits once to the type and the gradients once more; only the second rounds the
logits themselves too (by half a step of some units each: 2^-8 of a logit of 4 in bf16 moves its probability by 1.6%).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spread", [0.0, 0.2])
def test_no_less_exact_than_with_the_logits(dtype, spread, cuda_device):
    from wayfinder_attention_b200 import fused_linear, linear_token_logprobs, token_logprobs

    rows, V, d = 1024, 10007, 512
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(rows, d, device=cuda_device, generator=g).to(dtype).requires_grad_()
    w = (torch.randn(V, d, device=cuda_device, generator=g) * 2.5 * d ** -0.5).to(dtype).requires_grad_()
    t = torch.randint(0, V, (rows,), device=cuda_device, generator=g)
    gl = torch.randn(rows, device=cuda_device, generator=g) * spread - 1
    X, W = x.detach().double(), w.detach().double()
    lp = torch.log_softmax(X @ W.T, 1)
    dz = -lp.exp() * gl.double()[:, None]
    dz[torch.arange(rows, device=cuda_device), t] += gl.double()
    want = (lp.gather(1, t[:, None])[:, 0], dz @ W, dz.T @ X)

    def errors(logprob):
        grads = torch.autograd.grad(logprob, [x, w], gl)
        return [((a.detach().double() - b).norm() / b.norm()).item() for a, b in zip((logprob, *grads), want)]

    own, kept = errors(linear_token_logprobs(x, w, t).logprob), errors(token_logprobs(fused_linear(x, w), t).logprob)
    assert all(a <= b for a, b in zip(own, kept)), (own, kept)
    # the results' own rounding, and one rounding of dz as large again
    for a, b in zip(own[1:], want[1:]):
        rounding = ((b.to(dtype).double() - b).norm() / b.norm()).item()
        assert a <= 2 ** 0.5 * 1.1 * rounding, (a, rounding)
