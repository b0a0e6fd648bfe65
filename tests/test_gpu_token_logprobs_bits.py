"""fp32 gradients of token_logprobs to fp32's bits.

p = exp(x - m - log s): the exponential is within 2^-22 of its value, and its argument, of size
up to a, carries two roundings (2^-24 a each) and log s's own (2^-23 (1 + log s)).  The rms
over many logits of independent roundings is below half of that bound.
"""

import pytest
import torch

from dense_utils import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [128, 1000, 4001, 50001])
def test_fp32_gradient(V, cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(V)
    rows = 12
    x = (torch.randn(rows, V, device=cuda_device, generator=g) * 2.5).requires_grad_()
    tokens = torch.randint(0, V, (rows,), device=cuda_device, generator=g)
    gl = torch.randn(rows, device=cuda_device, generator=g)
    r = token_logprobs(x, tokens)
    dx, = torch.autograd.grad(r.logprob, x, gl)
    X = x.detach().double()
    logp = torch.log_softmax(X, -1)
    p = logp.exp()
    want = -p * gl.double()[:, None]
    want.scatter_add_(1, tokens[:, None], gl.double()[:, None])
    log_s = torch.logsumexp(X - X.amax(-1, keepdim=True), -1, keepdim=True)
    arg = 2.0 ** -22 + 2.0 ** -23 * (logp.abs() + 1 + 2 * log_s)
    bound = arg * p * gl.double().abs()[:, None] + 2.0 ** -24 * want.abs()
    within(dx, want, bound, "dx")
    other = torch.ones_like(want, dtype=torch.bool).scatter_(1, tokens[:, None], False)
    rel = ((dx.double() - want) / want)[other]
    # a row's log s is one rounding for all of its elements: compared with it taken out
    per_row = ((dx.double() - want) / want).masked_fill(~other, 0).sum(-1, keepdim=True) / (V - 1)
    left = (((dx.double() - want) / want) - per_row)[other]
    assert left.pow(2).mean().sqrt() <= 3.5e-7 and rel.abs().max() <= 4e-6
