"""fused_linear, layer_norm and token_logprobs where element offsets pass 2^31: the last rows are right."""

import pytest
import torch

from dense_utils import within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _release(cuda_device):
    yield
    torch.cuda.empty_cache()


def test_linear_offsets(cuda_device):
    """2.2e9 outputs, and as many inputs to the backward's products."""
    from wayfinder_attention_b200 import fused_linear

    M, N, K = 70000, 32000, 16
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn(M, K, device=cuda_device, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(N, K, device=cuda_device, generator=g) / 4).bfloat16().requires_grad_()
    y = fused_linear(x, w, activation="relu")
    rows = slice(M - 300, M)
    X, W = x.detach()[rows].double(), w.detach().double()
    z = X @ W.T
    size = X.abs() @ W.abs().T
    within(y[rows], z.clamp_min(0), 24 * 2.0 ** -23 * size, "y")
    dy = torch.zeros_like(y)
    dy[rows] = 1.0  # only the last rows' gradient is not 0
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    # z that rounds to another side of 0 changes a slope: leave those out of the oracle's reach
    slope = (y.detach()[rows] > 0).double()
    within(dx[rows], slope @ W, (N + 8) * 2.0 ** -23 * (slope @ W.abs()), "dx")
    within(dw, slope.T @ X, 400 * 2.0 ** -23 * (slope.T @ X.abs()), "dw")
    assert not dx[: M - 300].any()


def test_layer_norm_offsets(cuda_device):
    from wayfinder_attention_b200 import layer_norm

    rows, d = 550000, 4096
    x = torch.randn(rows, d, device=cuda_device, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones(d, device=cuda_device, dtype=torch.bfloat16)
    y = layer_norm(x, w)
    tail = x.detach()[-100:].double()
    h = (tail - tail.mean(1, keepdim=True)) / (tail.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    within(y[-100:], h, 2.0 ** -15 * (1 + h.abs()), "y")
    dx, = torch.autograd.grad(y, [x], y.detach())
    g = y.detach()[-100:].double()
    sd = (tail.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    want = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) / sd
    within(dx[-100:], want, 2.0 ** -15 * (1 + h.abs()) * (g.abs() + h.abs()) / sd, "dx")


def test_token_logprobs_offsets(cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    rows, V = 45000, 50001
    x = torch.randn(rows, V, device=cuda_device, dtype=torch.bfloat16).requires_grad_()
    t = torch.randint(0, V, (rows,), device=cuda_device)
    r = token_logprobs(x, t, top_n=3)
    tail = x.detach()[-50:].double()
    logp = torch.log_softmax(tail, 1)
    within(r.logprob[-50:], logp.gather(1, t[-50:, None])[:, 0], torch.tensor(1e-4), "logprob")
    order = torch.sort(tail, dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(r.top_tokens[-50:], order)
    dx, = torch.autograd.grad(r.logprob.sum(), [x])
    want = -logp.exp()
    want[torch.arange(50, device=cuda_device), t[-50:]] += 1
    within(dx[-50:], want, 1e-4 * want.abs(), "dlogits")
