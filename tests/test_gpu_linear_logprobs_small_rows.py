"""fp16 weights' gradients of linear_token_logprobs where one row's gradient is far below the largest one's.

Row 0's token is no other row's and has a bias of -60, so that its row of dW is gl (1 - p) x of that row alone (the
others add 2^-80 of theirs).  dz is rounded twice at most and the result once, by 2^-11 of themselves each; x may be
moved towards fp16's smallest steps, of 2^-24, by what 10 binades leave of the ratio.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,V,d", [(200, 1000, 64), (1024, 16384, 80), (70, 3001, 33)])
@pytest.mark.parametrize("ratio", [0, 5, 12, 16, 20, 24])
def test_a_rare_token_with_a_small_gradient(rows, V, d, ratio, cuda_device):
    from wayfinder_attention_b200 import linear_token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(ratio + rows)
    x = torch.randn(rows, d, generator=g, device=cuda_device).half().requires_grad_()
    w = (torch.randn(V, d, generator=g, device=cuda_device) * d ** -0.5).half().requires_grad_()
    b = torch.zeros(V, device=cuda_device, dtype=torch.float16)
    rare = V - 3
    b[rare] = -60.0
    b.requires_grad_()
    tokens = torch.randint(0, V - 10, (rows,), generator=g, device=cuda_device)
    tokens[0] = rare
    large = 2.0 ** 12
    gl = torch.full((rows,), large, device=cuda_device)
    gl[0] = large * 2.0 ** -ratio
    r = linear_token_logprobs(x, w, tokens, bias=b)
    dx, dw, db = torch.autograd.grad(r.logprob, [x, w, b], gl)
    want = gl[0].double() * x[0].detach().double()
    u, step = 2.0 ** -11, 2.0 ** -25
    off = 4 * u * want.abs() + gl[0].double() * 2 * step * 2.0 ** max(0, ratio - 10) + step
    assert ((dw[rare].double() - want).abs() <= off).all(), ((dw[rare].double() - want).abs() / off).max()
    assert abs(db[rare].item() - gl[0].item()) <= 4 * u * gl[0].item()
    # that row's dx against its own size: gl (w_t - sum p w)
    p = torch.softmax(x[0].detach().double() @ w.detach().double().T + b.detach().double(), 0)
    want = gl[0].double() * (w[rare].detach().double() - p @ w.detach().double())
    size = gl[0].double() * (w[rare].detach().double().abs() + p @ w.detach().double().abs())
    # p's own error is 2^-15 of it, its smallest step 2^-28 of the row's gradient
    least = gl[0].double() * 2.0 ** -28 * w.detach().double().abs().sum(0)
    assert ((dx[0].double() - want).abs() <= 4 * u * size + least + step).all()
