"""Rows whose mean is large beside their spread, and rows of one value.

A row of one value c whose sum is exact in fp32 has mean c and deviations of 0 exactly: y is
the bias, and the weight's gradient and dx get nothing but dx's own terms in g.  Otherwise the
mean carries its rounding, 2^-23 |mean| at most (the sum's error is below that where all
values share a sign), and h = (x - mean) rstd inherits it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 7, 256, 1001, 4096, 8193, 20000])
def test_rows_of_one_value(d, dtype, cuda_device):
    from wayfinder_attention_b200 import layer_norm

    x = torch.tensor([0.0, 1.0, -3.0, 160.0, 1000.0, -992.0], device=cuda_device)[:, None].expand(6, d)
    x = x.to(dtype).contiguous().requires_grad_()
    w, b = (torch.randn(d, device=cuda_device).to(dtype).requires_grad_() for _ in range(2))
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.expand(6, d))
    dy = torch.randn(6, d, device=cuda_device).to(dtype)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert not dw.any()
    g = dy.double() * w.detach().double()
    rstd = 1e-5 ** -0.5
    want = rstd * (g - g.mean(-1, keepdim=True))
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}[dtype]
    if dtype != torch.float16:  # 316 times g can pass fp16's end
        assert ((dx.double() - want).abs() <= u * want.abs() + rstd * 2.0 ** -20 * g.abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("d", [256, 1001, 4096, 9000])
def test_large_means(d, cuda_device):
    """fp32, mean 1000 and spread 1: the mean's rounding is all that h may be off by, and the same for a row."""
    from wayfinder_attention_b200 import layer_norm

    g = torch.Generator(device=cuda_device).manual_seed(d)
    x = (torch.randn(64, d, device=cuda_device, generator=g) + 1000).requires_grad_()
    y = layer_norm(x)
    X = x.detach().double()
    h = (X - X.mean(-1, keepdim=True)) / (X.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    assert (y.double() - h).abs().max() <= 1000 * 2.0 ** -22 + 2.0 ** -20 * h.abs().max()
    dy = torch.randn(64, d, device=cuda_device, generator=g)
    w = torch.ones(d, device=cuda_device, requires_grad=True)
    dw, = torch.autograd.grad(layer_norm(x, w), w, dy)
    want = (dy.double() * h).sum(0)
    assert ((dw.double() - want).abs() <= (dy.double().abs().sum(0)) * (1000 * 2.0 ** -22 + 2.0 ** -19)).all()
