"""An input that is changed in place between forward and backward is refused, whatever its rank."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(6, 32), (2, 3, 32), (2, 3, 2, 32), (32,)]


def _changed(t):
    with torch.no_grad():
        t.add_(1)


def _expect_refusal(out, t):
    _changed(t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear(shape, dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    for which in (0, 1):
        x = torch.randn(shape, device=cuda_device, dtype=dtype, requires_grad=True)
        w = torch.randn(8, 32, device=cuda_device, dtype=dtype, requires_grad=True)
        _expect_refusal(fused_linear(x, w, activation="gelu"), (x, w)[which])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer_norm(shape, dtype, cuda_device):
    from wayfinder_attention_b200 import layer_norm

    for which in (0, 1):
        x = torch.randn(shape, device=cuda_device, dtype=dtype, requires_grad=True)
        w = torch.randn(32, device=cuda_device, dtype=dtype, requires_grad=True)
        _expect_refusal(layer_norm(x, w), (x, w)[which])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_token_logprobs(shape, dtype, cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    x = torch.randn(shape, device=cuda_device, dtype=dtype, requires_grad=True)
    tokens = torch.zeros(shape[:-1], device=cuda_device, dtype=torch.int64)
    _expect_refusal(token_logprobs(x, tokens).logprob, x)
    if shape[:-1]:
        r = token_logprobs(x, tokens)
        _expect_refusal(r.logprob, tokens)


def test_what_is_not_saved_may_change(cuda_device):
    """bias, residual and the norm's bias are not needed; a strided x is kept as the copy that was made of it."""
    from wayfinder_attention_b200 import fused_linear, layer_norm

    x = torch.randn(2, 3, 32, device=cuda_device, requires_grad=True)
    w = torch.randn(8, 32, device=cuda_device, requires_grad=True)
    b, r = torch.randn(8, device=cuda_device, requires_grad=True), torch.randn(2, 3, 8, device=cuda_device, requires_grad=True)
    y = fused_linear(x, w, b, activation="silu", residual=r)
    want = torch.autograd.grad(y.sum(), [x, w, b, r], retain_graph=True)
    _changed(b), _changed(r)
    assert all(torch.equal(a, c) for a, c in zip(want, torch.autograd.grad(y.sum(), [x, w, b, r])))
    nb = torch.randn(32, device=cuda_device, requires_grad=True)
    y = layer_norm(x, None, nb)
    _changed(nb)
    y.sum().backward()
