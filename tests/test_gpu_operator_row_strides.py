"""One row, or none, whose row stride says nothing: a transposed column is a valid input and a valid gradient.

``torch.randn(d, 1).t()`` is (1, d) with strides (1, 1), contiguous by PyTorch's rules.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32]


def _row(*shape, dtype, dev, seed=0):
    """(1, d) or (0, d) with a row stride of 1."""
    g = torch.Generator().manual_seed(seed)
    n, d = shape
    t = torch.randn(d, n, generator=g).to(dev, dtype).t()
    assert t.stride(0) < d
    return t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("K,N", [(16, 8), (509, 130)])
def test_linear(K, N, act, dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    g = torch.Generator().manual_seed(1)
    w = torch.randn(N, K, generator=g).to(cuda_device, dtype)
    x = _row(1, K, dtype=dtype, dev=cuda_device)
    for a, b in ((x, w), (torch.randn(5, K, generator=g).to(cuda_device, dtype), x), (x, x)):
        with torch.no_grad():
            assert torch.equal(fused_linear(a, b, activation=act), fused_linear(a.clone(memory_format=torch.contiguous_format).reshape(a.shape), b.contiguous(), activation=act))
        # a consumer that takes y transposed gives its gradient transposed
        la, lb = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = fused_linear(la, lb, activation=act)
        dy = torch.randn(y.shape, generator=g).to(cuda_device, dtype)
        got = torch.autograd.grad(y.t(), [la, lb], dy.t(), retain_graph=True)
        want = torch.autograd.grad(y, [la, lb], dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    r = _row(1, N, dtype=dtype, dev=cuda_device, seed=3)
    assert torch.equal(fused_linear(x, w, residual=r), fused_linear(x, w, residual=r.reshape(N).clone()[None]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 24, 1001])
def test_layer_norm(d, dtype, cuda_device):
    from wayfinder_attention_b200 import layer_norm

    x = torch.randn(d, 1, device=cuda_device).to(dtype).t().requires_grad_()
    w, b = (torch.randn(d, device=cuda_device, dtype=dtype, requires_grad=True) for _ in range(2))
    y = layer_norm(x, w, b)
    dy = torch.randn(1, d, device=cuda_device).to(dtype)
    want = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
    got = torch.autograd.grad(y.t(), [x, w, b], dy.t().contiguous(), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    column = dy.reshape(d, 1).clone()
    got = torch.autograd.grad(y, [x, w, b], column.t())
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    flat = x.detach().reshape(d).clone()[None].requires_grad_()
    assert torch.equal(layer_norm(flat, w, b), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 40, 3000])
def test_token_logprobs(V, dtype, cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    x = torch.randn(V, 1, device=cuda_device).to(dtype).t()
    t = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    flat = x.reshape(V).clone()[None]
    grads = []
    for leaf in (x.clone(memory_format=torch.preserve_format).requires_grad_(), flat.requires_grad_()):
        r = token_logprobs(leaf, t, top_n=1)
        grads.append((*r, *torch.autograd.grad(r.logprob.sum(), leaf)))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear, layer_norm

    w = torch.randn(8, 16, device=cuda_device, dtype=dtype, requires_grad=True)
    x = torch.empty(16, 0, device=cuda_device, dtype=dtype).t().requires_grad_()
    for y, leaves in ((fused_linear(x, w), [x, w]), (layer_norm(x, w[0]), [x, w])):
        grads = torch.autograd.grad(y.t().sum(), leaves)
        assert grads[0].shape == (0, 16) and not grads[1].any()


def test_gradient_with_no_strides(cuda_device):
    """The gradient of a sum is one element for all, also where there is one row or one column."""
    from wayfinder_attention_b200 import fused_linear, layer_norm

    for M, N in ((1, 1), (1, 5), (5, 1)):
        x = torch.randn(M, 16, device=cuda_device, requires_grad=True)
        w = torch.randn(N, 16, device=cuda_device, requires_grad=True)
        y = fused_linear(x, w)
        one = torch.ones((), device=cuda_device).as_strided((M, N), (0, 0))
        dx, dw = torch.autograd.grad(y, [x, w], one)
        assert torch.allclose(dx, w.sum(0).expand(M, 16), atol=1e-5)
        assert torch.allclose(dw, x.sum(0).expand(N, 16), atol=1e-5)
        z = torch.randn(M, N, device=cuda_device, requires_grad=True)
        torch.autograd.grad(layer_norm(z), z, one)
