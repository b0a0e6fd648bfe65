"""The first call of a thread: nothing has made the device's context current there before it."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _in_a_new_thread(f):
    out = []

    def body():
        try:
            out.append(f())
        except Exception as e:  # noqa: BLE001
            out.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    return out[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    x, w = (torch.randn(n, 64, device=cuda_device).to(dtype) for n in (200, 40))
    want = fused_linear(x, w)  # the kernel is set up; its memory goes back to the allocator
    for _ in range(4):
        assert torch.equal(_in_a_new_thread(lambda: fused_linear(x, w)), want)


def test_linear_backward(cuda_device):
    """The products of dx and dw are the first that a fresh backward thread launches where dy is read as it lies."""
    from wayfinder_attention_b200 import fused_linear

    x, w = (torch.randn(n, 64, device=cuda_device, dtype=torch.bfloat16, requires_grad=True) for n in (200, 40))
    dy = torch.randn(200, 40, device=cuda_device, dtype=torch.bfloat16)
    want = torch.autograd.grad(fused_linear(x, w), [x, w], dy)
    for _ in range(4):
        got = _in_a_new_thread(lambda: torch.autograd.grad(fused_linear(x, w), [x, w], dy))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_logprobs_and_retrieval(cuda_device):
    from wayfinder_attention_b200 import causal_topk, layer_norm, token_logprobs

    a = torch.randn(1, 512, 32, device=cuda_device, dtype=torch.bfloat16)
    t = torch.zeros(1, 512, device=cuda_device, dtype=torch.int64)
    for f in (lambda: layer_norm(a), lambda: token_logprobs(a, t, top_n=3).top_tokens, lambda: causal_topk(a, a, 64)):
        want = f()
        assert torch.equal(_in_a_new_thread(f), want)
