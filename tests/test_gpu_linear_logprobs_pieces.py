"""linear_token_logprobs with a bias in training where the vocabulary's last piece leaves more partial sums of the
bias's gradient than a full one: all three gradients against 64 bits, and what lies behind the workspace."""

import ctypes

import pytest
import torch

from dense_utils import within
from test_gpu_linear_token_logprobs import _check, _inputs, _want

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free_memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,rows,V,d", [
    (torch.bfloat16, 8192, 50257, 768), (torch.float16, 8192, 50257, 768), (torch.float32, 2048, 32000, 4096),
])
def test_a_bias_over_several_pieces(dtype, rows, V, d, cuda_device):
    _check(*_inputs(rows, V, d, dtype, cuda_device))


@pytest.mark.parametrize("dtype,rows,V,d", [
    (torch.bfloat16, 8192, 50257, 768), (torch.float16, 8192, 50257, 768), (torch.float32, 2048, 32000, 1024),
])
def test_nothing_behind_the_workspace_is_written(dtype, rows, V, d, cuda_device):
    """The C entry on exactly the bytes that it asks for, with 1 MB behind them."""
    from wayfinder_attention_b200 import _lib, linear_token_logprobs

    lib = _lib.load_library()
    code = {torch.bfloat16: _lib.WF_DTYPE_BF16, torch.float16: _lib.WF_DTYPE_F16, torch.float32: _lib.WF_DTYPE_F32}[dtype]
    x, w, b, tokens = _inputs(rows, V, d, dtype, cuda_device)
    gl, gh = (torch.randn(rows, device=cuda_device) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    r = linear_token_logprobs(leaves[0], leaves[1], tokens, bias=leaves[2])
    want = torch.autograd.grad([r.logprob, r.entropy], leaves, [gl, gh])

    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def workspace(size):
        margin = 1 << 20
        t = torch.full((size + margin,), 0x5A, dtype=torch.uint8, device=cuda_device)
        return t, t[size:]

    logprob, entropy = (torch.empty(rows, device=cuda_device) for _ in range(2))
    stats = torch.empty(2, rows, device=cuda_device)
    size = lib.wf_linear_token_logprobs_workspace_bytes(rows, V, d, code, 1, 1)
    ws, behind = workspace(size)
    _lib.check(lib.wf_linear_token_logprobs(p(x), p(w), p(b), code, rows, V, d, d, d, p(tokens), -100, p(logprob), p(entropy),
                                            p(stats), p(ws), size, None, stream))
    assert (behind == 0x5A).all()
    grads = [torch.empty_like(t) for t in (x, w, b)]
    size = lib.wf_linear_token_logprobs_backward_workspace_bytes(rows, V, d, code, 1, 1)
    ws, behind = workspace(size)
    _lib.check(lib.wf_linear_token_logprobs_backward(
        p(x), p(w), p(b), code, rows, V, d, d, d, p(tokens), -100, p(stats), p(entropy), p(gl), p(gh), *map(p, grads), p(ws),
        size, None, stream))
    assert (behind == 0x5A).all()
    assert torch.equal(logprob, r.logprob) and torch.equal(entropy, r.entropy)
    for got, one in zip(grads, want):
        assert torch.equal(got, one)
    bound = _want(x, w, tokens, b, gl, gh)["db"]
    within(grads[2], *bound, "db")
