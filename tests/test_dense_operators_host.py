"""Refusals of fused_linear, layer_norm and token_logprobs that need no GPU: Python checks and the C ABI's."""

import ctypes

import pytest
import torch

from wayfinder_attention_b200 import _lib, fused_linear, layer_norm, token_logprobs


def test_fused_linear_refuses():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="d_in"):
        fused_linear(x, torch.zeros(6, 7))
    with pytest.raises(ValueError, match="d_in"):
        fused_linear(x, torch.zeros(0, 8))
    with pytest.raises(ValueError, match="d_in"):
        fused_linear(torch.zeros(4, 0), torch.zeros(6, 0))
    with pytest.raises(ValueError, match="bias"):
        fused_linear(x, w, torch.zeros(5))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=torch.zeros(6))
    with pytest.raises(ValueError, match="one type"):
        fused_linear(x, w, torch.zeros(6, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_linear(x, w)


def test_layer_norm_refuses():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match=r"d >= 1"):
        layer_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="weight and bias"):
        layer_norm(x, torch.zeros(7))
    with pytest.raises(ValueError, match="weight and bias"):
        layer_norm(x.half(), torch.zeros(8), torch.zeros(8, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer_norm(x)


def test_token_logprobs_refuses():
    x, t = torch.zeros(4, 80), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="vocab"):
        token_logprobs(torch.zeros(4, 0), t)
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(x, t.float())
    for n in (-1, 33):
        with pytest.raises(ValueError, match="top_n"):
            token_logprobs(x, t, top_n=n)
    with pytest.raises(ValueError, match="top_n"):
        token_logprobs(x[:, :3], t, top_n=4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_logprobs(x, t)


def test_abi_validates_before_launch():
    lib = _lib.load_library()
    p = ctypes.c_void_p(4096)

    def linear(dtype=0, M=4, N=8, K=8, xs=8, ws=8, act=0, x=p, y=p):
        return lib.wf_linear(x, p, None, None, dtype, M, N, K, xs, ws, 0, act, None, y, None, 0, None, None)

    assert linear(dtype=5) == _lib.WF_ERR_INVALID_ARGUMENT and b"dtype" in lib.wf_last_error()
    assert linear(K=0) == _lib.WF_ERR_INVALID_ARGUMENT and b"sizes" in lib.wf_last_error()
    assert linear(M=-1) == _lib.WF_ERR_INVALID_ARGUMENT
    assert linear(M=1 << 30) == _lib.WF_ERR_UNSUPPORTED
    assert linear(act=4) == _lib.WF_ERR_INVALID_ARGUMENT and b"activation" in lib.wf_last_error()
    assert linear(xs=7) == _lib.WF_ERR_INVALID_ARGUMENT and b"stride" in lib.wf_last_error()
    assert linear(x=None) == _lib.WF_ERR_INVALID_ARGUMENT and b"null" in lib.wf_last_error()
    assert linear(M=0, x=None, y=None) == _lib.WF_OK

    def linear_bwd(act=1, z=None, ds=8, n=0):
        return lib.wf_linear_backward(p, p, z, p, 0, 4, 8, 8, 8, 8, ds, act, p, p, p, None, n, None, None)

    assert linear_bwd() == _lib.WF_ERR_INVALID_ARGUMENT and b"pre-activations" in lib.wf_last_error()
    assert linear_bwd(z=p, ds=7) == _lib.WF_ERR_INVALID_ARGUMENT and b"stride" in lib.wf_last_error()
    assert linear_bwd(z=p) == _lib.WF_ERR_INVALID_ARGUMENT and b"workspace" in lib.wf_last_error()

    def norm(rows=4, d=8, pd=0, eps=1e-5, mean=None, rstd=None, xs=8, ys=8):
        return lib.wf_layer_norm(p, 0, rows, d, xs, None, None, pd, eps, p, ys, mean, rstd, None)

    assert norm(d=0) == _lib.WF_ERR_INVALID_ARGUMENT
    assert norm(pd=1) == _lib.WF_ERR_INVALID_ARGUMENT and b"weight" in lib.wf_last_error()
    assert norm(eps=float("nan")) == _lib.WF_ERR_INVALID_ARGUMENT and b"eps" in lib.wf_last_error()
    assert norm(mean=p) == _lib.WF_ERR_INVALID_ARGUMENT and b"null" in lib.wf_last_error()
    assert norm(ys=7) == _lib.WF_ERR_INVALID_ARGUMENT and b"stride" in lib.wf_last_error()
    assert norm(rows=0) == _lib.WF_OK
    n = lib.wf_layer_norm_backward_workspace_bytes(100, 64, 0)
    assert n >= 2 * 64 * 4
    rc = lib.wf_layer_norm_backward(p, p, 0, 100, 64, 64, 64, None, 0, p, p, p, p, p, p, n - 1, None)
    assert rc == _lib.WF_ERR_INVALID_ARGUMENT and b"workspace" in lib.wf_last_error()

    def logprobs(rows=4, vocab=50, n=0, top=None, tokens=p):
        return lib.wf_token_logprobs(p, 0, rows, vocab, vocab, tokens, -100, n, p, p, None, top, top, None, None)

    assert logprobs(vocab=0) == _lib.WF_ERR_INVALID_ARGUMENT
    assert logprobs(n=51, top=p) == _lib.WF_ERR_INVALID_ARGUMENT and b"top_n" in lib.wf_last_error()
    assert logprobs(n=40, top=p) == _lib.WF_ERR_UNSUPPORTED and b"maximum" in lib.wf_last_error()
    assert logprobs(n=5) == _lib.WF_ERR_INVALID_ARGUMENT and b"null" in lib.wf_last_error()
    assert logprobs(tokens=None) == _lib.WF_ERR_INVALID_ARGUMENT
    assert logprobs(rows=2 ** 31 - 1, vocab=1 << 20) == _lib.WF_ERR_UNSUPPORTED
    assert logprobs(rows=0) == _lib.WF_OK
    assert lib.wf_max_top_tokens() == 32


def test_kept_pre_activations_start_on_16_bytes():
    lib = _lib.load_library()
    p, off = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    bf16 = 0
    n = lib.wf_linear_backward_workspace_bytes(4, 8, 8, bf16, 1, 1, 1, 1)
    assert lib.wf_linear(p, p, None, None, bf16, 4, 8, 8, 8, 8, 0, 1, off, p, None, 0, None, None) == \
        _lib.WF_ERR_INVALID_ARGUMENT and b"z must be 16-byte aligned" in lib.wf_last_error()
    assert lib.wf_linear_backward(p, p, off, p, bf16, 4, 8, 8, 8, 8, 8, 1, p, p, p, p, n, None, None) == \
        _lib.WF_ERR_INVALID_ARGUMENT and b"z must be 16-byte aligned" in lib.wf_last_error()


def test_small_rounded_gradients_take_two_pieces_of_workspace():
    size = _lib.load_library().wf_linear_backward_workspace_bytes
    bf16, none, gelu, relu = 0, 0, 1, 2
    M, N, K = 1024, 1024, 1024  # 2^30 multiplications: the last size with two pieces
    once = 2 * M * N
    assert size(M, N, K, bf16, relu, 1, 1, 1) - size(M, N, K, bf16, none, 1, 1, 1) == once
    assert size(M, N, K, bf16, gelu, 1, 1, 1) >= size(M, N, K, bf16, relu, 1, 1, 1) + once
    assert size(M, N, 2 * K, bf16, gelu, 1, 1, 1) == size(M, N, 2 * K, bf16, relu, 1, 1, 1)
