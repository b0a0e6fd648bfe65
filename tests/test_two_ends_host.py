"""Refusals of token_embedding and linear_token_logprobs that need no GPU: Python checks and the C ABI's."""

import ctypes

import pytest
import torch

from wayfinder_attention_b200 import _lib, linear_token_logprobs, token_embedding


def test_token_embedding_refuses():
    t, w, p = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(6, 8), torch.zeros(5, 8)
    with pytest.raises(ValueError, match="vocab"):
        token_embedding(t, torch.zeros(6))
    for shape in ((0, 8), (6, 0)):
        with pytest.raises(ValueError, match="vocab"):
            token_embedding(t, torch.zeros(shape))
    with pytest.raises(ValueError, match="position_weight"):
        token_embedding(t, w, position_weight=torch.zeros(5, 7))
    with pytest.raises(ValueError, match="one type"):
        token_embedding(t, w, position_weight=p.half())
    with pytest.raises(ValueError, match="position_weight"):
        token_embedding(t, w, positions=t)
    for positions in (t[:1], t[0, :2], t[0, 0]):
        with pytest.raises(ValueError, match="positions"):
            token_embedding(t, w, position_weight=p, positions=positions)
    for padding in (-1, 6):
        with pytest.raises(ValueError, match="padding_index"):
            token_embedding(t, w, padding_index=padding)
    for scale in (float("inf"), float("nan"), 1e39, -1e300):
        with pytest.raises(ValueError, match="scale"):
            token_embedding(t, w, scale=scale)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_embedding(t, w)


def test_linear_token_logprobs_refuses():
    x, w, t = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(4, dtype=torch.int64)
    for bad in (torch.zeros(6, 7), torch.zeros(0, 8), torch.zeros(8)):
        with pytest.raises(ValueError, match="weight"):
            linear_token_logprobs(x, bad, t)
    with pytest.raises(ValueError, match="weight"):
        linear_token_logprobs(torch.zeros(4, 0), torch.zeros(6, 0), t)
    with pytest.raises(ValueError, match="tokens"):
        linear_token_logprobs(x, w, t[:3])
    with pytest.raises(ValueError, match="bias"):
        linear_token_logprobs(x, w, t, bias=torch.zeros(5))
    with pytest.raises(ValueError, match="one type"):
        linear_token_logprobs(x, w.half(), t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_token_logprobs(x, w, t)


def test_abi_validates_before_launch():
    lib = _lib.load_library()
    p = ctypes.c_void_p(4096)
    bad = _lib.WF_ERR_INVALID_ARGUMENT

    def embed(n=4, dtype=0, V=8, d=8, ws=8, pw=None, P=4, ps=8, positions=None, seq=4, w=p):
        return lib.wf_token_embedding(p, n, w, dtype, V, d, ws, 1.0, pw, P, ps, positions, seq, p, None, None)

    assert embed(dtype=3) == bad and b"dtype" in lib.wf_last_error()
    assert embed(n=-1) == bad and embed(V=0) == bad and embed(d=0) == bad
    assert embed(n=1 << 30) == _lib.WF_ERR_UNSUPPORTED and embed(d=1 << 22) == _lib.WF_ERR_UNSUPPORTED
    assert embed(ws=-1) == bad and b"stride" in lib.wf_last_error()
    assert embed(pw=p, P=0) == bad and embed(pw=p, seq=0) == bad and b"seq" in lib.wf_last_error()
    assert embed(w=None) == bad and b"null" in lib.wf_last_error()
    assert embed(n=0, w=None) == _lib.WF_OK

    def embed_bwd(tokens=p, positions=None, n=100, seq=10, d=64, out=p, places=20, dpos=p, ws=p, short=1, dtype=0):
        size = lib.wf_token_embedding_backward_workspace_bytes(n, 50 if out else 0, places if dpos else 0, d, 0,
                                                               positions is not None)
        return lib.wf_token_embedding_backward(tokens, positions, n, seq, p, dtype, d, d, 50, 1.0, -1, out, places, dpos, ws,
                                               size - short, None)

    assert embed_bwd() == bad and b"workspace" in lib.wf_last_error()
    assert embed_bwd(dpos=None) == bad and b"workspace" in lib.wf_last_error()
    assert embed_bwd(positions=p, out=None) == bad and b"workspace" in lib.wf_last_error()
    assert embed_bwd(seq=7) == bad and b"multiple of seq" in lib.wf_last_error()
    assert embed_bwd(tokens=None) == bad and b"null" in lib.wf_last_error()
    assert embed_bwd(places=0) == bad and embed_bwd(dtype=9) == bad
    assert embed_bwd(out=ctypes.c_void_p(4104)) == bad and b"aligned" in lib.wf_last_error()
    assert embed_bwd(out=None, dpos=None) == _lib.WF_OK  # nothing is asked for
    assert lib.wf_token_embedding_backward_workspace_bytes(0, 50, 0, 64, 0, 1) == 0

    def head(dtype=0, rows=4, V=8, d=8, xs=8, ws=8, tokens=p, n=0):
        return lib.wf_linear_token_logprobs(p, p, None, dtype, rows, V, d, xs, ws, tokens, -100, p, p, None, p, n, None, None)

    assert head(dtype=7) == bad and head(V=0) == bad and head(d=0) == bad and head(xs=7) == bad
    assert head(V=1 << 30) == _lib.WF_ERR_UNSUPPORTED
    assert head(tokens=None) == bad and b"null" in lib.wf_last_error()
    assert head() == bad and b"workspace" in lib.wf_last_error()
    assert head(rows=0) == _lib.WF_OK

    def head_bwd(stats=p, dx=p, n=0):
        return lib.wf_linear_token_logprobs_backward(p, p, None, 0, 4, 8, 8, 8, 8, p, -100, stats, p, p, None, dx, None, None,
                                                     p, n, None, None)

    assert head_bwd() == bad and b"workspace" in lib.wf_last_error()
    assert head_bwd(stats=None) == bad and b"null" in lib.wf_last_error()
    assert head_bwd(dx=None) == _lib.WF_OK  # nothing is asked for


def test_the_backward_holds_pieces_of_the_vocabulary():
    size = _lib.load_library().wf_linear_token_logprobs_backward_workspace_bytes
    for rows, V, d in ((8192, 50001, 1024), (32768, 131072, 256), (65536, 131072, 512)):
        rest = rows * d * 4 + (1 << 26)  # dx in fp32, sums
        assert size(rows, V, d, 0, 1, 1) <= max(1 << 29, 2048 * 2 * rows) + rest


def test_workspaces_of_sizes_that_no_call_takes():
    lib = _lib.load_library()
    huge = (1 << 30, 1 << 31, 1 << 61, 1 << 62, (1 << 63) - 1)
    for size in (lib.wf_linear_token_logprobs_workspace_bytes, lib.wf_linear_token_logprobs_backward_workspace_bytes):
        for n in huge:
            for dtype in range(3):
                assert size(n, 8, 8, dtype, 1, 1) == size(8, n, 8, dtype, 1, 1) == size(8, 8, n, dtype, 1, 1) == 0
    size = lib.wf_token_embedding_backward_workspace_bytes
    for n in huge:
        assert size(n, 8, 8, 8, 0, 1) == size(8, n, 8, 8, 0, 1) == size(8, 8, n, 8, 0, 1) == size(8, 8, 8, n, 0, 1) == 0


def test_the_fp16_backward_holds_pieces_of_the_weights_gradient():
    """It is summed in fp32 before its power of two comes off: a piece's rows of it have 512 MB at most."""
    size = _lib.load_library().wf_linear_token_logprobs_backward_workspace_bytes
    for rows, V, d in ((1, 262144, 4096), (16, 131072, 4096), (512, 131072, 8192), (8192, 50001, 1024)):
        rest = rows * d * 8 + (1 << 27)  # dx in fp32, x's copy, sums, shares of products
        assert size(rows, V, d, _lib.WF_DTYPE_F16, 1, 1) <= (2 << 29) + rest, (rows, V, d)


def test_indices_that_are_not_whole_numbers_are_refused():
    t, w = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(6, 8)
    with pytest.raises(TypeError):
        token_embedding(t, w, padding_index=1.5)
    with pytest.raises((TypeError, RuntimeError)):
        linear_token_logprobs(w[:2], w, t[0, :2], ignore_index=1.5)
