"""Captured backwards of token_embedding and linear_token_logprobs for some of their inputs, beside live graphs of the others."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["embedding", "head"])
def test_a_live_graph_of_a_leaf_that_is_not_asked_for(which, cuda_device):
    """autograd.grad for one input does not go to the other's leaf: captured, replayed, and the live graph still has its gradient."""
    from wayfinder_attention_b200 import linear_token_logprobs, token_embedding

    g = torch.Generator(device=cuda_device).manual_seed(1)
    w = torch.randn(300, 64, generator=g, device=cuda_device).requires_grad_()
    other = torch.randn(70, 64, generator=g, device=cuda_device)  # hidden rows, or the positions' table
    dy = torch.randn(70, 64, generator=g, device=cuda_device)
    tokens = torch.randint(0, 300, (70,), generator=g, device=cuda_device)

    def loss(leaf):
        if which == "embedding":
            return (token_embedding(tokens, w, position_weight=leaf) * dy).sum()
        return linear_token_logprobs(leaf, w, tokens).logprob.sum()

    def step():
        leaf = other.detach().requires_grad_()
        got, = torch.autograd.grad(loss(leaf), [leaf])
        return got

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    alive = loss(other.detach())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)
    dw, = torch.autograd.grad(alive, [w])
    assert torch.isfinite(dw).all() and dw.any()
