"""linear_token_logprobs where all that is left of a row are logits of fp32's lowest value, as a mask by that value leaves them."""

import math

import pytest
import torch

from dense_utils import within

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("V", [2, 37, 256, 700, 7001])
@pytest.mark.parametrize("banned", [False, True])
def test_logits_of_the_lowest_value(rows, V, banned, cuda_device):
    """The products vanish beside it: the row is even over the tokens that are not banned, and the vocabulary's end counts as nothing."""
    from wayfinder_attention_b200 import linear_token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(V + rows)
    x = torch.randn(rows, 24, generator=g, device=cuda_device)
    w = torch.randn(V, 24, generator=g, device=cuda_device)
    b = torch.full((V,), LOWEST, device=cuda_device)
    if banned:
        b[1::3] = -math.inf
    left = torch.isfinite(b)
    n = int(left.sum())
    tokens = torch.nonzero(left)[torch.randint(0, n, (rows,), generator=g, device=cuda_device), 0]
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    r = linear_token_logprobs(*leaves, tokens, bias=b)
    off = 2.0 ** -19 * (1 + math.log(V))  # as for other logits
    assert (r.logprob.double() + math.log(n)).abs().max() <= off
    assert (r.entropy.double() - math.log(n)).abs().max() <= off
    dx, dw = torch.autograd.grad(r.logprob.sum(), leaves)
    dz = -left.double().expand(rows, V) / n
    dz = dz.scatter_add(1, tokens[:, None], torch.ones(rows, 1, dtype=torch.float64, device=cuda_device))
    e = 4 * off * dz.abs() + 2.0 ** -22
    for name, got, a, ea, m in (("dx", dx, dz, e, w.double()), ("dw", dw, dz.T, e.T, x.double())):
        within(got, a @ m, ea @ m.abs() + (a.shape[1] + 8) * 2.0 ** -23 * (a.abs() @ m.abs()), name)


@pytest.mark.parametrize("V", [300, 5000])
def test_lowest_before_others(V, cuda_device):
    """A row whose first tokens are masked by the lowest value and whose last ones are not: those have all the weight."""
    from wayfinder_attention_b200 import linear_token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = torch.randn(70, 24, generator=g, device=cuda_device)
    w = torch.randn(V, 24, generator=g, device=cuda_device)
    b = torch.zeros(V, device=cuda_device)
    kept = 100
    b[:-kept] = LOWEST
    b[:-kept:3] = -math.inf
    tokens = torch.randint(V - kept, V, (70,), generator=g, device=cuda_device)
    r = linear_token_logprobs(x, w, tokens, bias=b)
    want = linear_token_logprobs(x, w[-kept:].contiguous(), tokens - (V - kept))
    off = 2.0 ** -18 * (1 + math.log(V))
    assert ((r.logprob - want.logprob).abs() <= off * (1 + want.logprob.abs())).all()
    assert ((r.entropy - want.entropy).abs() <= off).all()
