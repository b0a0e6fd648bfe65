"""linear_token_logprobs over rows that are sure of a token: what is left of 1 - p, of its logarithm and of the entropy.

x is +-1, the weight multiples of 1/16 up to 1, the bias has 8 bits: every logit is exact in fp32 whatever the order
of its sum, and so is its distance to the largest one.  What is left is the sums' own rounding: each addition onto a
sum of 1 + rest loses 2^-24, and a row has ADDS of them behind its largest logit at most (slices of the same tile; a
thread's parts and the levels of the join).  The logarithm and its difference add two roundings of values below 1e-4, and the
entropy the quotient's, as small.  p is an exponential (2^-22 of itself) of the token's log probability (its error).
"""

import math

import pytest
import torch

from dense_utils import ROUNDOFF, TYPES

pytestmark = pytest.mark.gpu

ADDS = 48
ROWS, V, D = 4096, 50001, 16


def _inputs(dtype, dev, rows, token, gap):
    g = torch.Generator(device=dev).manual_seed(token + rows)
    x = (torch.randint(0, 2, (rows, D), generator=g, device=dev) * 2 - 1).to(dtype)
    w = (torch.randint(-16, 17, (V, D), generator=g, device=dev) / 16).to(dtype)
    w[token] = 0
    b = torch.zeros(V, device=dev, dtype=dtype)
    b[token] = gap
    return x, w, b


def _exact(x, w, b, token):
    """Log probability of the token, its 1 - p and the entropy in 64 bits: from the sum over the others."""
    z = x.double() @ w.double().T + b.double()
    z -= z[:, token:token + 1].clone()
    others = z.exp()
    others[:, token] = 0
    rest = others.sum(1)
    lp = -torch.log1p(rest)
    # H = log(1 + rest) - sum over the others of p z
    H = torch.log1p(rest) - (others * z).sum(1) / (1 + rest)
    return lp, rest / (1 + rest), H


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [64, 65, ROWS])
@pytest.mark.parametrize("token", [40, V - 40, V // 2 + 37])
@pytest.mark.parametrize("gap", [21.0, 25.0, 29.5, 37.0])
def test_values_of_sure_rows(dtype, rows, token, gap, cuda_device):
    """1 - p between 1e-3 and 1e-10: above 64 rows as up to 64."""
    from wayfinder_attention_b200 import linear_token_logprobs

    x, w, b = _inputs(dtype, cuda_device, rows, token, gap)
    lp, left, H = _exact(x, w, b, token)
    assert left.max() < 4e-3
    r = linear_token_logprobs(x, w, torch.full((rows,), token, device=cuda_device), bias=b)
    assert (r.logprob <= 0).all() and (r.entropy >= 0).all()
    bound = (ADDS + 2) * 2.0 ** -24
    assert (r.logprob.double() - lp).abs().max() <= bound + 2.0 ** -17 * lp.abs().max()
    # (here and there the others' exponentials, with their arguments' rounding, 64 at most, are off by 2^-17 of themselves)
    assert (r.entropy.double() - H).abs().max() <= bound + 2.0 ** -17 * H.abs().max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [25.0, 29.5])
def test_gradients_of_sure_rows(dtype, gap, cuda_device):
    """The bias's gradient at the token of a batch with one row's gradient is that row's 1 - p: never below 0."""
    from wayfinder_attention_b200 import linear_token_logprobs

    rows, token = 512, V - 40
    x, w, b = _inputs(dtype, cuda_device, rows, token, gap)
    _, left, _ = _exact(x, w, b, token)
    b.requires_grad_()
    r = linear_token_logprobs(x, w, torch.full((rows,), token, device=cuda_device), bias=b)
    bound = (ADDS + 2 + 4) * 2.0 ** -24
    for row in (0, 1, 100, 511):
        db, = torch.autograd.grad(r.logprob[row], [b], retain_graph=True)
        got = db[token].item()
        assert got >= 0, (row, got)
        assert abs(got - left[row].item()) <= bound + 2 * ROUNDOFF[dtype] * left[row].item(), row
