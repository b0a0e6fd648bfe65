"""gelu over all of its negative side, where its values are small: relative error, not absolute.

The depth is 1 and the weight (or x) 1, so z is the input itself.  16-bit results are
evaluated to 2^-14 of themselves before their rounding down to z = -5.75, past which fp16 has
no bits left, and to 2^-10 down to z = -12.9, near bf16's end (its rounding is 2^-8).  fp32 goes by
erfc: 2^-21 (five units), and z^2 2^-23 for the two roundings of its argument.
"""

import math

import pytest
import torch

from dense_utils import within

pytestmark = pytest.mark.gpu


def _sweep(dtype, dev):
    if dtype == torch.float32:
        return -torch.linspace(1e-4, 12.9, 20000, device=dev)
    every = torch.arange(0x8000, 0x10000, device=dev, dtype=torch.int32).to(torch.int16).view(dtype)
    z = every.double()
    return every[torch.isfinite(z) & (z >= (-12.9 if dtype == torch.bfloat16 else -8.0)) & (z < -1e-3)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", ["many", "one"])
def test_negative_side(rows, dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    v = _sweep(dtype, cuda_device)
    one = torch.ones(1, 1, dtype=dtype, device=cuda_device)
    y = fused_linear(v[:, None], one, activation="gelu")[:, 0] if rows == "many" else \
        fused_linear(one, v[:, None], activation="gelu")[0]
    z = v.double()
    want = 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if dtype == torch.float32:
        rel = 2.0 ** -21 + z * z * 2.0 ** -23
    else:
        rel = torch.where(z >= -5.75, 2.0 ** -14, 2.0 ** -10)
    within(y, want, rel * want.abs(), "y")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_positive_side_and_ends(dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    v = -_sweep(dtype, cuda_device)
    v = torch.cat([v, torch.tensor([0.0, -0.0, 100.0, 6e4, -13.5, -14.0, -20.0, -100.0, -6e4], device=cuda_device).to(dtype)])
    y = fused_linear(v[:, None], torch.ones(1, 1, dtype=dtype, device=cuda_device), activation="gelu")[:, 0]
    z = v.double()
    want = 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    within(y, want, 2.0 ** -14 * want.abs() if dtype != torch.float32 else 2.0 ** -21 * want.abs(), "y")


def test_fp32_slope(cuda_device):
    """Phi(z) + z phi(z): each term to a few units and the argument's roundings, their sum once more."""
    from wayfinder_attention_b200 import fused_linear

    x = _sweep(torch.float32, cuda_device)[:, None].requires_grad_()
    w = torch.ones(1, 1, device=cuda_device)
    dx, = torch.autograd.grad(fused_linear(x, w, activation="gelu").sum(), x)
    z = x.detach().double()
    phi, density = 0.5 * torch.special.erfc(-z / math.sqrt(2)), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    within(dx, phi + density, (2.0 ** -21 + z * z * 2.0 ** -23) * (phi + density.abs()), "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", ["many", "one"])
def test_not_finite(rows, dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    v = torch.full((40,), 0.5, dtype=dtype, device=cuda_device)
    v[3], v[7], v[9] = math.inf, -math.inf, math.nan
    one = torch.ones(1, 1, dtype=dtype, device=cuda_device)
    y = fused_linear(v[:, None], one, activation="gelu")[:, 0] if rows == "many" else \
        fused_linear(one, v[:, None], activation="gelu")[0]
    assert y[3] == math.inf and y[7] == 0 and torch.isnan(y[9]) and torch.isfinite(y[10:]).all()
