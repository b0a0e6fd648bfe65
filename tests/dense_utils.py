"""Shared by the tests of the decoder's dense operators: unit roundoffs and bound checks."""

import torch

# the largest relative error of one rounding to the type
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# fp16's smallest steps: a result below 2^-14 is off by up to 2^-25 however small it is
UNDERFLOW = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """Elementwise |got - want| <= bound + one rounding of want to got's type; NaN and infinities in the same places."""
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, wanted {tuple(want.shape)}"
    dt, got, want = got.dtype, got.detach().double().cpu(), want.double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), f"{what}: finite in other places"
    assert torch.equal(torch.isnan(want), torch.isnan(got)), f"{what}: NaN in other places"
    assert torch.equal(want[~finite & ~torch.isnan(want)], got[~finite & ~torch.isnan(want)]), f"{what}: infinities"
    limit = bound.double().cpu().expand_as(want) + ROUNDOFF[dt] * (want.abs() + bound.double().cpu()) + UNDERFLOW[dt]
    over = ((got - want).abs() - limit)[finite]
    assert over.numel() == 0 or over.max().item() <= 0, (
        f"{what}: {int((over > 0).sum())} of {over.numel()} outside their bound, by up to {over.max().item():.3g}")
