"""relu on inputs of ordinary values, over few rows and many.

The slope jumps where z crosses 0, and a z within the sum's own error of 0 may fall on either
side; its sign is then the one that y shows.  Everything else of y and of the gradients is
held to rounding: dz is dy or 0 exactly, each output is a sum of products, rounded once.
Bounds: a sum over K products in fp32 is off by at most (K + 8) 2^-23 sum |a b|.
"""

import pytest
import torch

from dense_utils import ROUNDOFF, TYPES, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [
    (1, 1024, 256), (2, 777, 130), (4, 4096, 64), (7, 2056, 509), (8, 909, 1252), (12, 2048, 128),
    (15, 3000, 256), (16, 3776, 320), (17, 1021, 72), (89, 128, 1280), (700, 384, 704), (2000, 250, 65),
])
def test_random_inputs(M, N, K, dtype, cuda_device):
    from wayfinder_attention_b200 import fused_linear

    for seed in range(3):
        g = torch.Generator(device=cuda_device).manual_seed(seed * 1000 + M)
        draw = lambda *s, scale=1.0: (torch.randn(*s, device=cuda_device, generator=g) * scale).to(dtype)  # noqa: E731
        x, w, b = draw(M, K), draw(N, K, scale=K ** -0.5), draw(N, scale=0.1)
        dy = draw(M, N, scale=0.1)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        y = fused_linear(*leaves, activation="relu")
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        X, W, DY = x.detach().double(), w.detach().double(), dy.double()
        z = X @ W.T + b.detach().double()
        off = (K + 8) * 2.0 ** -23 * (X.abs() @ W.abs().T + b.detach().double().abs())
        within(y, z.clamp_min(0), off, "y")
        # fp16's smallest step can hide a positive z from y, which is why y alone does not decide
        doubtful = z.abs() <= off
        assert torch.equal((y > 0)[~doubtful & (z.abs() > 1e-7)], (z > 0)[~doubtful & (z.abs() > 1e-7)])
        open_ = torch.where(doubtful, y > 0, z > 0)
        # z = 0 passes nothing; a doubtful z whose y is 0 passed dy only if fp16 lost it
        dz = DY * open_
        slack = torch.where(doubtful & (y == 0) & (z > -off), DY.abs() * (dtype == torch.float16), 0.0)
        for what, got, want, more, depth in (
                ("dx", dx, dz @ W, slack @ W.abs(), (N + 8) * 2.0 ** -23 * (dz.abs() @ W.abs())),
                ("dw", dw, dz.T @ X, slack.T @ X.abs(), (M + 8) * 2.0 ** -23 * (dz.abs().T @ X.abs())),
                ("db", db, dz.sum(0), slack.sum(0), (M + 8) * 2.0 ** -23 * dz.abs().sum(0))):
            within(got, want, more + depth, f"{what}, seed {seed}")
            if not slack.any() and want.numel() >= 1024:
                # together: rounded once, nothing else
                once = ROUNDOFF[dtype] * want.norm() + 2.0 ** -22 * want.norm()
                assert (got.double() - want).norm() <= once, f"{what}, seed {seed}"
