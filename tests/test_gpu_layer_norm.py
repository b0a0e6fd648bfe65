"""layer_norm against its formulas in 64 bits, in every type, at the widths where its form changes.

Bounds.  fp32 statistics of a row whose largest value is k standard deviations (eps
counted in) are off by a few 2^-24 k; 2^-18 k leaves room for the sums' lengths.  Column
sums over R rows add (R + 8) 2^-23 of their absolute terms.  Each output is rounded once.
"""

import pytest
import torch

from dense_utils import TYPES, within

pytestmark = pytest.mark.gpu


def _want(x, w, b, eps, dy):
    x = x.double()
    W = torch.ones(x.shape[1]).double() if w is None else w.double()
    B = torch.zeros(x.shape[1]).double() if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    sd = ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mean) / sd
    k = 1 + x.abs().amax(1, keepdim=True) / sd
    y = h * W + B
    e = 2.0 ** -18 * k  # of h
    out = {"y": (y, e * (1 + h.abs()) * W.abs() + 2.0 ** -23 * B.abs())}
    if dy is not None:
        dy = dy.double()
        g = dy * W
        size = (g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)) / sd
        out["dx"] = ((g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) / sd, e * (1 + h.abs()) * size)
        R = x.shape[0]
        out["dw"] = ((dy * h).sum(0), ((dy.abs() * (1 + h.abs())) * (e + (R + 8) * 2.0 ** -23)).sum(0))
        out["db"] = (dy.sum(0), (R + 8) * 2.0 ** -23 * dy.abs().sum(0))
    return out


def _check(x, w, b, dy, dev, eps=1e-5):
    from wayfinder_attention_b200 import layer_norm

    leaves = [None if t is None else t.to(dev).requires_grad_() for t in (x, w, b)]
    with torch.no_grad():
        y0 = layer_norm(*leaves, eps=eps)
    y = layer_norm(*leaves, eps=eps)
    assert y.dtype == x.dtype and torch.equal(y, y0)
    want = _want(x, w, b, eps, dy)
    within(y, *want["y"], "y")
    names = [n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None]
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev))
    for n, gr in zip(names, grads):
        within(gr, *want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [
    (1, 1), (5, 2), (3, 7), (700, 256), (33, 264), (10, 511), (9, 512), (9, 513), (40, 520), (300, 1001), (17, 1024),
    (6, 2047), (5, 2048), (5, 2056), (7, 4096), (3, 4104), (3, 8192), (2, 8200), (2, 16391), (2, 20000), (3001, 64),
])
def test_sizes(rows, d, dtype, cuda_device):
    g = torch.Generator().manual_seed(rows * 31 + d)
    x = (torch.randn(rows, d, generator=g) * 2 + torch.randn(rows, 1, generator=g)).to(dtype)
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(dtype)
    b = (0.1 * torch.randn(d, generator=g)).to(dtype)
    _check(x, w, b, torch.randn(rows, d, generator=g).to(dtype), cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_w,with_b,f32", [(True, True, True), (True, False, False), (False, True, True),
                                               (False, False, False)])
def test_parameters(dtype, with_w, with_b, f32, cuda_device):
    g = torch.Generator().manual_seed(5)
    for rows, d in ((50, 384), (50, 77)):
        pt = torch.float32 if f32 else dtype
        x = torch.randn(rows, d, generator=g).to(dtype)
        w = (1 + 0.1 * torch.randn(d, generator=g)).to(pt) if with_w else None
        b = (0.1 * torch.randn(d, generator=g)).to(pt) if with_b else None
        _check(x, w, b, torch.randn(rows, d, generator=g).to(dtype), cuda_device, eps=1e-3)


@pytest.mark.parametrize("dtype", TYPES)
def test_hard_rows(dtype, cuda_device):
    """A large mean beside a small spread, constant rows, zeros, one NaN and one infinite row."""
    g = torch.Generator().manual_seed(6)
    for d in (256, 333, 3000):
        x = torch.randn(12, d, generator=g)
        x[0] += 100
        x[1] = 3.0
        x[2] = 0.0
        x[3] *= 1e-4
        x[4] *= 100
        x = x.to(dtype)
        _check(x, None, None, torch.randn(12, d, generator=g).to(dtype), cuda_device)
    from wayfinder_attention_b200 import layer_norm

    x = torch.randn(4, 256, generator=g).to(dtype)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    y = layer_norm(x.to(cuda_device)).cpu()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).any()
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_leading_axes_and_empty(dtype, cuda_device):
    from wayfinder_attention_b200 import layer_norm

    g = torch.Generator().manual_seed(7)
    wide = torch.randn(3, 40, 400, generator=g).to(dtype)
    for lo in (0, 1, 8):
        x = wide[..., lo:lo + 320]
        y = layer_norm(wide.to(cuda_device)[..., lo:lo + 320])
        assert y.shape == x.shape
        want, bound = _want(x.reshape(120, 320), None, None, 1e-5, None)["y"]
        within(y.reshape(120, 320), want, bound, f"offset {lo}")
    t = torch.randn(64, 50, generator=g).to(dtype)
    want, bound = _want(t.T.contiguous(), None, None, 1e-5, None)["y"]
    within(layer_norm(t.to(cuda_device).T), want, bound, "transposed")
    w = torch.ones(320, dtype=dtype, device=cuda_device, requires_grad=True)
    b = torch.ones(320, dtype=dtype, device=cuda_device, requires_grad=True)
    x = torch.empty(0, 320, dtype=dtype, device=cuda_device, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == dx.shape == (0, 320) and not dw.any() and not db.any()
    # one row's gradient broadcast over the rows
    xr = torch.randn(30, 320, generator=g).to(dtype).to(cuda_device).requires_grad_()
    _, db = torch.autograd.grad(layer_norm(xr, w, b).sum(), [xr, b])
    assert torch.equal(db, torch.full_like(db, 30.0))


def test_gradients_against_differences(cuda_device):
    """Central differences along a random direction, fp32, h = 2^-6 (cubic and rounding terms below 2e-3)."""
    from wayfinder_attention_b200 import layer_norm

    g = torch.Generator().manual_seed(8)
    x, w, b = torch.randn(29, 300, generator=g), 1 + 0.1 * torch.randn(300, generator=g), torch.randn(300, generator=g)
    dy = torch.randn(29, 300, generator=g)
    dev = [t.to(cuda_device) for t in (x, w, b)]
    leaves = [t.clone().requires_grad_() for t in dev]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy.to(cuda_device))
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=g)
        d /= d.norm()
        h = 2.0 ** -6
        at = []
        for s in (h, -h):
            t = [t0 + s * d.to(cuda_device) if j == i else t0 for j, t0 in enumerate(dev)]
            at.append((layer_norm(*t).double().cpu() * dy.double()).sum())
        slope = (gr.double().cpu() * d.double()).sum()
        assert abs((at[0] - at[1]) / (2 * h) - slope) <= 2e-3 * gr.double().norm().item(), i


def test_same_bits_twice_and_on_another_stream(cuda_device):
    from wayfinder_attention_b200 import layer_norm

    g = torch.Generator(device=cuda_device).manual_seed(9)
    x = torch.randn(5000, 384, device=cuda_device, generator=g).bfloat16().requires_grad_()
    w = torch.randn(384, device=cuda_device, generator=g).bfloat16().requires_grad_()
    dy = torch.randn(5000, 384, device=cuda_device, generator=g).bfloat16()

    def step():
        y = layer_norm(x, w)
        return (y, *torch.autograd.grad(y, [x, w], dy))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals_on_the_gpu(cuda_device):
    from wayfinder_attention_b200 import layer_norm

    x = torch.zeros(4, 8, device=cuda_device)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="float32"):
        layer_norm(x.half(), torch.ones(8, device=cuda_device, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="unsupported dtype"):
        layer_norm(x.double())
