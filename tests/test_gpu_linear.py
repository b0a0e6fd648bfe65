"""fused_linear against the formulas in 64 bits, in every type, at the sizes where it can go wrong.

Bounds.  A product over K terms in fp32, in any order and with truncating adds, is off by
at most (K + 8) 2^-23 sum |a b|.  The activations' slopes are below 1.13 and their second
derivatives below 0.8; their own evaluation is given 2^-20 (1 + |z|).  The backward reads
z rounded to the type (u |z|), rounds dz to it (u |dz|), and each output is rounded once.
"""

import math

import pytest
import torch

from dense_utils import ROUNDOFF, TYPES, within

pytestmark = pytest.mark.gpu

ACTS = ["none", "gelu", "relu", "silu"]


def _act(name, z):
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    return z, torch.ones_like(z)


def _inputs(M, N, K, dtype, act, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed + M * 7 + N * 3 + K)
    if act == "relu":
        # exact arithmetic, so that z = 0 is 0 for both: eighths, few of them
        draw = lambda *s: torch.randint(-4, 5, s, generator=g).double() / 8  # noqa: E731
        x, w = draw(M, K), draw(N, K)
    else:
        x = torch.randn(M, K, generator=g).double()
        w = torch.randn(N, K, generator=g).double() / K ** 0.5
    b = (torch.randint(-4, 5, (N,), generator=g).double() / 8) if bias else None
    r = torch.randn(M, N, generator=g).double() if residual else None
    dy = torch.randn(M, N, generator=g).double()
    return [None if t is None else t.to(dtype) for t in (x, w, b, r, dy)]


def _check(M, N, K, dtype, act, bias, residual, dev, train=True):
    from wayfinder_attention_b200 import fused_linear

    x, w, b, r, dy = _inputs(M, N, K, dtype, act, bias, residual)
    leaves = [None if t is None else t.to(dev).requires_grad_(train) for t in (x, w, b, r)]
    y = fused_linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    assert y.dtype == dtype
    X, W = x.double(), w.double()
    z = X @ W.T + (0 if b is None else b.double())
    size = X.abs() @ W.abs().T + (0 if b is None else b.double().abs())
    dz_z = (K + 8) * 2.0 ** -23 * size
    a, slope = _act(act, z)
    want = a + (0 if r is None else r.double())
    own = 0 if act in ("none", "relu") else 2.0 ** -20 * (1 + z.abs())
    within(y, want, 1.13 * dz_z + own + 2.0 ** -23 * want.abs(), "y")
    if not train:
        return
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev))))
    u = ROUNDOFF[dtype] if act != "none" else 0.0
    DY = dy.double()
    dz = DY * slope
    off = DY.abs() * (0.0 if act in ("none", "relu") else 0.8 * (u * z.abs() + dz_z) + 2.0 ** -20 * (1 + z.abs()))
    off = off + (u + 2.0 ** -23) * (dz.abs() + off)
    within(grads["dx"], dz @ W, off @ W.abs() + (N + 8) * 2.0 ** -23 * (dz.abs() @ W.abs()), "dx")
    within(grads["dw"], dz.T @ X, off.T @ X.abs() + (M + 8) * 2.0 ** -23 * (dz.abs().T @ X.abs()), "dw")
    if b is not None:
        within(grads["db"], dz.sum(0), off.sum(0) + (M + 8) * 2.0 ** -23 * dz.abs().sum(0), "db")
    if r is not None:
        assert torch.equal(grads["dr"].cpu(), dy)
    # the elementwise bounds add errors up as if they never cancelled; together they do:
    # two or three roundings of relative size u, independent of one another
    ref = {"dx": dz @ W, "dw": dz.T @ X}
    for n, v in ref.items():
        if v.norm() > 0 and v.numel() >= 1024:
            assert (grads[n].double().cpu() - v).norm() <= (3 * ROUNDOFF[dtype] + 2.0 ** -20) * v.norm(), n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [
    (1, 1024, 256),      # one token
    (1, 1, 1),
    (3, 17, 5),
    (8, 512, 320),
    (17, 100, 64),
    (33, 1000, 129),     # odd depth: rows that no 16-byte copy can start on
    (128, 128, 64),      # one tile exactly
    (129, 257, 72),      # one element over in each direction
    (200, 64, 1000),
    (1000, 250, 509),
    (2500, 40, 24),      # few columns, many rows
])
def test_sizes(M, N, K, dtype, cuda_device):
    _check(M, N, K, dtype, "gelu", True, True, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("M", [5, 300])
def test_epilogues(M, act, bias, residual, dtype, cuda_device):
    _check(M, 192, 136, dtype, act, bias, residual, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_depth(dtype, cuda_device):
    """Depths where a running sum has thousands of steps, forward and over the rows in dw."""
    _check(150, 70, 4104, dtype, "none", True, False, cuda_device)
    _check(9000, 136, 72, dtype, "silu", True, False, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_tiles(dtype, cuda_device):
    """More tiles than the GPU has SMs, forward (products alone: compared with torch's in 64 bits on the GPU)."""
    from wayfinder_attention_b200 import fused_linear

    g = torch.Generator(device=cuda_device).manual_seed(3)
    M, N, K = 5000, 2056, 200
    x = torch.randn(M, K, device=cuda_device, generator=g).to(dtype)
    w = (torch.randn(N, K, device=cuda_device, generator=g) / K ** 0.5).to(dtype)
    y = fused_linear(x, w)
    want = x.double() @ w.double().T
    within(y, want, (K + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T), "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 200])
def test_strides_and_leading_axes(rows, dtype, cuda_device):
    """Rows inside wider rows, at offsets of one element; a broadcast residual; a transposed weight; (B, T, d) inputs."""
    from wayfinder_attention_b200 import fused_linear

    g = torch.Generator().manual_seed(11)
    wide = torch.randn(2, rows, 300, generator=g).to(dtype)
    w = torch.randn(96, 200, generator=g).to(dtype) / 14
    r = torch.randn(96, generator=g).to(dtype)
    for lo in (0, 1, 8):
        x = wide[..., lo:lo + 200]
        want = x.double() @ w.double().T + r.double()
        bound = 208 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T) + 2.0 ** -23 * want.abs()
        wd = wide.to(cuda_device)
        for weight in (w.to(cuda_device), w.T.contiguous().to(cuda_device).T):
            y = fused_linear(wd[..., lo:lo + 200], weight, residual=r.to(cuda_device).expand(2, rows, 96))
            within(y, want, bound, f"offset {lo}")
    # gradients of broadcast inputs are summed by whoever expanded them
    xb = torch.randn(200, generator=g).to(dtype).to(cuda_device).requires_grad_()
    rb = r.to(cuda_device).requires_grad_()
    y = fused_linear(xb.expand(rows, 200), w.to(cuda_device), residual=rb.expand(rows, 96))
    dxb, drb = torch.autograd.grad(y.sum(), [xb, rb])
    u = ROUNDOFF[dtype]
    each = w.double().sum(0)
    within(dxb, rows * each, rows * (3 * u * each.abs() + 104 * 2.0 ** -23 * w.double().abs().sum(0))
           + rows ** 2 * u * each.abs(), "dx of a broadcast row")
    within(drb, torch.full((96,), float(rows)), torch.tensor(rows ** 2 * u), "dr of a broadcast row")


def test_empty_and_special_values(cuda_device):
    from wayfinder_attention_b200 import fused_linear

    w = torch.ones(24, 16, device=cuda_device, requires_grad=True)
    b = torch.ones(24, device=cuda_device, requires_grad=True)
    x = torch.empty(0, 16, device=cuda_device, requires_grad=True)
    y = fused_linear(x, w, b, activation="gelu")
    assert y.shape == (0, 24)
    dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    for dtype in TYPES:
        for rows in (3, 150):
            x = torch.zeros(rows, 64, dtype=dtype, device=cuda_device)
            x[1, 3] = float("nan")
            x[2, 5] = float("inf")
            w1 = torch.ones(40, 64, dtype=dtype, device=cuda_device)
            y = fused_linear(x, w1, activation="relu").float().cpu()
            assert torch.isnan(y[1]).all()
            assert not torch.isfinite(y[2]).any()  # inf, or NaN where the type is split for the product
            assert (y[0] == 0).all() and (y[3:] == 0).all()
            big = torch.full((1, 64), -200.0, dtype=dtype, device=cuda_device)
            for act in ("gelu", "silu"):
                assert (fused_linear(big, w1, activation=act) == 0).all()
                assert torch.equal(fused_linear(-big, w1, activation=act), fused_linear(-big, w1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(1, 257, 130), (5, 64, 512), (61, 96, 64), (300, 520, 200), (2047, 24, 72)])
def test_small_gradients_are_rounded_once(M, N, K, act, dtype, cuda_device):
    """dz keeps the bits that its type has no room for.  What is left beside the gradients' own
    rounding is z's (an eleven-bit one: at most 0.4 of it after the slope's derivative, so
    sqrt(1 + 0.16) = 1.08 for fp16); with dz rounded once more it would be sqrt 2."""
    from wayfinder_attention_b200 import fused_linear

    x, w, b, _, dy = _inputs(M, N, K, dtype, act, True, False, seed=3)
    leaves = [t.to(cuda_device).requires_grad_() for t in (x, w)]
    y = fused_linear(leaves[0], leaves[1], b.to(cuda_device), activation=act)
    dz = dy.double() * _act(act, x.double() @ w.double().T + b.double())[1]
    for got, want in zip(torch.autograd.grad(y, leaves, dy.to(cuda_device)), (dz @ w.double(), dz.T @ x.double())):
        once = (want.to(dtype).double() - want).norm()
        assert (got.cpu().double() - want).norm() <= 1.15 * once


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act, cuda_device):
    """Central differences of the operator itself along a random direction, fp32.

    With h = 2^-6 the cubic term is below h^2 |f'''| ~ 2.5e-4 of the direction's own
    size, and fp32 rounding over h below 1e-4 of it: 2e-3 bounds both.  relu has inputs
    whose z stays away from 0 by more than a step moves it.
    """
    from wayfinder_attention_b200 import fused_linear

    g = torch.Generator().manual_seed(21)
    M, N, K = 37, 52, 28
    x, w, b, r = (torch.randn(*s, generator=g) / d for s, d in (((M, K), 1), ((N, K), K ** 0.5), ((N,), 1), ((M, N), 1)))
    v = [torch.randn(t.shape, generator=g) / t.numel() ** 0.5 for t in (x, w, b, r)]
    if act == "relu":
        b = torch.where(torch.arange(N) % 2 == 0, 30.0, -30.0)
    dy = torch.randn(M, N, generator=g)
    dev = [t.to(cuda_device) for t in (x, w, b, r)]
    leaves = [t.clone().requires_grad_() for t in dev]
    y = fused_linear(*leaves[:3], activation=act, residual=leaves[3])
    grads = torch.autograd.grad(y, leaves, dy.to(cuda_device))
    for i, (gr, d) in enumerate(zip(grads, v)):
        h = 2.0 ** -6
        at = []
        for s in (h, -h):
            t = [t0 + s * d.to(cuda_device) if j == i else t0 for j, t0 in enumerate(dev)]
            at.append((fused_linear(*t[:3], activation=act, residual=t[3]).double().cpu() * dy.double()).sum())
        slope = (gr.double().cpu() * d.double()).sum()
        size = gr.double().norm().item() * d.double().norm().item()
        assert abs((at[0] - at[1]) / (2 * h) - slope) <= 2e-3 * size, i


def test_same_bits_twice_and_on_another_stream(cuda_device):
    from wayfinder_attention_b200 import check_status, fused_linear

    x, w, b, r, dy = [t.to(cuda_device) for t in _inputs(3000, 520, 264, torch.bfloat16, "gelu", True, True)]
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = fused_linear(x, w, b, activation="gelu", residual=r)
        return (y, *torch.autograd.grad(y, [x, w, b], dy))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [step() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for o in others:
        assert all(torch.equal(a, c) for a, c in zip(first, o))
    check_status()


def test_refusals_on_the_gpu(cuda_device):
    from wayfinder_attention_b200 import fused_linear

    x, w = torch.zeros(4, 8, device=cuda_device), torch.zeros(6, 8, device=cuda_device)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_linear(x, w.cpu())
    with pytest.raises(ValueError, match="one type"):
        fused_linear(x, w.half())
    with pytest.raises(ValueError, match="unsupported dtype"):
        fused_linear(x.double(), w.double())
    with pytest.raises(ValueError, match="status"):
        fused_linear(x.requires_grad_(), w, status=torch.zeros(1, dtype=torch.int32, device=cuda_device))
