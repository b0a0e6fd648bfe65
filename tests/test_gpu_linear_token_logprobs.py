"""linear_token_logprobs against its definition in 64 bits: values, entropy and gradients, masks, types, sizes, strides.

Bounds.  A logit over d terms, in any order and with truncating adds, is off by at most
ez_j = (d + 8) 2^-23 (sum |x w_j| + |b_j|), so log sum exp by at most E = max_j ez_j, a log
probability by ez_t + E and the entropy by sum_j p_j |ln p_j + H| (ez_j + E).  What is done
with the logits adds e = 2^-19 (1 + |lp| + log V), as for token_logprobs.  The gradient of a
logit carries the relative error of p and is rounded to the type before the products (twice,
so to the square of its roundoff, up to 2^30 multiplications; fp32 to its last bit); fp16's smallest steps are
2^-24 of the largest gradient there.  The products add (terms + 8) 2^-23 of their terms' sizes, and
each output is rounded once.
"""

import math

import pytest
import torch

from dense_utils import ROUNDOFF, TYPES, within

pytestmark = pytest.mark.gpu


def _want(x, w, tokens, b, gl=None, gh=None, ignore=-100):
    """Values with their bounds, in 64 bits, on the inputs' device."""
    dtype, (rows, d), V = x.dtype, x.shape, w.shape[0]
    x, w = x.double(), w.double()
    z, size = x @ w.T, x.abs() @ w.abs().T
    if b is not None:
        z = z + b.double()
        size = size + torch.where(torch.isfinite(b), b.double().abs(), 0.0)
    ez = (d + 8) * 2.0 ** -23 * size
    E = ez.amax(1, keepdim=True)
    none = (z == -math.inf).all(1)
    lp = z - z.amax(1, keepdim=True)
    lp = lp - torch.log(lp.exp().sum(1, keepdim=True))
    lp[none] = -math.inf
    p = torch.where(none[:, None], 0.0, lp.exp())
    H = torch.special.entr(p).sum(1)
    lp0 = torch.where(torch.isfinite(lp), lp, 0.0)
    e = 2.0 ** -19 * (1 + math.log(V) + lp0.abs())
    q = lp0 + H[:, None]
    eH = (p * q.abs() * (ez + E)).sum(1) + 2.0 ** -19 * (1 + math.log(V)) ** 2
    kept = tokens != ignore
    at = tokens.long().clamp(0, V - 1)[:, None]
    logprob = torch.where(kept, lp.gather(1, at)[:, 0], 0.0)
    logprob[kept & ((tokens < 0) | (tokens >= V))] = math.nan
    out = {"logprob": (logprob, (ez + E + e).gather(1, at)[:, 0]), "entropy": (H, eH)}
    if gl is not None:
        gl, gh = torch.where(kept, gl.double(), 0.0)[:, None], gh.double()[:, None]
        dz = -p * (gl + gh * q)
        one = torch.zeros_like(dz).scatter_(1, at, gl)
        rel = 4 * e + ez + E
        off = p * (rel * (gl.abs() + gh.abs() * (q.abs() + 1)) + gh.abs() * (ez + E + eH[:, None])) + 2.0 ** -22 * one.abs()
        dz = torch.where(none[:, None], 0.0, dz + one)
        u = ROUNDOFF[dtype]
        two = dtype != torch.float32 and rows * V * d <= 2 ** 30
        off = off + (2.0 ** -22 if dtype == torch.float32 else 2 * u * u if two else u) * (dz.abs() + off)
        least = (gl.abs() + 32 * gh.abs()).amax() * 2.0 ** -24 if dtype == torch.float16 else 0.0
        off = off + least * 2.0 ** -12
        dza = dz.abs()
        out["dx"] = (dz @ w, off @ w.abs() + (V + 8) * 2.0 ** -23 * (dza @ w.abs()))
        out["dw"] = (dz.T @ x, off.T @ x.abs() + (rows + 8) * 2.0 ** -23 * (dza.T @ x.abs()) + least * rows)
        out["db"] = (dz.sum(0), off.sum(0) + (rows + 8) * 2.0 ** -23 * dza.sum(0))
    return out


def _inputs(rows, V, d, dtype, dev, bias=True, seed=0, spread=2.5):
    g = torch.Generator(device=dev).manual_seed(seed + rows + 7 * V + 31 * d)
    x = torch.randn(rows, d, generator=g, device=dev).to(dtype)
    w = (torch.randn(V, d, generator=g, device=dev) * spread * d ** -0.5).to(dtype)
    b = (torch.randn(V, generator=g, device=dev) * 0.5).to(dtype) if bias else None
    tokens = torch.randint(0, V, (rows,), generator=g, device=dev)
    if rows > 3:
        tokens[2] = -100
    return x, w, b, tokens


def _poison(dev):
    """What the allocator hands out next holds NaN: nothing may read what it did not write."""
    t = torch.full((1 << 26,), math.nan, device=dev)
    del t


def _check(x, w, b, tokens, train=True, scale=1.0):
    from wayfinder_attention_b200 import linear_token_logprobs

    dev = x.device
    _poison(dev)
    r = linear_token_logprobs(x, w, tokens, bias=b)
    assert r.logprob.dtype == r.entropy.dtype == torch.float32 and r.logprob.shape == tokens.shape
    g = torch.Generator(device=dev).manual_seed(1)
    gl, gh = (torch.randn(len(tokens), generator=g, device=dev) * scale for _ in range(2))
    want = _want(x, w, tokens, b, gl, gh)
    within(r.logprob, *want["logprob"], "logprob")
    within(r.entropy, *want["entropy"], "entropy")
    if not train:
        return
    leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
    r2 = linear_token_logprobs(leaves[0], leaves[1], tokens, bias=leaves[2] if b is not None else None)
    assert torch.equal(r2.logprob.nan_to_num(7), r.logprob.nan_to_num(7)) and torch.equal(r2.entropy, r.entropy)
    grads = torch.autograd.grad([r2.logprob, r2.entropy], leaves, [gl, gh])
    for name, leaf, got in zip(("dx", "dw", "db"), leaves, grads):
        assert got.dtype == leaf.dtype and got.is_contiguous()
        within(got, *want[name], name)


SIZES = [
    (1, 1, 1), (1, 2, 8), (1, 128, 256), (3, 5, 7), (7, 300, 64), (130, 257, 72), (300, 1000, 33), (257, 513, 256),
    (1000, 128, 256), (64, 5000, 100), (5, 40000, 48), (700, 3001, 130), (2049, 700, 40), (127, 129, 1), (128, 256, 4096),
    (20, 131072, 16), (4000, 2, 24),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,d", SIZES)
def test_sizes(rows, V, d, dtype, cuda_device):
    _check(*_inputs(rows, V, d, dtype, cuda_device, bias=rows % 2 == 0))


@pytest.mark.parametrize("dtype,rows,V,d", [
    (torch.bfloat16, 16384, 20000, 16), (torch.float16, 16384, 20000, 16),  # one rounding of the logits' gradient
    (torch.bfloat16, 12000, 12000, 6), (torch.float16, 11991, 12001, 7),    # two pieces of it
    (torch.float32, 8193, 7001, 12),
])
def test_pieces_of_the_vocabulary(dtype, rows, V, d, cuda_device):
    """More than 512 MB of gradients of logits: several pieces of the vocabulary, dx summed over them."""
    _check(*_inputs(rows, V, d, dtype, cuda_device))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** 20])
def test_small_and_large_gradients(dtype, scale, cuda_device):
    """A mean over many rows, a loss scaled up: fp16 holds neither p times the one nor the other."""
    if dtype == torch.float16 and scale > 1:
        scale = 2.0 ** 8  # dx is fp16 itself
    for rows, V, d in ((200, 3000, 96), (70, 130, 33)):
        _check(*_inputs(rows, V, d, dtype, cuda_device), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_very_different_gradients(dtype, cuda_device):
    from wayfinder_attention_b200 import linear_token_logprobs

    x, w, b, tokens = _inputs(90, 1000, 64, dtype, cuda_device)
    gl = torch.ones(90, device=cuda_device) * 2.0 ** -torch.arange(90, device=cuda_device).remainder(20).float()
    gl[5], gl[7] = 0.0, 300.0
    gh = torch.zeros(90, device=cuda_device)
    x.requires_grad_()
    w.requires_grad_()
    r = linear_token_logprobs(x, w, tokens, bias=b)
    dx, dw = torch.autograd.grad(r.logprob, [x, w], gl)
    want = _want(x.detach(), w.detach(), tokens, b, gl, gh)
    # each row's dx against its own gradient's size
    within(dw, *want["dw"], "dw")
    for i in (0, 7, 19, 39, 59):
        one = _want(x.detach()[i:i + 1], w.detach(), tokens[i:i + 1], b, gl[i:i + 1], gh[i:i + 1])
        within(dx[i:i + 1], one["dx"][0], one["dx"][1], f"dx of row {i}")
    assert not dx[5].any() and not dx[2].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_one_gradient_are_not_all_off_to_one_side(dtype, cuda_device):
    """A mean's gradients are alike, here half a step of the type above a power of two: rounding dz must not scale them all.

    1024 x 128 -> 16384, past the sizes whose dz is in two pieces.  Off by the token's probability at
    most (6.2e-5 for logits within +-0.6 or so), which rounding 1 - p may lose: t = 2^-13 covers
    it; half a step would be 2^-8 in bf16 and 2^-11 in fp16.  The results' own rounding does not average
    out (dw's rows are x's times 1 + 2^-8, so 8 bits and half a step), but is monotone: a value within
    t of the exact one becomes something between what (1 - t) and (1 + t) times that become.
    """
    from wayfinder_attention_b200 import linear_token_logprobs

    rows, V, d = 1024, 16384, 128
    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = torch.randn(rows, d, generator=g, device=cuda_device).to(dtype).requires_grad_()
    w = (torch.randn(V, d, generator=g, device=cuda_device) * 0.1 * d ** -0.5).to(dtype).requires_grad_()
    b = torch.zeros(V, device=cuda_device, dtype=dtype, requires_grad=True)
    tokens = torch.randint(0, V, (rows,), generator=g, device=cuda_device)
    for size in (1.0, 1e-3):
        gl = torch.full((rows,), -size * (1 + ROUNDOFF[dtype]), device=cuda_device)
        gl[::9] = 0.0
        r = linear_token_logprobs(x, w, tokens, bias=b)
        grads = torch.autograd.grad(r.logprob, [x, w, b], gl)
        X, W = x.detach().double(), w.detach().double()
        dz = -torch.softmax(X @ W.T, 1)
        dz[torch.arange(rows, device=cuda_device), tokens] += 1
        dz *= gl.double()[:, None]
        for name, got, want in zip(("dx", "dw", "db"), grads, (dz @ W, dz.T @ X, dz.sum(0))):
            t = 2.0 ** -13
            low, along, high = (((v.double() * want).sum() / (want * want).sum()).item()
                                for v in ((want * (1 - t)).to(dtype), got, (want * (1 + t)).to(dtype)))
            assert low - t <= along <= high + t, (name, size, low, along, high)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 1000, 7001])
def test_banned_tokens(V, dtype, cuda_device):
    """A bias of -inf: for a share of the tokens, the given one among them, all but one, all."""
    x, w, b, tokens = _inputs(9, V, 40, dtype, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    share = b.clone()
    share[torch.rand(V, generator=g, device=cuda_device) < 0.5] = -math.inf
    share[tokens[0]], share[tokens[1]] = -math.inf, 0.25
    one = torch.full_like(b, -math.inf)
    one[V // 2] = 1.5
    every = torch.full_like(b, -math.inf)
    lowest = b.clone()
    lowest[: V // 2] = torch.finfo(dtype).min
    for bias in (share, one, every, lowest):
        _check(x, w, bias, tokens, train=False)
        from wayfinder_attention_b200 import linear_token_logprobs

        leaves = [t.clone().requires_grad_() for t in (x, w)]
        r = linear_token_logprobs(*leaves, tokens, bias=bias)
        gl, gh = torch.ones(9, device=cuda_device), torch.full((9,), -0.5, device=cuda_device)
        dx, dw = torch.autograd.grad([r.logprob, r.entropy], leaves, [gl, gh])
        want = _want(x, w, tokens, bias, gl, gh)
        within(dx, *want["dx"], "dx")
        within(dw, *want["dw"], "dw")


@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_near_the_ends_of_fp32(dtype, rows, cuda_device):
    """Logits of 8e32, and of -1e38 and 8e32 more, beside banned ones: the largest has all the weight, and nothing becomes NaN."""
    from wayfinder_attention_b200 import linear_token_logprobs

    x = torch.tensor([1e16, -1e16, 1.0, 0.0], device=cuda_device).repeat(rows // 4)[:, None].to(dtype)
    w = (torch.arange(700, device=cuda_device).remainder(50) * 1e14)[:, None].to(dtype)
    w[400], w[200] = 8e16, -8e16
    best = torch.tensor([400, 200, 400, 5], device=cuda_device).repeat(rows // 4)
    for base in (0.0, -1e38):
        b = torch.full((700,), base, device=cuda_device, dtype=dtype)
        b[::3] = -math.inf
        b[[200, 400, 5]] = base
        leaf = x.clone().requires_grad_()
        r = linear_token_logprobs(leaf, w, best, bias=b)
        assert torch.isfinite(r.entropy).all() and torch.isfinite(r.logprob).all()
        sure = torch.arange(rows, device=cuda_device) % 4 < 2
        assert (r.logprob[sure].abs() <= 1e-6).all() and (r.entropy[sure].abs() <= 1e-6).all()
        assert (r.entropy[3::4] - math.log(int(torch.isfinite(b).sum()))).abs().max() <= 1e-4  # equal logits
        dx, = torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), [leaf])
        assert torch.isfinite(dx).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_special_rows(dtype, cuda_device):
    """A NaN row and rows with infinite logits stay by themselves; logits of several hundred."""
    from wayfinder_attention_b200 import linear_token_logprobs

    x, w, b, tokens = _inputs(140, 700, 64, dtype, cuda_device)
    x[9] *= 60
    _check(x, w, b, tokens)
    big = b.clone()
    big[3] = math.inf
    r = linear_token_logprobs(x, w, tokens, bias=big)
    assert torch.isnan(r.entropy).all() and (torch.isnan(r.logprob) | (tokens == -100)).all()
    x[17, 5] = math.nan
    leaf = x.clone().requires_grad_()
    r = linear_token_logprobs(leaf, w, tokens, bias=b)
    others = torch.arange(140, device=cuda_device) != 17
    assert torch.isnan(r.logprob[17]) and torch.isnan(r.entropy[17])
    assert torch.isfinite(r.logprob[others]).all() and torch.isfinite(r.entropy[others]).all()
    dx, = torch.autograd.grad(r.logprob.sum(), [leaf])
    assert torch.isnan(dx[17]).all() and torch.isfinite(dx[others]).all()
    # without a gradient to its row, a NaN stays out of the others'
    dx, = torch.autograd.grad(linear_token_logprobs(leaf, w, tokens, bias=b).logprob[others].sum(), [leaf])
    assert torch.isfinite(dx[others]).all() and not dx[17].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_near_the_ends_of_fp32(dtype, cuda_device):
    """Gradients of 2^127 and of 2^-100 to a row's log probability, past the sizes whose dz is in two pieces.

    x is 2^-20 and the weight 0, so that every distribution is even and nothing else overflows.
    """
    from wayfinder_attention_b200 import linear_token_logprobs

    rows, V, d = 1024, 16384, 80
    x = torch.full((rows, d), 2.0 ** -20, device=cuda_device, dtype=dtype).requires_grad_()
    w = torch.zeros(V, d, device=cuda_device, dtype=dtype).requires_grad_()
    tokens = torch.arange(rows, device=cuda_device)
    for size in (2.0 ** 127, 1.9 * 2.0 ** 126, 2.0 ** -100):
        gl = torch.full((rows,), size, device=cuda_device)
        r = linear_token_logprobs(x, w, tokens)
        dx, dw = torch.autograd.grad(r.logprob, [x, w], gl)
        assert not dx.any()
        # row t of dw: x (1 - 1 / V) of its own row, less x / V of the others
        want = size * 2.0 ** -20 * (1 - rows / V)
        u = ROUNDOFF[dtype]
        assert (dw[:rows].double() / want - 1).abs().max() <= 3 * u + 2.0 ** -13, size
        assert (dw[rows:].double() / (-size * 2.0 ** -20 * rows / V) - 1).abs().max() <= 3 * u + 2.0 ** -13, size


def test_strides_leading_axes_and_empty(cuda_device):
    from wayfinder_attention_b200 import linear_token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda_device)  # noqa: E731
    for dtype in TYPES:
        for d, V in ((64, 200), (50, 333)):
            wide, wwide = rand(3, 5, d + 30).to(dtype), rand(V, d + 30).to(dtype) * 0.3
            tokens = torch.randint(0, V, (3, 5), generator=g, device=cuda_device)
            gl = rand(3, 5)
            for lo in (0, 1, 8, 13):
                leaves = [wide.clone().requires_grad_(), wwide.clone().requires_grad_()]
                r = linear_token_logprobs(leaves[0][..., lo:lo + d], leaves[1][:, lo:lo + d], tokens.int())
                dx, dw = torch.autograd.grad(r.logprob, leaves, gl)
                want = _want(wide[..., lo:lo + d].reshape(15, d), wwide[:, lo:lo + d], tokens.reshape(15), None,
                             gl.reshape(15), torch.zeros(15, device=cuda_device))
                within(r.logprob.reshape(15), *want["logprob"], "logprob")
                within(dx[..., lo:lo + d].reshape(15, d), *want["dx"], "dx")
                within(dw[:, lo:lo + d], *want["dw"], "dw")
                assert not dx[..., :lo].any() and not dw[:, lo + d:].any()
        # a transposed weight, a transposed x, one row of any stride, broadcast rows
        x, w = rand(64, 20).to(dtype).t(), (rand(64, 90) * 0.3).to(dtype).t()
        t = torch.randint(0, 90, (20,), generator=g, device=cuda_device)
        _check(x, w, None, t)
        _check(rand(64, 1).to(dtype).t(), w, None, t[:1])
        _check(rand(1, 64).to(dtype).expand(20, 64), w, None, t)
    x, w = torch.zeros(0, 8, device=cuda_device, requires_grad=True), torch.ones(5, 8, device=cuda_device, requires_grad=True)
    r = linear_token_logprobs(x, w, torch.zeros(0, dtype=torch.int64, device=cuda_device))
    dx, dw = torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), [x, w])
    assert r.logprob.shape == (0,) and dx.shape == (0, 8) and not dw.any()
    r = linear_token_logprobs(torch.zeros(8, device=cuda_device), torch.ones(50, 8, device=cuda_device),
                              torch.tensor(4, device=cuda_device))
    assert r.logprob.shape == () and abs(r.logprob.item() + math.log(50)) < 1e-6


def test_each_gradient_alone(cuda_device):
    """Only x, only the weight, only the bias; only logprob's, only entropy's gradient; no gradient at all from ignored rows."""
    from wayfinder_attention_b200 import linear_token_logprobs

    for dtype in TYPES:
        ts = _inputs(40, 300, 48, dtype, cuda_device)
        x, w, b, tokens = ts
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        r = linear_token_logprobs(leaves[0], leaves[1], tokens, bias=leaves[2])
        both = torch.autograd.grad(r.logprob.sum() - r.entropy.sum(), leaves, retain_graph=True)
        again = torch.autograd.grad(r.logprob.sum() - r.entropy.sum(), leaves, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(both, again))
        for i in range(3):
            args = [leaves[j] if j == i else t for j, t in enumerate((x, w, b))]
            s = linear_token_logprobs(args[0], args[1], tokens, bias=args[2])
            got, = torch.autograd.grad(s.logprob.sum() - s.entropy.sum(), [leaves[i]])
            assert torch.equal(got, both[i])
        zero = torch.zeros(40, device=cuda_device)
        for out, gl, gh in ((r.logprob, zero + 1, zero), (r.entropy, zero, zero + 1)):
            grads = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
            want = _want(x, w, tokens, b, gl, gh)
            for name, got in zip(("dx", "dw", "db"), grads):
                within(got, *want[name], name)
        r = linear_token_logprobs(leaves[0], leaves[1], torch.full_like(tokens, -100), bias=leaves[2])
        assert not r.logprob.any() and torch.isfinite(r.entropy).all()
        assert not any(t.any() for t in torch.autograd.grad(r.logprob.sum(), leaves))


def test_gradients_against_differences(cuda_device):
    """Central differences along a random direction, fp32, h = 2^-6 (cubic and rounding terms below 4e-3)."""
    from wayfinder_attention_b200 import linear_token_logprobs

    g = torch.Generator(device=cuda_device).manual_seed(12)
    for rows, V, d in ((13, 90, 30), (150, 3000, 64)):
        x, w, b, tokens = _inputs(rows, V, d, torch.float32, cuda_device, spread=1.0)
        gl, gh = (torch.randn(rows, generator=g, device=cuda_device) for _ in range(2))
        to = [torch.randn(t.shape, generator=g, device=cuda_device) * s for t, s in ((x, 1.0), (w, d ** -0.5), (b, 1.0))]
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        r = linear_token_logprobs(leaves[0], leaves[1], tokens, bias=leaves[2])
        grads = torch.autograd.grad([r.logprob, r.entropy], leaves, [gl, gh])
        h = 2.0 ** -6
        for i in range(3):
            at = []
            for s in (h, -h):
                ts = [t + s * to[i] if j == i else t for j, t in enumerate((x, w, b))]
                q = linear_token_logprobs(ts[0], ts[1], tokens, bias=ts[2])
                at.append((q.logprob.double() * gl + q.entropy.double() * gh).sum())
            slope = (grads[i].double() * to[i]).sum()
            assert abs((at[0] - at[1]) / (2 * h) - slope) <= 4e-3 * grads[i].double().norm() * to[i].norm(), i


def test_matches_the_logits_operators(cuda_device):
    """fp32: as token_logprobs of the product, to the logits' rounding."""
    from wayfinder_attention_b200 import fused_linear, linear_token_logprobs, token_logprobs

    x, w, b, tokens = _inputs(200, 900, 64, torch.float32, cuda_device)
    r, q = linear_token_logprobs(x, w, tokens, bias=b), token_logprobs(fused_linear(x, w, b), tokens)
    assert (r.logprob - q.logprob).abs().max() <= 1e-5 and (r.entropy - q.entropy).abs().max() <= 1e-5


def test_tokens_outside_the_vocabulary(cuda_device):
    from wayfinder_attention_b200 import check_status, linear_token_logprobs

    check_status()
    x, w, b, _ = _inputs(4, 300, 64, torch.float32, cuda_device)
    tokens = torch.tensor([5, 300, -1, -100], device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    r = linear_token_logprobs(x, w, tokens, bias=b, status=status)
    assert torch.isnan(r.logprob[1:3]).all() and r.logprob[3].item() == 0 and torch.isfinite(r.entropy).all()
    assert status.item() == 1
    linear_token_logprobs(x, w, tokens, bias=b)
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()
    far = torch.tensor([5, 2 ** 40, -2 ** 62, 2 ** 32 + 7], device=cuda_device)
    leaf = x.clone().requires_grad_()
    r = linear_token_logprobs(leaf, w, far, bias=b)
    assert torch.isnan(r.logprob[1:]).all()
    dx, = torch.autograd.grad(r.logprob[:1].sum(), [leaf])
    assert torch.isfinite(dx).all() and dx[0].any() and not dx[1:].any()
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()
    r = linear_token_logprobs(x, w, torch.tensor([5, 7, 7, -1], device=cuda_device), bias=b, ignore_index=-1)
    assert r.logprob[3].item() == 0 and torch.isfinite(r.logprob).all()
    check_status()


def test_another_stream_a_graph_and_another_thread(cuda_device):
    import threading

    from wayfinder_attention_b200 import linear_token_logprobs

    for dtype in TYPES:
        x, w, b, tokens = _inputs(600, 2000, 72, dtype, cuda_device)

        def step(x, w, b, tokens):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            r = linear_token_logprobs(leaves[0], leaves[1], tokens, bias=leaves[2])
            return r.logprob.detach(), r.entropy.detach(), *torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), leaves)

        first = step(x, w, b, tokens)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step(x, w, b, tokens)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, second))
        got = []
        t = threading.Thread(target=lambda: got.append(step(x, w, b, tokens)))
        t.start()
        t.join()
        assert all(torch.equal(p, q) for p, q in zip(first, got[0]))
        static = [t.clone() for t in (x, w, b, tokens)]
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):  # two graphs of the same inputs, replayed in turn
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*static)
            graphs.append((graph, out))
        static[0].copy_(torch.flip(x, (0,)))
        static[3].copy_(torch.flip(tokens, (0,)))
        for graph, _ in graphs:
            graph.replay()
        want = step(torch.flip(x, (0,)), w, b, torch.flip(tokens, (0,)))
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals_on_the_gpu(cuda_device):
    from wayfinder_attention_b200 import linear_token_logprobs

    x, w = torch.zeros(4, 8, device=cuda_device), torch.zeros(80, 8, device=cuda_device)
    t = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_token_logprobs(x, w, t.cpu())
    with pytest.raises(ValueError, match="unsupported dtype"):
        linear_token_logprobs(x.double(), w.double(), t)
    with pytest.raises(ValueError, match="status"):
        linear_token_logprobs(x, w.requires_grad_(), t, status=torch.zeros(1, dtype=torch.int32, device=cuda_device))
    for which in (0, 1, 2):  # changed between forward and backward
        ts = [torch.randn(4, 8, device=cuda_device, requires_grad=True), torch.randn(80, 8, device=cuda_device, requires_grad=True),
              torch.randn(80, device=cuda_device, requires_grad=True)]
        r = linear_token_logprobs(ts[0], ts[1], t, bias=ts[2])
        with torch.no_grad():
            ts[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            r.logprob.sum().backward()
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        linear_token_logprobs(fwAD.make_dual(x, torch.ones_like(x)), w, t)
    x.requires_grad_()
    r = linear_token_logprobs(x, w, t)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(r.logprob.sum(), [x], create_graph=True)
