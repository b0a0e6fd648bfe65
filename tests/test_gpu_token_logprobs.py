"""token_logprobs against its definition in 64 bits: values, entropy, alternatives with ties, masks, gradients.

Bounds.  Differences to the row's maximum and the log of the sum are off by a few
2^-24 (|lp| + log V); 2^-19 (1 + |lp| + log V) leaves room for the sum's length.  The
gradient's factors carry the same relative error, and dlogits is rounded once.
Alternatives are compared exactly: they are the lowest indices of the largest logits.
"""

import math

import pytest
import torch

from dense_utils import TYPES, within

pytestmark = pytest.mark.gpu


def _want(x, tokens, top_n, gl=None, gh=None, ignore=-100):
    """Rows of any mask; x in its own type on the CPU."""
    x = x.double()
    rows, V = x.shape
    none = (x == -math.inf).all(1)
    most = x.amax(1, keepdim=True)
    lp = x - most  # apart from the log of the sum: x = -3e38 leaves no bits for it
    lp = lp - torch.log(lp.exp().sum(1, keepdim=True))
    p = lp.exp()
    H = torch.special.entr(p).sum(1)
    lp[none], p[none], H[none] = -math.inf, 0.0, 0.0
    e = 2.0 ** -19 * (1 + math.log(V) + torch.where(torch.isfinite(lp), lp.abs(), 0.0))
    kept = tokens != ignore
    at = tokens.clamp(0, V - 1)
    logprob = torch.where(kept, lp.gather(1, at[:, None])[:, 0], 0.0)
    logprob[kept & ((tokens < 0) | (tokens >= V))] = math.nan
    out = {"logprob": (logprob, e.gather(1, at[:, None])[:, 0]), "entropy": (H, torch.tensor(2.0 ** -19 * (1 + math.log(V)) ** 2))}
    if top_n:
        order = torch.sort(torch.where(torch.isnan(x), math.inf, x), dim=1, descending=True, stable=True).indices
        out["top_tokens"] = order[:, :top_n]
        out["top_logprobs"] = (lp.gather(1, out["top_tokens"]), e.gather(1, out["top_tokens"]))
    if gl is not None:
        gl = torch.where(kept, gl.double(), 0.0)
        q = torch.where(p > 0, lp, 0.0) + H[:, None]
        d = -p * (gl[:, None] + gh.double()[:, None] * q)
        size = p * (gl.abs()[:, None] + gh.double().abs()[:, None] * (q.abs() + 1))
        one = torch.zeros_like(d).scatter_(1, at[:, None], gl[:, None])
        d = torch.where(none[:, None], 0.0, d + one)
        out["dlogits"] = (d, 4 * e * size + 2.0 ** -22 * one.abs())
    return out


def _check(x, tokens, top_n, dev, grad=True):
    from wayfinder_attention_b200 import token_logprobs

    want = _want(x, tokens, top_n)
    r = token_logprobs(x.to(dev), tokens.to(dev), top_n=top_n)
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32
    assert r.top_tokens.dtype == torch.int64 and r.top_tokens.shape == (*tokens.shape, top_n)
    within(r.logprob, *want["logprob"], "logprob")
    within(r.entropy, *want["entropy"], "entropy")
    if top_n:
        assert torch.equal(r.top_tokens.cpu(), want["top_tokens"])
        within(r.top_logprobs, *want["top_logprobs"], "top_logprobs")
    if not grad:
        return
    g = torch.Generator().manual_seed(1)
    gl, gh = torch.randn(len(tokens), generator=g), torch.randn(len(tokens), generator=g)
    leaf = x.to(dev).requires_grad_()
    r2 = token_logprobs(leaf, tokens.to(dev), top_n=top_n)
    assert torch.equal(r2.logprob, r.logprob) or torch.isnan(r.logprob).any()
    zero = torch.zeros_like(gl)
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        outs = [o for o, w in ((r2.logprob, a), (r2.entropy, b)) if w is not None]
        dx, = torch.autograd.grad(outs, [leaf], [w.to(dev) for w in (a, b) if w is not None], retain_graph=True)
        assert dx.dtype == x.dtype
        within(dx, *_want(x, tokens, 0, zero if a is None else a, zero if b is None else b)["dlogits"], "dlogits")


def _logits(rows, V, dtype, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, V, (rows,), generator=g)
    if rows > 3:
        tokens[2] = -100
    return (torch.randn(rows, V, generator=g) * scale).to(dtype), tokens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,top_n", [
    (1, 1, 1), (1, 2, 2), (3, 5, 0), (7, 31, 31), (9, 33, 32), (1, 128, 5), (300, 128, 3), (20, 255, 8), (11, 257, 1),
    (5, 1000, 20), (5, 1024, 32), (5, 1025, 20), (40, 4099, 5), (3, 32768, 32), (1, 50001, 1), (700, 1500, 4),
    (2, 131072, 32), (160, 9000, 0),
])
def test_sizes(rows, V, top_n, dtype, cuda_device):
    x, tokens = _logits(rows, V, dtype, rows + V)
    _check(x, tokens, top_n, cuda_device)


@pytest.mark.parametrize("V", [60, 900, 5000, 40000])
def test_ties_and_orders(V, cuda_device):
    """Equal logits everywhere, few distinct values, ascending and descending rows, both zeros."""
    g = torch.Generator().manual_seed(V)
    x = torch.stack([
        torch.zeros(V),
        torch.randint(0, 3, (V,), generator=g).float(),
        torch.arange(V).float() / V * 8,
        -torch.arange(V).float() / V * 8,
        torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0),
        torch.cat([torch.full((V - 40,), -1.0), torch.full((40,), 2.0)]),
    ])
    for dtype in TYPES:
        _check(x.to(dtype), torch.arange(6), 32, cuda_device)
        _check(x.to(dtype), torch.arange(6), 5, cuda_device, grad=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 1000, 7001, 60000])
def test_banned_tokens(V, dtype, cuda_device):
    """-inf logits: a share of the row, all but one, all of it, and the given token among them; the type's lowest value too."""
    x, tokens = _logits(8, V, dtype, V)
    tokens[2] = 3
    g = torch.Generator().manual_seed(2)
    x[0, torch.rand(V, generator=g) < 0.5] = -math.inf
    x[1] = -math.inf
    x[1, V // 2] = 1.5
    x[2] = -math.inf
    x[3, tokens[3]] = -math.inf
    x[4, : V // 2] = torch.finfo(dtype).min
    x[5, :-2] = -math.inf
    _check(x, tokens, min(V, 20), cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 3000, 30000])
def test_large_and_special_logits(V, dtype, cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    x, tokens = _logits(5, V, dtype, V, scale=1.0)
    x[0] += 300.0
    x[1] -= 300.0
    x[2] *= 60
    x[3] = torch.finfo(dtype).min
    _check(x, tokens, 4, cuda_device)
    x[1, 7] = math.nan
    x[1, 3] = -math.nan
    x[2, 9] = math.inf
    r = token_logprobs(x.to(cuda_device), tokens.to(cuda_device), top_n=3)
    assert torch.isnan(r.logprob[1]) and torch.isnan(r.entropy[1])
    assert r.top_tokens[1, :2].tolist() == [3, 7] and torch.isnan(r.top_logprobs[1]).all()
    assert r.top_tokens[2, 0].item() == 9 and torch.isnan(r.entropy[2])
    assert torch.isfinite(r.logprob[[0, 3, 4]]).all()


def test_strides_leading_axes_and_empty(cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    g = torch.Generator().manual_seed(4)
    for dtype in TYPES:
        for V in (200, 2500):
            wide = torch.randn(3, 4, V + 30, generator=g).to(dtype)
            tokens = torch.randint(0, V, (3, 4), generator=g)
            for lo in (0, 1, 8, 13):
                x = wide[..., lo:lo + V]
                leaf = wide.to(cuda_device).requires_grad_()
                r = token_logprobs(leaf[..., lo:lo + V], tokens.to(cuda_device, torch.int32), top_n=2)
                gl = torch.randn(12, generator=g)
                want = _want(x.reshape(12, V), tokens.reshape(12), 2, gl, torch.zeros(12))
                within(r.logprob.reshape(12), *want["logprob"], "logprob")
                assert torch.equal(r.top_tokens.reshape(12, 2).cpu(), want["top_tokens"])
                dw, = torch.autograd.grad(r.logprob, [leaf], gl.reshape(3, 4).to(cuda_device))
                within(dw[..., lo:lo + V].reshape(12, V), *want["dlogits"], "dlogits")
                assert not dw[..., :lo].any() and not dw[..., lo + V:].any()
    r = token_logprobs(torch.empty(0, 50, device=cuda_device), torch.empty(0, dtype=torch.int64, device=cuda_device), 3)
    assert r.logprob.shape == (0,) and r.top_tokens.shape == (0, 3)
    r = token_logprobs(torch.zeros(50, device=cuda_device), torch.tensor(4, device=cuda_device))
    assert r.logprob.shape == () and abs(r.logprob.item() + math.log(50)) < 1e-6


def test_gradients_against_differences(cuda_device):
    """Central differences along a random direction, fp32, h = 2^-6 (cubic and rounding terms below 2e-3)."""
    from wayfinder_attention_b200 import token_logprobs

    g = torch.Generator().manual_seed(12)
    for V in (90, 3000):
        x, tokens = _logits(13, V, torch.float32, V)
        gl, gh = torch.randn(13, generator=g), torch.randn(13, generator=g)
        d = torch.randn(13, V, generator=g)
        leaf = x.to(cuda_device).requires_grad_()
        r = token_logprobs(leaf, tokens.to(cuda_device))
        dx, = torch.autograd.grad([r.logprob, r.entropy], [leaf], [gl.to(cuda_device), gh.to(cuda_device)])
        h = 2.0 ** -6
        at = []
        for s in (h, -h):
            q = token_logprobs((x + s * d).to(cuda_device), tokens.to(cuda_device))
            at.append((q.logprob.double().cpu() * gl + q.entropy.double().cpu() * gh).sum())
        slope = (dx.double().cpu() * d).sum()
        assert abs((at[0] - at[1]) / (2 * h) - slope) <= 2e-3 * dx.double().norm().item() * d.norm().item()


def test_tokens_outside_the_vocabulary(cuda_device):
    from wayfinder_attention_b200 import check_status, token_logprobs

    check_status()
    x, _ = _logits(4, 300, torch.float32, 1)
    tokens = torch.tensor([5, 300, -1, -100])
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    r = token_logprobs(x.to(cuda_device), tokens.to(cuda_device), status=status)
    assert torch.isnan(r.logprob[1:3]).all() and r.logprob[3].item() == 0 and torch.isfinite(r.entropy).all()
    assert status.item() == 1
    token_logprobs(x.to(cuda_device), tokens.to(cuda_device))
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()
    r = token_logprobs(x.to(cuda_device), torch.tensor([5, 7, 7, -1]).to(cuda_device), ignore_index=-1)
    assert r.logprob[3].item() == 0 and torch.isfinite(r.logprob).all()
    check_status()


def test_same_bits_on_another_stream(cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    x, tokens = _logits(6, 70000, torch.bfloat16, 3)
    x, tokens = x.to(cuda_device), tokens.to(cuda_device)
    first = token_logprobs(x, tokens, top_n=32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = token_logprobs(x, tokens, top_n=32)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals_on_the_gpu(cuda_device):
    from wayfinder_attention_b200 import token_logprobs

    x, t = torch.zeros(4, 80, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_logprobs(x, t.cpu())
    with pytest.raises(ValueError, match="unsupported dtype"):
        token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="status"):
        token_logprobs(x.requires_grad_(), t, status=torch.zeros(1, dtype=torch.int32, device=cuda_device))
