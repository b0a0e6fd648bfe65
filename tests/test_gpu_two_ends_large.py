"""token_embedding and linear_token_logprobs where offsets pass 2^31, and where calls overlap."""

import math

import pytest
import torch

from dense_utils import ROUNDOFF, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free_memory():
    yield
    torch.cuda.empty_cache()


def test_embedding_rows_and_gradients_past_2_31(cuda_device):
    """y and dy of 2.2e9 elements: rows at their ends are copies, sums over whole tables are exact (small integers)."""
    from wayfinder_attention_b200 import token_embedding

    n, d, V = 66000, 33024, 90
    w = torch.randint(-8, 9, (V, d), device=cuda_device).bfloat16().requires_grad_()
    tokens = torch.randint(0, V, (n,), device=cuda_device)
    y = token_embedding(tokens, w)
    for lo in (0, n // 2, n - 300):
        assert torch.equal(y[lo:lo + 300], w[tokens[lo:lo + 300]])
    dy = torch.ones((), device=cuda_device, dtype=torch.bfloat16).expand(n, d).contiguous()
    dy[-1] = 3.0
    dw, = torch.autograd.grad(y, [w], dy)
    count = torch.bincount(tokens, minlength=V).double()
    count[tokens[-1]] += 2
    within(dw, count[:, None].expand(V, d), torch.zeros(1), "dweight")


def test_embedding_table_past_2_31(cuda_device):
    from wayfinder_attention_b200 import token_embedding

    V, d = 70000, 32768
    w = torch.zeros(V, d, device=cuda_device, dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, 65535, 65536, V - 2, V - 1], device=cuda_device)
    w[rows] = torch.randn(6, d, device=cuda_device).bfloat16()
    w.requires_grad_()
    tokens = torch.cat([rows, rows[:3]])
    y = token_embedding(tokens, w)
    assert torch.equal(y, w[tokens])
    dy = torch.randn(9, d, device=cuda_device).bfloat16()
    dw, = torch.autograd.grad(y, [w], dy)
    within(dw[rows[3:]], dy[3:6], torch.zeros(1), "rows with one token")
    two = dy[:3].double() + dy[6:].double()
    within(dw[rows[:3]], two, 2.0 ** -23 * two.abs(), "rows with two")
    dw[rows] = 0
    assert not dw.any()


@pytest.mark.parametrize("rows", [8, 70])
def test_weight_past_2_31(rows, cuda_device):
    """1.1 million rows of 2048: log probabilities, and the gradients of the weight's first and last rows."""
    from wayfinder_attention_b200 import linear_token_logprobs

    V, d = 1_100_000, 2048
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    w = torch.empty(V, d, device=cuda_device, dtype=torch.bfloat16)
    for lo in range(0, V, 100_000):
        w[lo:lo + 100_000] = torch.randn(min(100_000, V - lo), d, generator=g, device=cuda_device) * d ** -0.5
    x = torch.randn(rows, d, generator=g, device=cuda_device).bfloat16()
    tokens = torch.randint(0, V, (rows,), generator=g, device=cuda_device)
    tokens[0], tokens[1] = V - 1, 0
    z = torch.cat([x.double() @ w[lo:lo + 100_000].double().T for lo in range(0, V, 100_000)], 1)
    lse = torch.logsumexp(z, 1)
    lp = z.gather(1, tokens[:, None])[:, 0] - lse
    ez = (d + 8) * 2.0 ** -23 * x.abs().double().sum(1) * w[:1000].abs().amax().item() * 1.3  # over any one logit's terms
    w.requires_grad_()
    x.requires_grad_()
    r = linear_token_logprobs(x, w, tokens)
    within(r.logprob, lp, 2 * ez + 2.0 ** -19 * 32, "logprob")
    gl = torch.randn(rows, generator=g, device=cuda_device)
    dx, dw = torch.autograd.grad(r.logprob, [x, w], gl)
    u = ROUNDOFF[torch.bfloat16]
    X, p = x.detach().double(), torch.exp(z - lse[:, None])
    for part in (slice(0, 300), slice(V - 300, V)):
        ids = torch.arange(V, device=cuda_device)[part]
        dz = gl[:, None].double() * ((tokens[:, None] == ids).double() - p[:, part])
        off = (u + 1e-4) * dz.abs() + 1e-7 * p[:, part]
        within(dw[part], dz.T @ X, off.T @ X.abs(), "dweight")
    dz = -gl[:, None].double() * p
    dz.scatter_add_(1, tokens[:, None], gl[:, None].double())
    with torch.no_grad():
        want = sum(dz[:, lo:lo + 100_000] @ w[lo:lo + 100_000].double() for lo in range(0, V, 100_000))
        size = sum(dz[:, lo:lo + 100_000].abs() @ w[lo:lo + 100_000].double().abs() for lo in range(0, V, 100_000))
    within(dx, want, (u + 2e-4) * size, "dx")


def test_rows_past_2_31(cuda_device):
    """1.1 million rows over 2100 tokens: the logits' gradients of one piece have 2.3e9 elements."""
    from wayfinder_attention_b200 import linear_token_logprobs

    rows, V, d = 1_100_000, 2100, 16
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn(rows, d, generator=g, device=cuda_device).bfloat16().requires_grad_()
    w = torch.randn(V, d, generator=g, device=cuda_device).bfloat16().requires_grad_()
    tokens = torch.randint(0, V, (rows,), generator=g, device=cuda_device)
    r = linear_token_logprobs(x, w, tokens)
    dx, dw = torch.autograd.grad(r.logprob.sum(), [x, w])
    X, W, u = x.detach().double(), w.detach().double(), ROUNDOFF[torch.bfloat16]
    want = torch.zeros(V, d, dtype=torch.float64, device=cuda_device)
    size = torch.zeros_like(want)
    for lo in range(0, rows, 50_000):
        xs, ts = X[lo:lo + 50_000], tokens[lo:lo + 50_000]
        z = xs @ W.T
        lse = torch.logsumexp(z, 1, keepdim=True)
        dz = -torch.exp(z - lse)
        dz.scatter_add_(1, ts[:, None], torch.ones_like(lse))
        want += dz.T @ xs
        size += dz.abs().T @ xs.abs()
        if lo in (0, 1_050_000):
            within(r.logprob[lo:lo + 50_000], (z.gather(1, ts[:, None]) - lse)[:, 0], torch.tensor(2.0 ** -17), "logprob")
            within(dx[lo:lo + 50_000], dz @ W, (u + 1e-4) * (dz.abs() @ W.abs()), "dx")
    # sums of a million rows in fp32, by tiles: (rows + 8) 2^-23 at most of the sizes, and dz's rounding
    within(dw, want, (u + (rows + 8) * 2.0 ** -23) * size, "dweight")


def test_calls_that_overlap(cuda_device):
    """Two streams at once, each with its own tensors, give what they give alone."""
    from wayfinder_attention_b200 import linear_token_logprobs, token_embedding

    g = torch.Generator(device=cuda_device).manual_seed(2)

    def case(rows, V, d):
        w = (torch.randn(V, d, generator=g, device=cuda_device) * d ** -0.5).bfloat16()
        return w, torch.randint(0, V, (rows,), generator=g, device=cuda_device)

    def step(w, tokens):
        leaf = w.detach().requires_grad_()
        h = token_embedding(tokens, leaf, scale=4.0)
        r = linear_token_logprobs(h, leaf, tokens.roll(-1))
        return r.logprob.detach(), *torch.autograd.grad(r.logprob.mean() + r.entropy.mean(), [leaf])

    cases = [case(4000, 3000, 128), case(50, 20000, 256), case(20000, 200, 64), case(3000, 9000, 72)]
    alone = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        together = []
        for c, s in zip(cases, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                together.append(step(*c))
        torch.cuda.synchronize()
        for a, b in zip(alone, together):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_tables_that_nothing_counts_for(cuda_device):
    """All tokens are padding, or outside: zeros throughout, whatever the memory held."""
    from wayfinder_attention_b200 import check_status, token_embedding

    for n, V in ((5, 40), (9000, 70000), (70000, 300)):
        w, pw = (torch.randn(k, 24, device=cuda_device, requires_grad=True) for k in (V, 3))
        held = torch.full((1 << 24,), math.nan, device=cuda_device)
        del held
        y = token_embedding(torch.full((n,), 7, device=cuda_device), w, padding_index=7)
        dw, = torch.autograd.grad(y.sum(), [w])
        assert not dw.any()
        bad = torch.full((n,), V, device=cuda_device)
        y = token_embedding(bad, w, position_weight=pw, positions=bad)
        assert not any(t.any() for t in torch.autograd.grad(y.sum(), [w, pw]))
        with pytest.raises(RuntimeError, match="out of range"):
            check_status()
