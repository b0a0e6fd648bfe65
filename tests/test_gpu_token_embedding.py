"""token_embedding against its definition in 64 bits: rows, gradients of both tables, types, sizes, distributions of tokens.

Bounds.  A row is one fp32 multiply-add, rounded once.  A table's row is a sum of L rows of dy in
fp32: off by at most (L + 2) 2^-24 of the sum of their sizes, times the scale, and rounded once.
"""

import math

import pytest
import torch

from dense_utils import TYPES, within

pytestmark = pytest.mark.gpu


def _sums(index, g, rows, scale=1.0):
    """Sums of g's rows by index with their bound; indices outside [0, rows) count nowhere."""
    ok = (index >= 0) & (index < rows)
    index, g = index[ok], g.double()[ok]
    zero = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device)
    want, size = zero.index_add(0, index, g), zero.index_add(0, index, g.abs())
    count = torch.bincount(index, minlength=rows).double()[:, None]
    return want * scale, (count + 2) * 2.0 ** -24 * size * abs(scale)


def _check(tokens, w, pw=None, positions=None, scale=1.0, padding=None, seed=0):
    from wayfinder_attention_b200 import token_embedding

    dev, dtype = w.device, w.dtype
    kw = dict(scale=scale, positions=positions, padding_index=padding)
    t = torch.full((1 << 24,), math.nan, device=dev)  # what the allocator hands out next holds NaN
    del t
    y = token_embedding(tokens, w, position_weight=pw, **kw)
    assert y.dtype == dtype and y.shape == (*tokens.shape, w.shape[1]) and y.is_contiguous()
    flat = tokens.reshape(-1).long()
    want, place = w.double()[flat] * scale, None
    size = want.abs()
    if pw is not None:
        place = torch.arange(tokens.shape[-1] if tokens.dim() else 1, device=dev) if positions is None else positions.long()
        place = (place.expand(tokens.shape) if tokens.dim() else place).reshape(-1)
        want = want + pw.double()[place]
        size = size + pw.double()[place].abs()
    within(y.reshape(want.shape), want, 2.0 ** -23 * size, "y")
    g = torch.Generator(device=dev).manual_seed(seed)
    dy = torch.randn(y.shape, generator=g, device=dev).to(dtype)
    leaves = [x.detach().clone().requires_grad_() for x in (w, pw) if x is not None]
    y2 = token_embedding(tokens, leaves[0], position_weight=leaves[1] if pw is not None else None, **kw)
    assert torch.equal(y2, y)
    grads = torch.autograd.grad(y2, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y2, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    rows = dy.reshape(flat.numel(), -1)
    counted = torch.where(flat == padding, -1, flat) if padding is not None else flat
    within(grads[0], *_sums(counted, rows, w.shape[0], scale), "dweight")
    if padding is not None:
        assert not grads[0][padding].any()
    if pw is not None:
        within(grads[1], *_sums(place, rows, pw.shape[0]), "dposition_weight")


def _tables(V, P, d, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + V + d)
    return (torch.randn(V, d, generator=g, device=dev).to(dtype),
            torch.randn(P, d, generator=g, device=dev).to(dtype) if P else None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,V,P,d", [
    ((1,), 1, 0, 1), ((1, 1), 2, 1, 8), ((8, 1), 128, 16, 256), ((3, 7), 5, 9, 33), ((2, 31), 500, 31, 64),
    ((5, 200), 128, 256, 256), ((4, 1000), 3, 1003, 40), ((3, 4097), 50001, 4097, 16), ((2, 3, 700), 511, 700, 130),
    ((1, 8193), 512, 0, 72), ((700, 9), 40, 9, 24), ((9000, 1), 7, 2, 8), ((1, 300), 30, 300, 2056), ((2, 40), 300000, 64, 48),
])
def test_sizes(shape, V, P, d, dtype, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(len(shape) + V)
    w, pw = _tables(V, P, d, dtype, cuda_device)
    tokens = torch.randint(0, V, shape, generator=g, device=cuda_device)
    _check(tokens, w, pw, scale=1.0 if V % 2 else d ** 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["zipf", "all the same", "two", "sorted", "descending", "each once", "last row"])
def test_distributions_of_tokens(kind, dtype, cuda_device):
    """Lists of every length: one row with all tokens, rows that cross many chunks, rows with one token."""
    n, V, d = 20000, 30000, 40
    g = torch.Generator(device=cuda_device).manual_seed(1)
    at = torch.arange(n, device=cuda_device)
    tokens = {
        "zipf": (torch.exp(torch.rand(n, generator=g, device=cuda_device, dtype=torch.float64) * math.log(V)).long() - 1),
        "all the same": torch.full((n,), 77, device=cuda_device),
        "two": torch.where(torch.rand(n, generator=g, device=cuda_device) < 0.3, 5, V - 1),
        "sorted": at // 50, "descending": (n - 1 - at) // 3, "each once": torch.randperm(V, generator=g, device=cuda_device)[:n],
        "last row": torch.where(at % 3 == 0, V - 1, at % 70),
    }[kind]
    w, pw = _tables(V, 200, d, dtype, cuda_device)
    _check(tokens.view(100, 200), w, pw)
    _check(tokens.view(100, 200), w, pw, positions=tokens.view(100, 200) % 200, padding=77 if kind == "all the same" else None)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 4095, 4096, 4097, 8191, 8192, 12289, 300000])
def test_lengths(n, cuda_device):
    """Around a chunk's and a block's edges; more blocks than add up their counts by themselves."""
    g = torch.Generator(device=cuda_device).manual_seed(n)
    for V in (1, 300, 70000):
        w, _ = _tables(V, 0, 16, torch.float32, cuda_device)
        _check(torch.randint(0, V, (n,), generator=g, device=cuda_device), w)


@pytest.mark.parametrize("dtype", TYPES)
def test_positions_padding_and_types_of_ids(dtype, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    w, pw = _tables(90, 64, 56, dtype, cuda_device)
    tokens = torch.randint(0, 90, (6, 50), generator=g, device=cuda_device)
    tokens[:, 40:] = 0
    some = torch.randint(0, 64, (6, 50), generator=g, device=cuda_device)
    _check(tokens, w, pw, padding=0)
    _check(tokens.int(), w, pw, positions=some.int(), padding=0, scale=-3.5)
    _check(tokens, w, pw, positions=some[0], padding=89)
    _check(tokens.t(), w, pw, positions=some.t())  # ids of other strides
    _check(tokens[0, 0], w, pw)  # one token, no axis
    _check(tokens.reshape(2, 3, 50), w, pw)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype, cuda_device):
    from wayfinder_attention_b200 import token_embedding

    g = torch.Generator(device=cuda_device).manual_seed(5)
    wide = torch.randn(60, 100, generator=g, device=cuda_device).to(dtype)
    tokens = torch.randint(0, 60, (4, 30), generator=g, device=cuda_device)
    for lo in (0, 1, 8, 13):
        for d in (64, 37):
            _check(tokens, wide[:, lo:lo + d], wide[20:50, lo:lo + d])
    _check(tokens % 50, wide.t()[:50], wide.t()[40:80])
    _check(tokens, wide[:1].expand(60, 100), wide[:1].expand(30, 100))  # a table of one row for all
    # gradients of any stride: a slice, a broadcast, a transpose
    leaf = wide.clone().requires_grad_()
    y = token_embedding(tokens, leaf)
    dy = torch.randn(4, 30, 200, generator=g, device=cuda_device).to(dtype)
    for grad in (dy[..., 50:150], dy[..., 3:103], dy[:1, :1, :100].expand(4, 30, 100),
                 dy[..., :100].transpose(0, 1).contiguous().transpose(0, 1), dy[:, :1, 7:8].expand(4, 30, 100)):
        got, = torch.autograd.grad(y, [leaf], grad, retain_graph=True)
        within(got, *_sums(tokens.reshape(-1), grad.reshape(120, 100), 60), "dweight")


def test_empty(cuda_device):
    from wayfinder_attention_b200 import token_embedding

    w, pw = (torch.randn(5, 8, device=cuda_device, requires_grad=True) for _ in range(2))
    for shape in ((0,), (3, 0), (0, 4)):
        y = token_embedding(torch.zeros(shape, dtype=torch.int64, device=cuda_device), w, position_weight=pw)
        assert y.shape == (*shape, 8)
        assert not any(t.any() for t in torch.autograd.grad(y.sum(), [w, pw]))


def test_ids_outside_their_tables(cuda_device):
    from wayfinder_attention_b200 import check_status, token_embedding

    check_status()
    w, pw = _tables(30, 8, 24, torch.float32, cuda_device)
    tokens = torch.tensor([3, 30, -1, 2 ** 40, 5, 29], device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    y = token_embedding(tokens, w, status=status)
    bad = torch.tensor([False, True, True, True, False, False], device=cuda_device)
    assert status.item() == 1 and torch.equal(torch.isnan(y).all(1), bad) and torch.equal(y[~bad], w[tokens[~bad]])
    token_embedding(tokens, w)
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()
    # they add nothing to the table's gradient; a position outside its table neither
    leaves = [t.clone().requires_grad_() for t in (w, pw)]
    y = token_embedding(tokens, leaves[0], position_weight=leaves[1], positions=torch.tensor([0, 1, 2, 3, 8, -5], device=cuda_device))
    assert torch.isnan(y[4:]).all()
    dy = torch.randn_like(y)
    dw, dp = torch.autograd.grad(y, leaves, dy)
    within(dw, *_sums(tokens, dy, 30), "dweight")
    within(dp, *_sums(torch.tensor([0, 1, 2, 3, 8, -5], device=cuda_device), dy, 8), "dposition_weight")
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()
    # sequences longer than the table of positions
    y = token_embedding(torch.zeros(2, 12, dtype=torch.int64, device=cuda_device), leaves[0], position_weight=leaves[1])
    assert torch.isnan(y[:, 8:]).all() and torch.isfinite(y[:, :8]).all()
    dp, = torch.autograd.grad(y, [leaves[1]], torch.ones_like(y))
    assert torch.equal(dp, torch.full_like(dp, 2.0))
    with pytest.raises(RuntimeError, match="out of range"):
        check_status()


def test_gradient_against_differences(cuda_device):
    """The operator is linear in its tables: a difference is exact but for fp32 rounding (2^-16 of the sizes)."""
    from wayfinder_attention_b200 import token_embedding

    g = torch.Generator(device=cuda_device).manual_seed(8)
    w, pw = _tables(40, 50, 24, torch.float32, cuda_device)
    tokens = torch.randint(0, 40, (3, 50), generator=g, device=cuda_device)
    leaves = [w.clone().requires_grad_(), pw.clone().requires_grad_()]
    y = token_embedding(tokens, leaves[0], scale=4.0, position_weight=leaves[1])
    dy = torch.randn(y.shape, generator=g, device=cuda_device)
    grads = torch.autograd.grad(y, leaves, dy)
    to = [torch.randn(t.shape, generator=g, device=cuda_device) for t in leaves]
    for i in range(2):
        ts = [t + (to[j] if j == i else 0) for j, t in enumerate((w, pw))]
        moved = token_embedding(tokens, ts[0], scale=4.0, position_weight=ts[1])
        diff = ((moved.double() - y.detach().double()) * dy).sum()
        assert abs(diff - (grads[i].double() * to[i]).sum()) <= 2.0 ** -16 * dy.norm() * moved.norm()


def test_another_stream_a_graph_and_another_thread(cuda_device):
    import threading

    from wayfinder_attention_b200 import token_embedding

    g = torch.Generator(device=cuda_device).manual_seed(9)
    w, pw = _tables(3000, 900, 72, torch.bfloat16, cuda_device)
    tokens = torch.randint(0, 3000, (12, 800), generator=g, device=cuda_device)
    positions = torch.randint(0, 900, (12, 800), generator=g, device=cuda_device)
    dy = torch.randn(12, 800, 72, generator=g, device=cuda_device).bfloat16()

    def step(tokens):
        leaves = [t.detach().requires_grad_() for t in (w, pw)]
        y = token_embedding(tokens, leaves[0], scale=2.0, position_weight=leaves[1], positions=positions)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    first = step(tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step(tokens)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    got = []
    t = threading.Thread(target=lambda: got.append(step(tokens)))
    t.start()
    t.join()
    assert all(torch.equal(a, b) for a, b in zip(first, got[0]))
    static = tokens.clone()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(static)
        graphs.append((graph, out))
    static.copy_(torch.flip(tokens, (1,)))
    for graph, _ in graphs:
        graph.replay()
    want = step(torch.flip(tokens, (1,)))
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_one_sequence_longer_than_the_tokens(cuda_device):
    """Through the C ABI, whose seq is any number: positions 0, 1, ... n - 1."""
    import ctypes

    from wayfinder_attention_b200 import _lib

    w, pw = _tables(30, 50, 16, torch.float32, cuda_device)
    tokens = torch.arange(20, device=cuda_device)
    for seq in (20, 21, 1 << 31, 1 << 32, (1 << 40) + 3):
        y = torch.full((20, 16), math.nan, device=cuda_device)
        at = [ctypes.c_void_p(t.data_ptr()) for t in (tokens, w, pw, y)]
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        rc = _lib.load_library().wf_token_embedding(at[0], 20, at[1], _lib.WF_DTYPE_F32, 30, 16, 16, 1.0, at[2], 50, 16,
                                                    None, seq, at[3], None, stream)
        assert rc == _lib.WF_OK and torch.equal(y, w[:20] + pw[:20]), seq


def test_refusals_on_the_gpu(cuda_device):
    from wayfinder_attention_b200 import token_embedding

    w, t = torch.zeros(4, 8, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_embedding(t.cpu(), w)
    with pytest.raises(ValueError, match="unsupported dtype"):
        token_embedding(t, w.double())
    with pytest.raises(ValueError, match="status"):
        token_embedding(t, w.requires_grad_(), status=torch.zeros(1, dtype=torch.int32, device=cuda_device))
    y = token_embedding(t, w)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = token_embedding(t, w)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), [w], create_graph=True)
