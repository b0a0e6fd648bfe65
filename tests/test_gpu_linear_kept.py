"""The pre-activations that wf_linear keeps for its backward, against 64 bits.

Where y's rows do not start on 16 bytes, y leaves a tile by element stores and the kept
pre-activations by bulk stores, slice after slice through the same staging buffers.

Bounds: a sum over K products in fp32 is off by at most (K + 8) 2^-23 sum |x w|, and what
is kept is rounded once, to fp16 for the 16-bit types and to fp32 for fp32.
"""

import pytest
import torch

from dense_utils import TYPES, within

pytestmark = pytest.mark.gpu

NONE, GELU, SILU = 0, 1, 3


def _kept(x, w, bias, residual, act):
    """(z, y) of one forward through the C ABI."""
    from wayfinder_attention_b200 import _lib

    lib, code = _lib.load_library(), _lib.dtype_code(x.dtype)
    (M, K), N = x.shape, w.shape[0]
    z = torch.full((M, (N + 7) // 8 * 8), float("nan"), device=x.device,
                   dtype=torch.float32 if x.dtype == torch.float32 else torch.float16)
    y = torch.empty(M, N, device=x.device, dtype=x.dtype)
    n = lib.wf_linear_workspace_bytes(M, N, K, code, x.stride(0) * x.element_size() % 16 == 0,
                                      w.stride(0) * w.element_size() % 16 == 0)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=x.device)
    status = torch.zeros(1, dtype=torch.int32, device=x.device)
    _lib.check(lib.wf_linear(x.data_ptr(), w.data_ptr(), bias.data_ptr(),
                             None if residual is None else residual.data_ptr(), code, M, N, K, x.stride(0),
                             w.stride(0), N, act, z.data_ptr(), y.data_ptr(), ws.data_ptr() if n else None, n,
                             status.data_ptr(), _lib.stream_ptr(x.device)))
    assert status.item() == 0
    return z[:, :N], y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,N,K", [
    (300, 1021, 64),     # several tiles and slices, the smallest depth: stores follow one another closely
    (6001, 1021, 64),    # more tiles than SMs
    (20000, 255, 72),
    (1531, 1021, 509),   # operands laid out first
    (130, 1023, 200),    # few tiles
    (3000, 1024, 64),    # rows on 16 bytes: every store is a bulk one
])
def test_kept_values(M, N, K, residual, dtype, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(M + N)
    draw = lambda *s, scale=1.0: (torch.randn(*s, device=cuda_device, generator=g) * scale).to(dtype)  # noqa: E731
    x, w, b = draw(M, K), draw(N, K, scale=K ** -0.5), draw(N, scale=0.1)
    r = draw(M, N) if residual else None
    want = x.double() @ w.double().T + b.double()
    off = (K + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T + b.double().abs())
    for _ in range(3):
        z, y = _kept(x, w, b, r, SILU)
        within(z, want, off, "z")
        a = want * torch.sigmoid(want)
        within(y, a if r is None else a + r.double(), 1.13 * off + 2.0 ** -20 * (1 + want.abs()), "y")
