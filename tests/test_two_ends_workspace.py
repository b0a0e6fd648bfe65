"""The workspace that linear_token_logprobs' documentation states, in every type and alignment."""

import pytest

from wayfinder_attention_b200 import _lib

MB = 1 << 20
SIZES = [(1, 131072, 4096), (16, 50257, 768), (64, 32000, 4096), (512, 128256, 1024), (2048, 32000, 4096),
         (8192, 50257, 768), (8193, 50001, 1001), (32768, 131072, 256), (200000, 32000, 64)]


@pytest.mark.parametrize("dtype", [_lib.WF_DTYPE_BF16, _lib.WF_DTYPE_F16, _lib.WF_DTYPE_F32])
@pytest.mark.parametrize("rows,V,d", SIZES)
@pytest.mark.parametrize("direct", [0, 1])
def test_what_is_stated(rows, V, d, dtype, direct):
    """Laid-out inputs, a piece of dz (dW too in fp16), dx in fp32 and x's copy; 64 MB for sums and shares of products."""
    lib = _lib.load_library()
    f32, padded = dtype == _lib.WF_DTYPE_F32, (d + 7) // 8 * 8
    laid_out = (rows + V) * padded * (6 if f32 else 0 if direct else 2)
    small = 64 * MB
    forward = lib.wf_linear_token_logprobs_workspace_bytes(rows, V, d, dtype, direct, direct)
    # 12 bytes a row, run and warp: 1024 runs of 4 warps at most
    assert laid_out <= forward <= laid_out + small + rows * 12 * 4 * min(1024, 2 + 148 * 128 // rows)
    backward = lib.wf_linear_token_logprobs_backward_workspace_bytes(rows, V, d, dtype, direct, direct)
    column = rows * (10 if f32 else 4 if rows <= 64 or rows * V * d <= 1 << 30 else 2)
    piece = max(512 * MB, 2048 * column)
    dw = max(512 * MB, 2048 * 4 * padded) if dtype == _lib.WF_DTYPE_F16 else 0
    assert laid_out <= backward <= laid_out + min(piece, V * column + 8 * column) + min(dw, (V + 8) * 4 * padded) + small \
        + rows * padded * (4 + 2)
    if f32 and V == 131072 and d == 4096:
        assert 3.2e9 < forward < 3.3e9  # the figure of the documentation
