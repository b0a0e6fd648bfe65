"""What wf_linear asks its caller to allocate."""

from wayfinder_attention_b200 import _lib

BF16, F16, F32 = 0, 1, 2


def test_few_rows_need_none():
    """One launch that streams the weight as it lies: nothing is laid out, split or joined."""
    size = _lib.load_library().wf_linear_workspace_bytes
    for dtype in (BF16, F16, F32):
        for direct in (0, 1):
            assert all(size(M, 4096, 4096, dtype, direct, direct) == 0 for M in (1, 2, 8))
    assert size(9, 4096, 4096, F32, 1, 1) >= 6 * (4096 * 4096 + 9 * 4096)
    assert size(9, 4096, 4095, BF16, 0, 0) >= 2 * 4096 * 4096
