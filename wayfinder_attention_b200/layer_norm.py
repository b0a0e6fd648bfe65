"""Layer norm over the last axis, with its backward (``wf_layer_norm``).

What the decoder's ``nn.LayerNorm`` computes (``routing_attention/models/transformer.py:26-72``):
one pass over the rows each way, statistics in fp32, and the weight's and bias's
gradients reduced in a fixed order.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib


@functools.lru_cache(maxsize=4096)
def _backward_workspace_bytes(rows: int, d: int, dtype: int) -> int:
    return _lib.load_library().wf_layer_norm_backward_workspace_bytes(rows, d, dtype)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _launch(x, weight, bias, eps, param_dtype, keep_stats, shape):
    dev = x.device
    rows, d = x.shape
    y = x.new_empty(shape)
    stats = torch.empty(2, rows, dtype=torch.float32, device=dev) if keep_stats else None
    at = stats.data_ptr() if keep_stats else None
    with _lib.on_device(dev):
        rc = _lib.load_library().wf_layer_norm(
            x.data_ptr(), _lib.dtype_code(x.dtype), rows, d, x.stride(0), _ptr(weight), _ptr(bias),
            _lib.dtype_code(param_dtype), eps, y.data_ptr(), d, at, at + 4 * rows if keep_stats else None,
            _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    return y, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, param_dtype):
        x2 = _lib.rows_of(x)
        y, stats = _launch(x2, weight, bias, eps, param_dtype, True, x.shape)
        ctx.save_for_backward(x2, weight, stats)
        ctx.param_dtype = param_dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _, _ = ctx.needs_input_grad
        rows, d = x.shape
        dev = x.device
        g = _lib.rows_of(dy)
        dx = x.new_empty(dy.shape) if need_x else None
        dw = torch.empty(d, dtype=ctx.param_dtype, device=dev) if need_w else None
        db = torch.empty(d, dtype=ctx.param_dtype, device=dev) if need_b else None
        code = _lib.dtype_code(x.dtype)
        n = _backward_workspace_bytes(rows, d, code) if need_w or need_b else 0
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        at = stats.data_ptr()
        with _lib.on_device(dev):
            rc = _lib.load_library().wf_layer_norm_backward(
                x.data_ptr(), g.data_ptr(), code, rows, d, x.stride(0), g.stride(0), _ptr(weight),
                _lib.dtype_code(ctx.param_dtype), at, at + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n,
                _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc)
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, rounded once.

    x: (..., d) CUDA tensor of bfloat16, float16 or float32; weight and bias: (d,), both of
    x's type or both float32, or None.  Differentiable in x, weight and bias.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected x (..., d) with d >= 1, got {tuple(x.shape)}")
    if eps < 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    tensors, param_dtype, need_grad = [x], x.dtype, x.requires_grad
    for p in (weight, bias):
        if p is not None:
            if p.shape != x.shape[-1:]:
                raise ValueError(f"weight and bias must be ({x.shape[-1]},), got {tuple(p.shape)}")
            if p.dtype not in (x.dtype, torch.float32) or (len(tensors) > 1 and p.dtype != param_dtype):
                raise ValueError(f"weight and bias must both be {x.dtype} or float32, got {p.dtype}")
            param_dtype = p.dtype
            need_grad = need_grad or p.requires_grad
            tensors.append(p)
    _lib.require_cuda(*tensors)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if need_grad and torch.is_grad_enabled():
        return _LayerNormFunction.apply(x, weight, bias, eps, param_dtype)
    y, _ = _launch(_lib.rows_of(x), weight, bias, eps, param_dtype, False, x.shape)
    return y
