"""Linear layer with bias, activation and residual in the product's epilogue (``wf_linear``).

The decoder's projections and FFN (``routing_attention/models/transformer.py:26-72``) run
``nn.Linear``, the activation and the residual add as separate layers; ``fused_linear``
is one pass over the product, and differentiable in every input.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "gelu": 1, "relu": 2, "silu": 3}


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.load_library().wf_linear_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _backward_workspace_bytes(*sizes: int) -> int:
    return _lib.load_library().wf_linear_backward_workspace_bytes(*sizes)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _launch(x, weight, bias, residual, act, keep_z, shape, status):
    """y of the given shape (and the pre-activations z when the backward will want them); x and residual as rows."""
    dev = x.device
    M, K = x.shape
    N = weight.shape[0]
    y = x.new_empty(shape)
    z = x.new_empty((M, N)) if keep_z else None
    code = _lib.dtype_code(x.dtype)
    xp, xs, wp, w_stride = x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0)
    size = 4 if code == _lib.WF_DTYPE_F32 else 2
    n = _workspace_bytes(M, N, K, code, (xp | xs * size) & 15 == 0, (wp | w_stride * size) & 15 == 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    st = _lib.status_arg(dev, status)
    with _lib.on_device(dev):
        rc = _lib.load_library().wf_linear(
            xp, wp, _ptr(bias), _ptr(residual), code, M, N, K, xs, w_stride,
            0 if residual is None else residual.stride(0), act, _ptr(z), y.data_ptr(), _ptr(ws), n, st,
            _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    _lib.status_after(dev, status)
    return y, z


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x2, w2 = _lib.rows_of(x), _lib.rows_of(weight)
        r2 = None if residual is None else _lib.rows_of(residual)
        y, z = _launch(x2, w2, bias, r2, act, act != 0, (*x.shape[:-1], w2.shape[0]), None)
        ctx.save_for_backward(x2, w2, z)
        ctx.act, ctx.x_shape = act, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        M, K = x.shape
        N = weight.shape[0]
        dev = x.device
        g = _lib.rows_of(dy)
        dx = x.new_empty(ctx.x_shape) if need_x else None
        dw = x.new_empty((N, K)) if need_w else None
        db = x.new_empty(N) if need_b else None
        if need_x or need_w or need_b:
            code = _lib.dtype_code(x.dtype)
            n = _backward_workspace_bytes(M, N, K, code, ctx.act, _lib.on_16_bytes(x), _lib.on_16_bytes(weight),
                                          _lib.on_16_bytes(g))
            ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            st = _lib.status_arg(dev, None)
            with _lib.on_device(dev):
                rc = _lib.load_library().wf_linear_backward(
                    x.data_ptr(), weight.data_ptr(), _ptr(z), g.data_ptr(), code, M, N, K, x.stride(0),
                    weight.stride(0), g.stride(0), ctx.act, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n, st,
                    _lib.stream_ptr(dev))
            if rc:
                _lib.check(rc)
            _lib.status_after(dev, None)
        return dx, dw, db, (dy if need_r else None), None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
                 residual: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one kernel; products and sums in fp32, one rounding.

    x: (..., d_in); weight: (d_out, d_in); bias: (d_out,) or None; residual: the output's
    shape (..., d_out) or None; all CUDA tensors of one type (bfloat16, float16 or
    float32).  activation: "none", "gelu" (the erf form), "relu" or "silu".
    Differentiable in x, weight, bias and residual; the backward reads the
    pre-activations as rounded to x's type and gives every gradient in it.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of {', '.join(ACTIVATIONS)}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"expected x (..., d_in) and weight (d_out, d_in) with widths >= 1, got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    shape = (*x.shape[:-1], weight.shape[0])
    tensors = [x, weight]
    if bias is not None:
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"bias {tuple(bias.shape)} does not match d_out={weight.shape[0]}")
        bias = bias.contiguous()
        tensors.append(bias)
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual {tuple(residual.shape)} does not have the output's shape {shape}")
        tensors.append(residual)
    dtype, need_grad = x.dtype, False
    for t in tensors:
        if t.dtype != dtype:
            raise ValueError(f"x, weight, bias and residual must have one type, got {dtype} and {t.dtype}")
        need_grad = need_grad or t.requires_grad
    _lib.require_cuda(*tensors)
    if need_grad and torch.is_grad_enabled():
        if status is not None:
            raise ValueError("status is not supported on the differentiable path")
        return _LinearFunction.apply(x, weight, bias, residual, ACTIVATIONS[activation])
    y, _ = _launch(_lib.rows_of(x), _lib.rows_of(weight), bias, None if residual is None else _lib.rows_of(residual),
                   ACTIVATIONS[activation], False, shape, status)
    return y


def project(layer: torch.nn.Linear, x: torch.Tensor, fused: bool, activation: str = "none",
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """An ``nn.Linear`` of a model: through ``fused_linear``, or as PyTorch layers (no activation then)."""
    if fused:
        return fused_linear(x, layer.weight, layer.bias, activation=activation, residual=residual)
    y = layer(x)
    return y if residual is None else residual + y
