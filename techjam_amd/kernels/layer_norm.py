"""Layer norm on the HIP kernels, forward and backward.

The reference's norms are ``torch.nn.LayerNorm``
(``torch_transformer_benchmark.py:125-172``). ``elementwise.py`` has the norm
that closes a residual pass in inference; ``layer_norm`` is the norm by itself,
for every width up to ``MAX_WIDTH``, with gradients.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ..errors import UnsupportedCaseError
from . import _lib
from .attention import _ptr, _require_device, _stream_ptr
from .differential import DTYPES, on_device, refuse_tangents

#: Widest row the kernels take.
MAX_WIDTH = 16384


@lru_cache(maxsize=256)
def _workspace_floats(rows: int, width: int) -> int:
    return _lib.lib().tj_layer_norm_bwd_workspace_bytes(rows, width) // 4


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as ``[rows, width]`` with unit column stride: a view where its
    leading dimensions have one stride in common (below 2^23 elements), else a
    copy."""
    width = t.shape[-1]
    if t.is_contiguous():
        if t.ndim != 2:
            t = t.view(-1, width)
        # A single row is contiguous whatever its row stride is.
        return t if t.shape[0] != 1 or t.stride(0) == width else t.as_strided((1, width), (width, 1))
    t = t.reshape(-1, width)
    if (t.stride(1) != 1 and width > 1) or t.stride(0) >= 1 << 23:
        return t.contiguous()
    return t


def _forward(x, weight, bias, eps, stats, y_dtype):
    rows2d = _rows(x)
    rows, width = rows2d.shape
    dev = x.device
    y = torch.empty_like(x, dtype=y_dtype, memory_format=torch.contiguous_format)
    # mean [rows], then 1 / sqrt(var + eps) [rows], in one tensor.
    moments = x.new_empty(2 * rows, dtype=torch.float32) if stats else None
    mean = moments.data_ptr() if stats and rows else None
    w_dtype = _lib.TJ_F32
    if weight is not None or bias is not None:
        w_dtype = DTYPES[(bias if weight is None else weight).dtype]
    with on_device(dev):
        code = _lib.lib().tj_layer_norm_fwd(
            rows2d.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), DTYPES[x.dtype], DTYPES[y_dtype], w_dtype, rows, width,
            rows2d.stride(0), width, eps, mean, mean and mean + 4 * rows, _stream_ptr(dev))
    if code:
        _lib.check(code, "tj_layer_norm_fwd")
    return y, moments


def _backward(ctx, dy):
    x, weight, moments = ctx.saved_tensors
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dy2d, x2d = _rows(dy), _rows(x)
    rows, width = x2d.shape
    dev = x.device
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    w_torch = ctx.bias_dtype if weight is None else weight.dtype
    dw = moments.new_empty(width, dtype=w_torch) if need_w else None
    db = moments.new_empty(width, dtype=w_torch) if need_b else None
    if rows == 0:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_(), None, None
    mean = moments.data_ptr()
    ws = moments.new_empty(_workspace_floats(rows, width)) if need_w or need_b else None
    with on_device(dev):
        code = _lib.lib().tj_layer_norm_bwd(
            dy2d.data_ptr(), x2d.data_ptr(), _ptr(weight), mean, mean + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db),
            DTYPES[x.dtype], DTYPES[dy.dtype], _lib.TJ_F32 if w_torch is None else DTYPES[w_torch], rows, width,
            dy2d.stride(0), x2d.stride(0), width, _ptr(ws), 0 if ws is None else 4 * ws.numel(), _stream_ptr(dev))
    if code:
        _lib.check(code, "tj_layer_norm_bwd")
    return dx, dw, db, None, None


#: Under create_graph: the gradients, with an error for whoever differentiates
#: them. Without it the plain function, whose call is leaner by 3 to 4 us of
#: about 120 for the forward and backward pass of 256 rows of 256.
_backward_once = once_differentiable(_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, y_dtype):
        y, moments = _forward(x, weight, bias, eps, True, y_dtype)
        ctx.save_for_backward(x, weight, moments)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _check_param(name, p, width, dtype, dev) -> None:
    if p.shape != (width,) or p.device != dev or not p.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {width} elements on {dev}")
    if p.dtype != torch.float32 and p.dtype != dtype:
        raise ValueError(f"{name} must be float32 or {dtype}, not {p.dtype}")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, norm_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Layer norm over the last dimension of ``x``; differentiable in all three tensors.

    ``x`` is float32, float16 or bfloat16 with a last dimension of at most
    ``MAX_WIDTH``, of any shape and strides (read in place where the rows have
    one common stride). ``weight`` and ``bias`` are contiguous ``[width]``, both
    float32 or both of ``x``'s type, each optional; their gradients come in their
    type. Statistics and sums are float32, the output is contiguous and of
    ``x``'s type, or float32 with ``norm_dtype=torch.float32`` (the norm of
    16-bit rows not rounded to 16 bits). The gradients' sums over the rows have
    a fixed order, so equal calls give equal bits. Second derivatives and
    forward-mode ones (``torch.autograd.forward_ad``) are not implemented and
    refused. While a training step is captured into a graph, no graph of an
    earlier eager call on the same leaves may be alive (delete its outputs first).
    """
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError("x must have a last dimension to normalise over")
    if x.dtype not in DTYPES:
        raise UnsupportedCaseError(f"dtype {x.dtype} is not supported (float32, float16 or bfloat16)")
    width = x.shape[-1]
    if width > MAX_WIDTH:
        raise UnsupportedCaseError(f"width {width} is not supported (at most {MAX_WIDTH})")
    refuse_tangents(x, weight, bias)
    dev = _require_device(x)
    if weight is not None:
        _check_param("weight", weight, width, x.dtype, dev)
    if bias is not None:
        _check_param("bias", bias, width, x.dtype, dev)
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError("weight and bias must share a dtype")
    if norm_dtype is None:
        norm_dtype = x.dtype
    elif norm_dtype not in (torch.float32, x.dtype):
        raise ValueError(f"norm_dtype must be float32 or {x.dtype}, not {norm_dtype}")
    eps = float(eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, norm_dtype)
    return _forward(x, weight, bias, eps, False, norm_dtype)[0]


class LayerNorm(torch.nn.LayerNorm):
    """``torch.nn.LayerNorm`` over one dimension, same parameters and state-dict
    names, whose forward is :func:`layer_norm`."""

    def __init__(self, width: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device=None, dtype=None) -> None:
        super().__init__(width, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises over the last dimension alone")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.ndim == 0 or x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"x must have a last dimension of {self.normalized_shape[0]}, not {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
