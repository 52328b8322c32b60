"""Python entry points of the HIP differential-attention kernels.

Differential attention replaces a head's softmax map by the difference of two,
``O_h = (P_0 - lam_h P_1) V`` with ``P_m = softmax(scale q_{2h+m} k_{2h+m}^T)``
and a learned weight ``lam``. The reference has no counterpart; the functions
stand beside ``scaled_dot_product_attention``, take strided ``[B, H, S, D]``
views the same way, and have gradients.
"""

from __future__ import annotations

import contextlib
from functools import lru_cache
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..errors import UnsupportedCaseError
from . import _lib
from .attention import _ptr, _require_device, _stream_ptr

#: Largest head dim of q and k, and of v.
MAX_HEAD_DIM = 128
MAX_VALUE_DIM = 256
#: Largest scale whose product with log2 e is a float32.
MAX_SCALE = 2.0 ** 127

DTYPES = {torch.float32: _lib.TJ_F32, torch.float16: _lib.TJ_F16, torch.bfloat16: _lib.TJ_BF16}


def on_device(device: torch.device):
    """The device's own context when it is not the current one: a kernel is
    launched on the current device, whatever its stream's."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def tangents_enabled() -> bool:
    """Whether tensors may carry forward-mode tangents that operators have to hand on."""
    return forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()


def refuse_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Forward-mode derivatives are not implemented. A dual tensor need not
    require grad, so without a look at it a call outside of autograd would
    return its output without the tangent, which torch takes as zero."""
    if tangents_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise UnsupportedCaseError("forward-mode derivatives are not implemented")


def _readable(t: torch.Tensor) -> bool:
    """Unit innermost stride, rows and base aligned to 16 bytes, 64 rows within 2 GiB."""
    sb, sh, ss, sd = t.stride()
    size = t.element_size()
    return sd == 1 and not (sb | sh | ss) & (16 // size - 1) and not t.data_ptr() & 15 and ss * 64 * size < 1 << 31


def _rows_view(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself when the kernels can read it in place, else a contiguous copy."""
    if _readable(t):
        return t
    if min(t.shape[:3]) <= 1:
        # The stride of a dimension of at most one is never used, may be anything,
        # and stays what it is in contiguous(): 0 instead.
        t = t.as_strided(t.shape, [0 if n <= 1 else st for n, st in zip(t.shape[:3], t.stride())] + [t.stride(3)])
        if _readable(t):
            return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _empty_heads(b: int, h: int, s: int, d: int, like: torch.Tensor) -> torch.Tensor:
    """A ``[B, H, S, D]`` tensor whose storage is ``[B, S, H, D]``, what
    merging the heads or splitting a projection views for free."""
    return like.new_empty_strided((b, h, s, d), (s * h * d, d, h * d, 1))


def _check(q, k, v, lam, lengths, what: str, cached: bool) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q must be [B, 2H, S, D], k [B, 2Hk, S, D] and v [B, Hk, S, Dv]")
    (b, h2, sq, d), (_, hk2, sk, _), (_, hk, _, dv) = q.shape, k.shape, v.shape
    if k.shape != (b, 2 * hk, sk, d) or v.shape[0] != b or v.shape[2] != sk:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if h2 % 2 or hk == 0 or h2 == 0 or (h2 // 2) % hk:
        raise ValueError(f"{h2} query heads are not pairs shared evenly by {hk} value heads")
    if not cached and sq != sk:
        raise ValueError(f"q has {sq} tokens and k {sk}; new tokens against a cache are "
                         "differential_attention_cached")
    if q.dtype not in DTYPES:
        raise UnsupportedCaseError(f"dtype {q.dtype} is not supported (float32, float16 or bfloat16)")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share a dtype")
    if not 0 < d <= MAX_HEAD_DIM or not 0 < dv <= MAX_VALUE_DIM:
        raise UnsupportedCaseError(f"head dims {d} and {dv} are not supported (at most {MAX_HEAD_DIM} and "
                                   f"{MAX_VALUE_DIM})")
    if not isinstance(lam, torch.Tensor) or not lam.is_floating_point() or lam.shape not in ((), (1,), (h2 // 2,)):
        raise ValueError(f"lam must be a floating-point tensor of one or {h2 // 2} elements")
    refuse_tangents(q, k, v, lam)
    dev = _require_device(q, k, v, lam)
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.device != dev or lengths.shape != (b,)
                                or not lengths.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous int32 tensor of {b} elements on {dev}")


def _padded(q, k, v):
    """Head dims that fill no whole 16 bytes are zero-padded to the next that
    does: zeros add nothing to a score and give columns that are cut off."""
    vec = 16 // q.element_size()
    if q.shape[-1] % vec:
        pad = (0, -q.shape[-1] % vec)
        q, k = F.pad(q, pad), F.pad(k, pad)
    if v.shape[-1] % vec:
        v = F.pad(v, (0, -v.shape[-1] % vec))
    return q, k, v


@lru_cache(maxsize=256)
def _workspace_floats(b: int, h: int, hk: int, sq: int, sk: int, dv: int, cached: int) -> int:
    return _lib.lib().tj_diff_attn_workspace_bytes(b, h, hk, sq, sk, dv, cached) // 4


@lru_cache(maxsize=256)
def _backward_floats(b: int, h: int, hk: int, s: int) -> int:
    return _lib.lib().tj_diff_attn_bwd_workspace_bytes(b, h, hk, s) // 4


def _forward(q, k, v, lam, lengths, scale, causal, cached, stats):
    """One kernel call on padded inputs: ``(out, maps, lse)``, the last two None without ``stats``."""
    b, h2, sq, d = q.shape
    _, hk, sk, dv = v.shape
    h = h2 // 2
    q, k, v = _rows_view(q), _rows_view(k), _rows_view(v)
    dev = q.device
    out = _empty_heads(b, h, sq, dv, q)
    maps = lse = None
    if stats:
        maps, lse = lam.new_empty((b, h, sq, 2, dv)), lam.new_empty((b, h, 2, sq))
    floats = _workspace_floats(b, h, hk, sq, sk, dv, int(cached))
    ws = lam.new_empty(floats) if floats else None
    with on_device(dev):
        code = _lib.lib().tj_diff_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), DTYPES[q.dtype], b, h, hk, sq, sk, d, dv,
            _lib.strides4(q), _lib.strides4(k), _lib.strides4(v), _lib.strides4(out), scale, int(causal), int(cached),
            lam.data_ptr(), int(lam.numel() > 1), _ptr(lengths), _ptr(lse), _ptr(maps), _ptr(ws), 4 * floats,
            _stream_ptr(dev))
    _lib.check(code, "tj_diff_attn_fwd")
    return out, maps, lse


def _backward(ctx, dout):
    q, k, v, lam, lengths, maps, lse = ctx.saved_tensors
    b, h2, s, d = q.shape
    _, hk, _, dv = v.shape
    h = h2 // 2
    q, k, v, dout = _rows_view(q), _rows_view(k), _rows_view(v), _rows_view(dout)
    dev = q.device
    dq, dk = _empty_heads(b, h2, s, d, q), _empty_heads(b, 2 * hk, s, d, q)
    dvv = _empty_heads(b, hk, s, dv, q)
    dlam = lam.new_empty(lam.shape)
    if b == 0 or s == 0:
        return dq, dk, dvv, dlam.zero_(), None, None, None
    floats = _backward_floats(b, h, hk, s)
    ws = lam.new_empty(floats)
    with on_device(dev):
        code = _lib.lib().tj_diff_attn_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), maps.data_ptr(), lse.data_ptr(),
            dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dvv.data_ptr(), dlam.data_ptr(), DTYPES[q.dtype],
            b, h, hk, s, d, dv, *map(_lib.strides4, (q, k, v, dout, dq, dk, dvv)), ctx.scale, int(ctx.causal),
            lam.data_ptr(), int(lam.numel() > 1), _ptr(lengths), ws.data_ptr(), 4 * floats, _stream_ptr(dev))
    _lib.check(code, "tj_diff_attn_bwd")
    return dq, dk, dvv, dlam, None, None, None


#: Under create_graph: the gradients, with an error for whoever differentiates
#: them. Without it the plain function, whose call is leaner.
_backward_once = once_differentiable(_backward)


class _DifferentialAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, lengths, scale, causal):
        out, maps, lse = _forward(q, k, v, lam, lengths, scale, causal, False, True)
        ctx.save_for_backward(q, k, v, lam, lengths, maps, lse)
        ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        return _backward_once(ctx, dout) if torch.is_grad_enabled() else _backward(ctx, dout)


def _scale(scale: Optional[float], d: int) -> float:
    scale = d ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"scale must be at most 2^127 in magnitude, not {scale}")
    return scale


def differential_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lam: torch.Tensor,
    *,
    is_causal: bool = False,
    scale: Optional[float] = None,
    valid_len: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Differential attention of whole sequences, ``[B, H, S, Dv]``; differentiable.

    ``q`` is ``[B, 2H, S, D]`` (heads ``2h`` and ``2h + 1`` are the two maps of
    output head ``h``), ``k`` ``[B, 2Hk, S, D]`` and ``v`` ``[B, Hk, S, Dv]``; with
    fewer key heads than query heads, ``H / Hk`` neighbouring heads share one.
    ``lam``, the second map's weight, is one number for all heads or ``[H]``.
    float32, float16 or bfloat16, ``D <= 128``, ``Dv <= 256``; float32 is
    computed in float32 throughout. Any strides; views whose rows are aligned to
    16 bytes are read in place.

    ``valid_len`` (int32 ``[B]`` on the device) masks keys ``j >= valid_len[b]``
    and zeroes rows ``i >= valid_len[b]``, as in ``scaled_dot_product_attention``;
    what those rows and keys hold is not read, and their gradients are zero.
    ``scale`` defaults to ``D ** -0.5``; its magnitude is at most 2^127.

    A NaN or an infinity among the valid inputs spoils what depends on it; one in
    ``v`` under ``is_causal`` also the up to 31 rows before it in its tile of 32
    tokens, as 0 times NaN.

    The output's storage is ``[B, S, H, Dv]``, so that merging the heads is a
    view. Gradients come for q, k, v and lam (summed over what shares a weight);
    their sums have a fixed order, so equal calls give equal bits. In float16 the
    gradient of ``k`` sums its rows at one scale: beside an output gradient 1e6
    times larger in the same sequence and key head, a row's share loses bits. Second
    derivatives and forward-mode ones (``torch.autograd.forward_ad``) are not
    implemented and refused. For the backward pass a call keeps its inputs and
    both maps' outputs in float32, ``8 * B * H * S * (Dv + 1)`` bytes.

    A training step can be captured into a graph as any of torch's: while it is
    captured, no graph of an earlier eager call on the same leaves may be alive
    (delete its outputs first).
    """
    _check(q, k, v, lam, valid_len, "valid_len", False)
    scale = _scale(scale, q.shape[-1])
    dv = v.shape[-1]
    q, k, v = _padded(q, k, v)
    lam = lam.float().contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or lam.requires_grad):
        out = _DifferentialAttention.apply(q, k, v, lam, valid_len, scale, bool(is_causal))
    else:
        out = _forward(q, k, v, lam, valid_len, scale, bool(is_causal), False, False)[0]
    return out if out.shape[-1] == dv else out[..., :dv]


def differential_attention_cached(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lam: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Differential attention of each sequence's newest tokens, ``[B, H, T, Dv]``.

    ``q`` ``[B, 2H, T, D]`` holds the ``T`` newest tokens (one, for plain
    decoding), ``k_cache`` ``[B, 2Hk, C, D]`` and ``v_cache`` ``[B, Hk, C, Dv]``
    the keys and values of the sequences so far, these tokens' own included;
    ``lengths`` (int32 ``[B]`` on the device) counts them. Token ``t`` sees the
    keys up to its position ``lengths[b] - T + t``; tokens at a negative position
    (a sequence shorter than ``T``, an empty slot of the batch) get zeros. Lengths
    are clipped to ``C``, and what the caches hold behind them is not read. ``B *
    H * T`` is below 2^24 where ``T * H / Hk`` is at most 64.

    How the keys are shared among the GPU's units follows the batch's lengths, so
    a sequence's last bits may differ beside other sequences; equal calls give
    equal bits.

    Layouts, types and ``lam`` as in :func:`differential_attention`. No
    gradients: inputs that require them are refused while they are enabled, as
    are forward-mode tangents.
    """
    if lengths is None:
        raise ValueError("lengths must be given: a cache's capacity is not its sequences' length")
    _check(q, k_cache, v_cache, lam, lengths, "lengths", True)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k_cache, v_cache, lam)):
        raise UnsupportedCaseError("differential_attention_cached has no gradients; call it under torch.no_grad()")
    scale = _scale(scale, q.shape[-1])
    dv = v_cache.shape[-1]
    q, k, v = _padded(q, k_cache, v_cache)
    out = _forward(q, k, v, lam.detach().float().contiguous(), lengths, scale, True, True, False)[0]
    return out if out.shape[-1] == dv else out[..., :dv]
