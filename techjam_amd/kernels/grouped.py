"""Python entry points of the HIP attention kernels with grouped heads.

``packed_attention`` is the softmax attention of ``scaled_dot_product_attention``
for sequences of different lengths laid end to end, with several query heads on
one key head and with gradients; ``tree_attention`` that of each sequence's
newest tokens, or of drafts that form trees, against a cache. The reference pads
its batches and has as many key heads as query heads
(``src/implementations/sdpa.py:46-78``).
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
import torch.nn.functional as F

from ..errors import UnsupportedCaseError
from . import _lib
from .attention import _ptr, _require_device, _stream_ptr
from .differential import DTYPES, _empty_heads, _rows_view, _scale, refuse_tangents

#: Largest head dim of q and k, and of v.
MAX_HEAD_DIM = 128
#: Most drafted tokens of a sequence that form trees.
MAX_DRAFTS = 64


def _readable(t: torch.Tensor) -> bool:
    """Unit innermost stride, rows and base aligned to 16 bytes, 64 tokens within 2 GiB, heads within 2^31 elements."""
    st, sh, sd = t.stride()
    size = t.element_size()
    return (sd == 1 and not (st | sh) & (16 // size - 1) and not t.data_ptr() & 15 and st * 64 * size < 1 << 31
            and sh < 1 << 31)


def _tokens_view(t: torch.Tensor) -> torch.Tensor:
    """``t`` ``[T, H, D]`` itself when the kernels can read it in place, else a contiguous copy."""
    if _readable(t):
        return t
    if min(t.shape[:2]) <= 1:
        # The stride of a dimension of at most one is never used, may be anything,
        # and stays what it is in contiguous(): 0 instead.
        t = t.as_strided(t.shape, [0 if n <= 1 else st for n, st in zip(t.shape[:2], t.stride())] + [t.stride(2)])
        if _readable(t):
            return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _launch(dev: torch.device, entry: str, *args) -> None:
    """Calls the library with the device current and its current stream as the last argument."""
    if torch._C._cuda_getDevice() == dev.index:
        code = getattr(_lib.lib(), entry)(*args, _stream_ptr(dev))
    else:
        with torch.cuda.device(dev):
            code = getattr(_lib.lib(), entry)(*args, _stream_ptr(dev))
    if code:
        _lib.check(code, entry)


def _check_types(q, k, v, h: int, hk: int) -> None:
    if h == 0 or hk == 0 or h % hk:
        raise ValueError(f"{h} query heads are not shared evenly by {hk} key heads")
    if q.dtype not in DTYPES:
        raise UnsupportedCaseError(f"dtype {q.dtype} is not supported (float32, float16 or bfloat16)")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share a dtype")
    d, dv = q.shape[-1], v.shape[-1]
    if not 0 < d <= MAX_HEAD_DIM or not 0 < dv <= MAX_HEAD_DIM:
        raise UnsupportedCaseError(f"head dims {d} and {dv} are not supported (at most {MAX_HEAD_DIM})")


def _check_ints(name: str, t, shape, dev: torch.device) -> None:
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev or t.shape != shape
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {dev}")


def check_offsets(offsets, dev: torch.device) -> None:
    """Refuses what cannot be the offsets of sequences laid end to end."""
    if not isinstance(offsets, torch.Tensor) or offsets.ndim != 1 or offsets.shape[0] == 0:
        raise ValueError("offsets must be an int32 tensor of one element more than there are sequences")
    _check_ints("offsets", offsets, offsets.shape, dev)


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


# -- packed sequences ---------------------------------------------------------

@lru_cache(maxsize=256)
def _backward_floats(t: int, n: int, h: int, hk: int) -> int:
    return _lib.lib().tj_packed_attn_bwd_workspace_bytes(t, n, h, hk) // 4


def _forward(q, k, v, offsets, valid_len, scale, causal, stats):
    """One kernel call on padded inputs: ``(out, rest, lse)``, the last two for the backward pass:
    None without ``stats``, and no ``rest`` of float32."""
    t, h, d = q.shape
    _, hk, dv = v.shape
    q, k, v = _tokens_view(q), _tokens_view(k), _tokens_view(v)
    out = q.new_empty((t, h, dv))
    lse = q.new_empty((t, h), dtype=torch.float32) if stats else None
    rest = torch.empty_like(out) if stats and q.dtype != torch.float32 else None
    _launch(q.device, "tj_packed_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), DTYPES[q.dtype],
            t, offsets.shape[0] - 1, h, hk, d, dv, _lib.strides3(q), _lib.strides3(k), _lib.strides3(v), _lib.strides3(out),
            scale, causal, offsets.data_ptr(), _ptr(valid_len), _ptr(lse), _ptr(rest))
    return out, rest, lse


def _backward(ctx, dout):
    q, k, v, out, rest, lse, offsets, valid_len = ctx.saved_tensors
    t, h, d = q.shape
    _, hk, dv = v.shape
    n = offsets.shape[0] - 1
    q, k, v, dout = _tokens_view(q), _tokens_view(k), _tokens_view(v), _tokens_view(dout)
    dq, dk, dvv = q.new_empty((t, h, d)), q.new_empty((t, hk, d)), q.new_empty((t, hk, dv))
    floats = _backward_floats(t, n, h, hk)
    ws = lse.new_empty(floats)
    _launch(q.device, "tj_packed_attn_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(rest),
            lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dvv.data_ptr(), DTYPES[q.dtype], t, n, h, hk, d, dv,
            *map(_lib.strides3, (q, k, v, out, dout, dq, dk, dvv)), ctx.scale, ctx.causal,
            offsets.data_ptr(), _ptr(valid_len), ws.data_ptr(), 4 * floats)
    return dq, dk, dvv, None, None, None, None


class _OnceOnly(torch.autograd.Function):
    """Hands gradients on as functions of what they were computed from, whose derivatives are refused. (They
    depend on the inputs also where the output gradient requires none.)"""

    @staticmethod
    def forward(ctx, dq, dk, dv, *inputs):
        return dq, dk, dv

    @staticmethod
    def backward(ctx, *grads):
        raise UnsupportedCaseError("packed_attention is differentiable once: second derivatives are not implemented")


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, valid_len, scale, causal):
        out, rest, lse = _forward(q, k, v, offsets, valid_len, scale, causal, True)
        ctx.save_for_backward(q, k, v, out, rest, lse, offsets, valid_len)
        ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        if not torch.is_grad_enabled():
            return _backward(ctx, dout)
        with torch.no_grad():  # under create_graph
            grads = _backward(ctx, dout)
        return *_OnceOnly.apply(*grads[:3], *ctx.saved_tensors[:3], dout), *grads[3:]


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    offsets: torch.Tensor,
    *,
    is_causal: bool = False,
    scale: Optional[float] = None,
    valid_len: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of sequences laid end to end, ``[T, H, Dv]``; differentiable.

    ``q`` is ``[T, H, D]``, ``k`` ``[T, Hk, D]`` and ``v`` ``[T, Hk, Dv]``; with fewer key heads
    than query heads, ``H / Hk`` neighbouring heads share one. float32, float16 or
    bfloat16, ``D`` and ``Dv`` at most 128; float32 is computed in float32 throughout. Any
    strides; views whose rows are aligned to 16 bytes (heads of one fused
    projection) are read in place.

    ``offsets`` (int32 ``[N + 1]`` on the device) says where the ``N`` sequences begin and where the
    last one ends: tokens ``offsets[n] .. offsets[n + 1] - 1`` see each other and nobody else
    (under ``is_causal`` those up to themselves). Sequences may be empty. The offsets
    do not decrease and lie within 0 and ``T``; ones that do not give wrong rows, which cannot
    be told without waiting for the device. With ``valid_len`` (int32 ``[N]``) only the first
    ``valid_len[n]`` rows of each hold tokens: a right-padded batch ``[B, S, H, D]`` is ``B``
    sequences of ``S`` rows. Rows that hold no token, also those before the first and behind the last
    sequence, come out as zeros; what they hold is not read, and their gradients are zero.

    ``scale`` defaults to ``D ** -0.5``; its magnitude is at most 2^127. Scores are float32 numbers, exact to
    2^-24 of their size; rows with one beyond 2^27 may come out as NaN. A NaN or an infinity
    among a sequence's tokens spoils what depends on it, and under ``is_causal``, as 0 times NaN,
    up to 31 neighbours that do not: one in ``v`` the outputs of tokens before it, one in ``k`` their
    gradients, one in ``q`` or the output gradient the gradients of keys behind it.

    Gradients come for q, k and v; their sums have a fixed order, so equal calls give equal
    bits. In float16 the gradient of ``k`` sums its rows at one scale: beside an output gradient 1e6
    times larger in the same sequence and key head, a row's share loses bits. Second
    derivatives and forward-mode ones (``torch.autograd.forward_ad``) are not implemented and
    refused. For the backward pass a call keeps its inputs, its output, ``4 * T * H`` bytes and, of 16-bit
    types, what rounding took from the output (``2 * T * H * Dv`` bytes); an output that was changed in place is refused there, as everywhere in torch.

    A training step can be captured into a graph as any of torch's: while it is captured, no
    graph of an earlier eager call on the same leaves may be alive (delete its outputs first).
    """
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError("q must be [T, H, D], k [T, Hk, D] and v [T, Hk, Dv]")
    (t, h, d), (_, hk, dv) = q.shape, v.shape
    if k.shape != (t, hk, d) or v.shape[0] != t:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    _check_types(q, k, v, h, hk)
    scale = _scale(scale, d)
    refuse_tangents(q, k, v)
    dev = _require_device(q, k, v)
    check_offsets(offsets, dev)
    if valid_len is not None:
        _check_ints("valid_len", valid_len, (offsets.shape[0] - 1,), dev)
    q, k, v = _padded(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _PackedAttention.apply(q, k, v, offsets, valid_len, scale, bool(is_causal))
    else:
        out = _forward(q, k, v, offsets, valid_len, scale, bool(is_causal), False)[0]
    return out if out.shape[-1] == dv else out[..., :dv]


# -- drafted tokens against a cache ---------------------------------------------

def _queries_view(t: torch.Tensor) -> torch.Tensor:
    """``_rows_view`` of the new tokens, whose heads the kernels reach by 32-bit numbers of elements."""
    if t.stride(1) >= 1 << 31:
        # One head's stride is never used.
        t = t.contiguous() if t.shape[1] > 1 else t.as_strided(t.shape, (t.stride(0), 0, *t.stride()[2:]))
    return _rows_view(t)


def check_parents(parents: torch.Tensor, b: int, t: int, dev: torch.device) -> None:
    """Refuses what cannot be the parents of ``t`` drafts of each of ``b`` sequences."""
    if t > MAX_DRAFTS:
        raise UnsupportedCaseError(f"trees of {t} drafts are not supported (at most {MAX_DRAFTS})")
    _check_ints("parents", parents, (b, t), dev)


@lru_cache(maxsize=256)
def _tree_floats(dtype: int, b: int, h: int, hk: int, t: int, c: int, d: int, dv: int) -> int:
    return _lib.lib().tj_tree_attn_workspace_bytes(dtype, b, h, hk, t, c, d, dv) // 4


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lengths: torch.Tensor,
    parents: Optional[torch.Tensor] = None,
    *,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Attention of each sequence's newest tokens against its cache, ``[B, H, T, Dv]``.

    ``q`` ``[B, H, T, D]`` holds the ``T`` newest tokens, ``k_cache`` ``[B, Hk, C, D]`` and ``v_cache``
    ``[B, Hk, C, Dv]`` the keys and values of the sequences so far, these tokens' own included;
    ``lengths`` (int32 ``[B]`` on the device) counts them, so token ``t`` stands at position
    ``lengths[b] - T + t`` of the cache. Lengths are clipped to ``C``, and what the caches hold
    behind them is not read.

    Without ``parents`` the tokens follow each other (one of them, for plain decoding): each
    sees the keys up to its position. With ``parents`` (int32 ``[B, T]`` on the device, ``T`` at
    most 64) they are drafts that form trees: ``parents[b, t]`` is the draft before draft ``t``,
    -1 for those that continue the sequence itself, and a draft sees the keys in front of the drafts, those on
    its line of parents and its own. Parents stand before their children (``parents[b, t] < t``); a
    draft whose parent does not (``T``, say) is not there, so that sequences may have
    fewer than ``T``, and neither is one on whose line such a draft stands. Tokens that are
    not there and those at a negative position (a sequence shorter than ``T``, an empty slot of the
    batch) get zeros; what the cache holds in the place of drafts that are not there may be anything.

    A NaN or an infinity in the value of one token spoils what depends on it and may spoil, as
    0 times NaN, the other tokens of this call.

    How the keys are shared among the GPU's units follows the batch's lengths, so a sequence's last
    bits may differ beside other sequences; equal calls give equal bits. ``B * H * T`` is below
    2^23 - 2^16.

    Heads, types and ``scale`` as in :func:`packed_attention`; any strides. The output's storage is
    ``[B, T, H, Dv]``, so that merging the heads is a view. No gradients: inputs that require
    them are refused while they are enabled, as are forward-mode tangents.
    """
    if q.ndim != 4 or k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("q must be [B, H, T, D], k_cache [B, Hk, C, D] and v_cache [B, Hk, C, Dv]")
    (b, h, t, d), (_, hk, c, dv) = q.shape, v_cache.shape
    if k_cache.shape != (b, hk, c, d) or v_cache.shape[0] != b:
        raise ValueError(f"shapes do not fit: q {tuple(q.shape)}, k_cache {tuple(k_cache.shape)}, "
                         f"v_cache {tuple(v_cache.shape)}")
    _check_types(q, k_cache, v_cache, h, hk)
    scale = _scale(scale, d)
    if parents is not None:
        check_parents(parents, b, t, q.device)
    if lengths is None:
        raise ValueError("lengths must be given: a cache's capacity is not its sequences' length")
    refuse_tangents(q, k_cache, v_cache)
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k_cache, v_cache)):
        raise UnsupportedCaseError("tree_attention has no gradients; call it under torch.no_grad()")
    dev = _require_device(q, k_cache, v_cache)
    _check_ints("lengths", lengths, (b,), dev)
    q, k, v = _padded(q, k_cache, v_cache)
    q, k, v = _queries_view(q), _rows_view(k), _rows_view(v)
    dtype = DTYPES[q.dtype]
    d, wide = q.shape[-1], v.shape[-1]
    out = _empty_heads(b, h, t, wide, q)
    floats = _tree_floats(dtype, b, h, hk, t, c, d, wide)
    ws = q.new_empty(floats, dtype=torch.float32) if floats else None
    _launch(dev, "tj_tree_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dtype, b, h, hk, t, c, d, wide,
            _lib.strides4(q), _lib.strides4(k), _lib.strides4(v), _lib.strides4(out), scale,
            lengths.data_ptr(), _ptr(parents), _ptr(ws), 4 * floats)
    return out if wide == dv else out[..., :dv]
