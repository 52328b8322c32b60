"""Softmax self-attention with grouped heads for the encoder: training, packed sequences, drafted trees.

The reference's encoder attends within padded batches, without gradients on its
fused paths and without a cache (``torch_transformer_benchmark.py:75-121``);
``TransformerConfig(..., attention="grouped")`` builds its blocks with the module
below instead: the same softmax attention, whose ``num_heads`` query heads share
``kv_heads`` key and value heads. It trains on the kernels, takes sequences laid end
to end, and runs token by token or over trees of drafted tokens.
"""

from __future__ import annotations

from typing import List, Optional

import torch
import torch.nn as nn

from ..kernels.grouped import check_parents, packed_attention, tree_attention
from ..model import Linear, not_captured, prefix_lengths


class GroupedCache:
    """Keys and values of a batch's sequences for one layer, of ``capacity`` tokens each."""

    def __init__(self, batch: int, capacity: int, kv_heads: int, head_dim: int, dtype=torch.float32, device=None) -> None:
        self.k = torch.zeros(batch, kv_heads, capacity, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros(batch, kv_heads, capacity, head_dim, dtype=dtype, device=device)

    def check_type(self, dtype: torch.dtype) -> None:
        """Refuses keys and values of another type, which a copy would round in silence."""
        if dtype != self.k.dtype:
            raise ValueError(f"the cache holds {self.k.dtype}, the call's keys and values are {dtype}: "
                             "create the state in that dtype")


class GroupedState:
    """Every layer's cache and the sequences' settled lengths (int32 ``[B]`` on the device).

    ``longest`` bounds the lengths on the host, so that a step past the capacity is
    refused without asking the device. ``drafts`` counts the drafted tokens that stand in the
    caches behind what is settled (``accept``).
    """

    def __init__(self, config, batch: int, capacity: int, dtype=torch.float32, device=None) -> None:
        if batch <= 0 or capacity <= 0:
            raise ValueError("batch and capacity must be positive")
        kv_heads, head_dim = grouped_heads(config)
        self.capacity = capacity
        self.layers: List[GroupedCache] = [
            GroupedCache(batch, capacity, kv_heads, head_dim, dtype, device) for _ in range(config.num_layers)]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.longest = 0
        self.drafts = 0

    def check_drafts(self, parents, tokens: int) -> None:
        check_parents(parents, self.lengths.shape[0], tokens, self.lengths.device)

    def reserve(self, tokens: int) -> None:
        if self.longest + tokens > self.capacity:
            raise ValueError(f"{tokens} more tokens exceed the cache's capacity of {self.capacity} "
                             f"(up to {self.longest} in use)")

    @torch.no_grad()
    def accept(self, path: torch.Tensor, counts: torch.Tensor) -> None:
        """Settles drafts of the last step over a tree: the first ``counts[b]`` of ``path[b]`` (integers ``[B, M]``
        and ``[B]``), drafts from parent to child, become the sequence's next tokens. Their keys and values
        move to the places behind what was settled; the other drafts are dropped.

        ``counts`` on the host say how long the longest sequence is now; on the device they are not
        waited for, and the bound grows by ``M``, until :meth:`recount`. Not for graphs: a replay would
        settle tokens that the bound does not count.
        """
        not_captured()
        if self.drafts == 0:
            raise ValueError("there are no drafts to accept: the last call was no step over a tree")
        b = self.lengths.shape[0]
        if path.ndim != 2 or path.shape[0] != b or path.shape[1] > self.drafts or counts.shape != (b,):
            raise ValueError(f"path must be [{b}, M] with at most {self.drafts} drafts and counts [{b}], "
                             f"not {tuple(path.shape)} and {tuple(counts.shape)}")
        for name, t in (("path", path), ("counts", counts)):
            if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
                raise ValueError(f"{name} must be integers, not {t.dtype}")
        m, device = path.shape[1], self.lengths.device
        most = m if counts.is_cuda else min(m, max(0, int(counts.max())))
        path = path.to(device).long().clamp(0, self.drafts - 1)
        counts = counts.to(device=device, dtype=torch.int32).clamp(0, m)
        rows, settled = torch.arange(b, device=device)[:, None], self.lengths[:, None].long()
        source, place = settled + path, settled + torch.arange(m, device=device)
        for cache in self.layers:
            cache.k[rows, :, place] = cache.k[rows, :, source]
            cache.v[rows, :, place] = cache.v[rows, :, source]
        self.lengths += counts
        self.longest += most
        self.drafts = 0

    def recount(self) -> None:
        """Asks the device (and waits for it) how long the longest sequence is."""
        not_captured()
        self.longest = int(self.lengths.max())


def grouped_heads(config) -> tuple:
    """``(kv_heads, head_dim)`` of a config; as many key heads as query heads when it does not say."""
    kv_heads = getattr(config, "kv_heads", None) or config.num_heads
    return kv_heads, config.d_model // config.num_heads


class GroupedSelfAttention(nn.Module):
    """Multi-head self-attention with grouped heads, a stand-in for ``HipSelfAttention``.

    Differentiable (the gradients run on the kernels of ``kernels/grouped.py``), float32,
    float16 or bfloat16 like its parameters. Padded rows come out as zeros.
    """

    def __init__(self, d_model: int, num_heads: int, kv_heads: Optional[int] = None) -> None:
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if d_model % num_heads:
            raise ValueError("d_model must be divisible by num_heads")
        if kv_heads <= 0 or num_heads % kv_heads:
            raise ValueError("num_heads must be divisible by kv_heads")
        self.d_model = d_model
        self.num_heads = num_heads
        self.kv_heads = kv_heads
        self.head_dim = d_model // num_heads
        self.scale = self.head_dim ** -0.5
        self.q_proj = Linear(d_model, d_model)
        self.k_proj = Linear(d_model, kv_heads * self.head_dim)
        self.v_proj = Linear(d_model, kv_heads * self.head_dim)
        self.out_proj = Linear(d_model, d_model)

    def qkv(self, x):
        """``[..., H, dh]`` and ``[..., Hk, dh]`` twice, views of the projections."""
        lead = x.shape[:-1]
        return (self.q_proj(x).view(*lead, self.num_heads, self.head_dim),
                self.k_proj(x).view(*lead, self.kv_heads, self.head_dim),
                self.v_proj(x).view(*lead, self.kv_heads, self.head_dim))

    def context(self, x, valid_token_mask=None, causal=False, valid_len=None, cache: Optional[GroupedCache] = None):
        """Attention output before the output projection, ``[B, S, D]``; with ``cache`` the
        keys and values of these first ``S`` tokens go there. The batch is ``B`` sequences of ``S`` rows
        laid end to end."""
        if valid_len is None and valid_token_mask is not None:
            valid_len = prefix_lengths(valid_token_mask)
        b, s, _ = x.shape
        q, k, v = self.qkv(x)
        if cache is not None:
            cache.check_type(k.dtype)
            cache.k[:, :, :s] = k.transpose(1, 2)
            cache.v[:, :, :s] = v.transpose(1, 2)
        offsets = torch.arange(0, b * s + 1, s, dtype=torch.int32, device=x.device) if s else x.new_zeros(b + 1, dtype=torch.int32)
        out = packed_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), offsets, is_causal=causal,
                               scale=self.scale, valid_len=valid_len)
        return out.reshape(b, s, self.d_model)

    def forward(self, x, valid_token_mask=None, causal=False, valid_len=None, cache=None):
        out = self.out_proj(self.context(x, valid_token_mask, causal, valid_len, cache))
        if valid_token_mask is not None:
            out = out.masked_fill(~valid_token_mask[..., None], 0)
        return out

    def packed(self, x, offsets, causal=False, keep=None):
        """``x`` ``[T, D]``, sequences laid end to end from ``offsets`` on; ``keep(k, v)`` gets the keys and values."""
        q, k, v = self.qkv(x)
        if keep is not None:
            keep(k, v)
        out = packed_attention(q, k, v, offsets, is_causal=causal, scale=self.scale)
        return self.out_proj(out.flatten(1))

    def step(self, x, cache: GroupedCache, lengths, place, parents=None):
        """``x`` ``[B, T, D]``: the next ``T`` tokens of each sequence, or drafts with their
        ``parents``, the last of ``lengths`` (these included), whose places in the cache are ``place``
        (int64 ``[B, T]``)."""
        q, k, v = self.qkv(x)
        cache.check_type(k.dtype)
        rows = torch.arange(x.shape[0], device=x.device)[:, None]
        cache.k[rows, :, place] = k
        cache.v[rows, :, place] = v
        heads = tree_attention(q.transpose(1, 2), cache.k, cache.v, lengths, parents, scale=self.scale)
        return self.out_proj(heads.transpose(1, 2).flatten(2))
