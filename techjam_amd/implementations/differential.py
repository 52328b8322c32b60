"""Differential self-attention for the encoder: training, inference and cached steps.

The reference's encoder has softmax attention only
(``torch_transformer_benchmark.py:75-121``); ``TransformerConfig(...,
attention="differential")`` builds its blocks with the module below instead.
Each of ``num_heads`` heads has two query and two key heads of half its width,
one value head of the whole width, a learned weight of its second map, and a
layer norm of its own output; with the same projections as softmax attention,
the parameter count differs by the weights and the norm alone.
"""

from __future__ import annotations

import math
from typing import List, Optional

import torch
import torch.nn as nn

from ..kernels.differential import differential_attention, differential_attention_cached
from ..kernels.layer_norm import LayerNorm
from ..model import Linear, prefix_lengths


def initial_weight(depth: int) -> float:
    """The second map's weight in layer ``depth`` (from 0) before training: 0.2
    at first, towards 0.8 in deep layers."""
    return 0.8 - 0.6 * math.exp(-0.3 * depth)


class DifferentialCache:
    """Keys and values of a batch's sequences for one layer, of ``capacity`` tokens each."""

    def __init__(self, batch: int, capacity: int, num_heads: int, head_dim: int, dtype=torch.float32, device=None) -> None:
        self.k = torch.zeros(batch, 2 * num_heads, capacity, head_dim // 2, dtype=dtype, device=device)
        self.v = torch.zeros(batch, num_heads, capacity, head_dim, dtype=dtype, device=device)


class DifferentialState:
    """Every layer's cache and the sequences' lengths (int32 ``[B]`` on the device).

    ``longest`` bounds the lengths on the host, so that a step past the
    capacity is refused without asking the device.
    """

    def __init__(self, config, batch: int, capacity: int, dtype=torch.float32, device=None) -> None:
        if batch <= 0 or capacity <= 0:
            raise ValueError("batch and capacity must be positive")
        head_dim = config.d_model // config.num_heads
        self.capacity = capacity
        self.layers: List[DifferentialCache] = [
            DifferentialCache(batch, capacity, config.num_heads, head_dim, dtype, device) for _ in range(config.num_layers)]
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.longest = 0

    def reserve(self, tokens: int) -> None:
        if self.longest + tokens > self.capacity:
            raise ValueError(f"{tokens} more tokens exceed the cache's capacity of {self.capacity} "
                             f"(up to {self.longest} in use)")


class DifferentialSelfAttention(nn.Module):
    """Multi-head differential self-attention, a stand-in for ``HipSelfAttention``.

    Differentiable (the gradients run on the kernels of
    ``kernels/differential.py`` and ``kernels/layer_norm.py``), float32, float16
    or bfloat16 like its parameters. Padded rows come out as zeros.
    """

    def __init__(self, d_model: int, num_heads: int, depth: int = 0) -> None:
        super().__init__()
        if d_model % (2 * num_heads):
            raise ValueError("d_model must be divisible by 2 * num_heads")
        self.d_model = d_model
        self.num_heads = num_heads
        self.head_dim = d_model // num_heads
        self.scale = (self.head_dim // 2) ** -0.5
        self.q_proj = Linear(d_model, d_model)
        self.k_proj = Linear(d_model, d_model)
        self.v_proj = Linear(d_model, d_model)
        self.out_proj = Linear(d_model, d_model)
        start = initial_weight(depth)
        self.lam = nn.Parameter(torch.full((num_heads,), start))
        # The norm takes a head's output to unit size; its weight starts where
        # the difference of the maps leaves it.
        self.head_norm = LayerNorm(self.head_dim)
        nn.init.constant_(self.head_norm.weight, 1.0 - start)

    def qkv(self, x):
        """``[B, 2H, S, dh / 2]`` twice and ``[B, H, S, dh]``, strided views of the projections."""
        b, s, _ = x.shape
        q, k, v = self.q_proj(x), self.k_proj(x), self.v_proj(x)
        half = (b, s, 2 * self.num_heads, self.head_dim // 2)
        return (q.view(half).transpose(1, 2), k.view(half).transpose(1, 2),
                v.view(b, s, self.num_heads, self.head_dim).transpose(1, 2))

    def _merge(self, heads):
        """Norm of each head, and the heads side by side."""
        b, _, s, _ = heads.shape
        return self.head_norm(heads.transpose(1, 2)).reshape(b, s, self.d_model)

    def context(self, x, valid_token_mask=None, causal=False, valid_len=None, cache: Optional[DifferentialCache] = None):
        """Normed heads before the output projection, ``[B, S, D]``; with ``cache``
        the keys and values of these first ``S`` tokens go there."""
        if valid_len is None and valid_token_mask is not None:
            valid_len = prefix_lengths(valid_token_mask)
        q, k, v = self.qkv(x)
        if cache is not None:
            cache.k[:, :, :x.shape[1]] = k
            cache.v[:, :, :x.shape[1]] = v
        return self._merge(differential_attention(q, k, v, self.lam, is_causal=causal, scale=self.scale,
                                                  valid_len=valid_len))

    def forward(self, x, valid_token_mask=None, causal=False, valid_len=None, cache=None):
        out = self.out_proj(self.context(x, valid_token_mask, causal, valid_len, cache))
        if valid_token_mask is not None:
            out = out.masked_fill(~valid_token_mask[..., None], 0)
        return out

    def step(self, x, cache: DifferentialCache, lengths, place):
        """``x`` ``[B, T, D]``: the next ``T`` tokens of each sequence, the last
        of ``lengths`` (these included), whose places in the cache are ``place``
        (int64 ``[B, T]``)."""
        q, k, v = self.qkv(x)
        if k.dtype != cache.k.dtype:
            raise ValueError(f"the cache holds {cache.k.dtype}, the step's keys and values are {k.dtype}: "
                             "create the state in that dtype")
        rows = torch.arange(x.shape[0], device=x.device)[:, None]
        cache.k[rows, :, place] = k.transpose(1, 2)
        cache.v[rows, :, place] = v.transpose(1, 2)
        heads = differential_attention_cached(q, cache.k, cache.v, self.lam, lengths, scale=self.scale)
        return self.out_proj(self._merge(heads))
