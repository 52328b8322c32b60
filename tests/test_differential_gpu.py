"""Differential attention, forward, backward and cached, against its definition in float64 (GPU).

Bounds come element by element from ``differential_reference``; subnormal
results may be off by half their spacing besides.
"""

from __future__ import annotations

import pytest
import torch

from differential_reference import assert_within, attention

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# Half the spacing of fp16's subnormals; the other types' are far below anything here.
FLOOR = {torch.float32: 1e-40, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}


def heads(g, b, h, s, d, dtype, std=1.0):
    """A [B, H, S, D] view of [B, S, H, D] storage."""
    return (torch.randn(b, s, h, d, generator=g) * std).to(dtype).cuda().transpose(1, 2)


def inputs(dtype, b, h, hk, s, d, dv, seed=0, shared=False):
    g = torch.Generator().manual_seed(seed)
    lam = 0.2 + 0.6 * torch.rand(1 if shared else h, generator=g)
    return (heads(g, b, 2 * h, s, d, dtype, 1.5), heads(g, b, 2 * hk, s, d, dtype), heads(g, b, hk, s, dv, dtype),
            (lam.reshape(()) if shared else lam).cuda(), heads(g, b, h, s, dv, dtype, 0.3))


def lengths_of(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


# b, h, hk, s, d, dv, causal, lengths
SHAPES = {
    "one_token": (2, 2, 2, 1, 32, 64, True, None),
    "short": (2, 2, 1, 31, 32, 64, True, (31, 7)),
    "tile": (1, 2, 2, 128, 64, 128, True, None),
    "past_tile": (2, 2, 2, 129, 64, 128, False, (129, 65)),
    "odd": (3, 3, 1, 197, 64, 128, True, (197, 0, 33)),
    "wide": (1, 2, 1, 150, 128, 256, True, None),
    "wide_padded": (2, 1, 1, 67, 128, 256, False, (1, 66)),
    "narrow": (2, 4, 2, 70, 16, 32, True, None),
    "odd_dims": (1, 2, 2, 45, 40, 80, True, None),
    "uneven_dims": (2, 2, 1, 90, 64, 48, False, (90, 50)),
    "tiny_dims": (1, 1, 1, 33, 3, 5, True, None),
    "keys_shared_by_five": (1, 10, 2, 77, 32, 64, True, None),
    "long": (1, 1, 1, 1100, 64, 128, True, None),
    "keys_in_parts": (1, 1, 1, 2300, 64, 128, True, None),
    "keys_in_parts_padded": (2, 2, 1, 2090, 32, 64, False, (2090, 700)),
    "keys_in_parts_wide": (1, 1, 1, 2049, 128, 256, True, None),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda, shape, dtype):
    from techjam_amd.kernels import differential_attention

    b, h, hk, s, d, dv, causal, lens = SHAPES[shape]
    q, k, v, lam, _ = inputs(TYPES[dtype], b, h, hk, s, d, dv)
    lengths = None if lens is None else lengths_of(*lens)
    with torch.no_grad():
        out = differential_attention(q, k, v, lam, is_causal=causal, valid_len=lengths)
    want = attention(q, k, v, lam, causal=causal, lengths=lengths)
    assert out.dtype == q.dtype
    assert_within(out, want["out"], "out", FLOOR[q.dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(cuda, shape, dtype):
    from techjam_amd.kernels import differential_attention

    b, h, hk, s, d, dv, causal, lens = SHAPES[shape]
    q, k, v, lam, dout = inputs(TYPES[dtype], b, h, hk, s, d, dv, seed=1)
    lengths = None if lens is None else lengths_of(*lens)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    out = differential_attention(*leaves, is_causal=causal, valid_len=lengths)
    grads = torch.autograd.grad(out, leaves, dout)
    want = attention(q, k, v, lam, causal=causal, lengths=lengths, dout=dout)
    assert_within(out, want["out"], "out", FLOOR[q.dtype])
    for name, got in zip(("dq", "dk", "dv", "dlam"), grads):
        assert_within(got, want[name], name, FLOOR[q.dtype] if name != "dlam" else 1e-40)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_weight_sums_over_heads(cuda, dtype):
    from techjam_amd.kernels import differential_attention

    q, k, v, lam, dout = inputs(TYPES[dtype], 2, 4, 2, 50, 32, 64, seed=2, shared=True)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    out = differential_attention(*leaves, is_causal=True)
    dlam = torch.autograd.grad(out, leaves, dout)[3]
    want = attention(q, k, v, lam, causal=True, dout=dout)["dlam"]
    assert dlam.shape == ()
    assert_within(dlam, (want[0].sum(), want[1].sum()), "dlam")


# b, h, hk, new, capacity, d, dv, lengths
CACHES = {
    "first_token": (2, 2, 2, 1, 16, 64, 128, (1, 1)),
    "one": (1, 8, 8, 1, 300, 64, 128, (257,)),
    "ragged": (4, 4, 1, 1, 900, 64, 128, (900, 1, 0, 333)),
    "few": (2, 6, 2, 5, 400, 32, 64, (400, 3)),
    "past_the_end": (2, 2, 1, 1, 64, 32, 64, (70, -3)),
    "wide": (1, 4, 1, 2, 200, 128, 256, (199,)),
    "rows_of_two_tiles": (2, 4, 1, 16, 270, 64, 128, (270, 40)),
    "a_chunk": (2, 2, 1, 90, 700, 64, 128, (700, 95)),
    "a_chunk_in_parts": (2, 4, 2, 90, 4500, 64, 128, (4500, 600)),
    "a_chunk_in_a_long_cache": (3, 2, 1, 70, 3000, 128, 256, (90, 0, 2999)),
    "odd_dims": (2, 2, 2, 1, 130, 40, 80, (130, 99)),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", CACHES)
def test_cached(cuda, shape, dtype):
    from techjam_amd.kernels import differential_attention_cached

    b, h, hk, new, cap, d, dv, lens = CACHES[shape]
    g = torch.Generator().manual_seed(3)
    t = TYPES[dtype]
    q = heads(g, b, 2 * h, new, d, t, 1.5)
    k = torch.randn(b, 2 * hk, cap, d, generator=g).to(t).cuda()
    v = torch.randn(b, hk, cap, dv, generator=g).to(t).cuda()
    lam = torch.rand(h, generator=g).cuda()
    lengths = lengths_of(*lens)
    want = attention(q, k, v, lam, causal=True, lengths=lengths, cached=True)["out"]
    for i, n in enumerate(lens):  # what lies behind a sequence's end is not read
        k[i, :, max(n, 0):] = float("nan")
        v[i, :, max(n, 0):] = float("inf")
    out = differential_attention_cached(q, k, v, lam, lengths)
    assert_within(out, want, "out", FLOOR[t])


@pytest.mark.parametrize("dtype", TYPES)
def test_padding_is_not_read(cuda, dtype):
    from techjam_amd.kernels import differential_attention

    t = TYPES[dtype]
    q, k, v, lam, dout = inputs(t, 3, 2, 1, 140, 64, 128, seed=4)
    lens = (140, 61, 0)
    lengths = lengths_of(*lens)
    want = attention(q, k, v, lam, causal=False, lengths=lengths, dout=dout)
    for i, n in enumerate(lens):
        for x, bad in ((q, "nan"), (k, "inf"), (v, "nan"), (dout, "nan")):
            x[i, :, n:] = float(bad)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, lam)]
    out = differential_attention(*leaves, valid_len=lengths)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, got in zip(("out", "dq", "dk", "dv", "dlam"), (out, *grads)):
        assert_within(got, want[name], name, FLOOR[t] if name != "dlam" else 1e-40)


# b, h, hk, capacity, lengths: how the keys are cut depends on all of a batch's lengths
BATCHES = {
    "past_a_wave_of_sequences": (150, 2, 1, 80, [(37 * i) % 81 if i % 5 else 0 for i in range(150)]),
    "one_long_among_short": (9, 2, 2, 5000, [3, 1, 0, 5000, 2, 31, 32, 33, 64]),
    "last_alone": (70, 1, 1, 300, [0] * 69 + [300]),
    "equal": (16, 4, 1, 2048, [2048] * 16),
    "short_in_a_long_cache": (3, 4, 2, 40000, [700, 701, 40]),
    "more_than_run_at_once": (40, 32, 32, 70, [(13 * i) % 71 for i in range(40)]),
    "two_waves_of_sequences": (128, 1, 1, 200, [(53 * i) % 201 for i in range(128)]),
    "all_empty": (3, 2, 1, 64, [0, 0, 0]),
    "no_capacity": (2, 2, 1, 0, [0, 5]),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", BATCHES)
def test_cached_batches(cuda, shape, dtype):
    from techjam_amd.kernels import differential_attention_cached

    b, h, hk, cap, lens = BATCHES[shape]
    d, dv = 64, 128
    g = torch.Generator().manual_seed(6)
    t = TYPES[dtype]
    q = heads(g, b, 2 * h, 1, d, t, 1.5)
    k = torch.randn(b, 2 * hk, cap, d, generator=g).to(t).cuda()
    v = torch.randn(b, hk, cap, dv, generator=g).to(t).cuda()
    lam = torch.rand(h, generator=g).cuda()
    lengths = lengths_of(*lens)
    want = attention(q, k, v, lam, causal=True, lengths=lengths, cached=True)["out"]
    for i, n in enumerate(lens):
        k[i, :, n:] = float("nan")
        v[i, :, n:] = float("nan")
    out = differential_attention_cached(q, k, v, lam, lengths)
    assert_within(out, want, "out", FLOOR[t])
    assert torch.equal(out, differential_attention_cached(q, k, v, lam, lengths))


# Launches that fill the chip run other workgroups than those above. Heads are
# independent: the first, a middle and the last key head are compared.
# b, h, hk, s, d, dv, causal, lengths
MANY_HEADS = {
    "64_rows_d64": (3, 44, 44, 70, 64, 128, True, (70, 33, 0)),
    "64_rows_d32": (2, 80, 40, 66, 32, 64, False, None),
    "64_rows_d128": (2, 90, 90, 70, 128, 256, True, (70, 65)),
    "128_rows_d64": (8, 64, 64, 130, 64, 128, True, None),
    "128_rows_d64_shared": (8, 128, 64, 70, 64, 128, False, (70, 1, 33, 64, 65, 0, 69, 70)),
    "128_rows_d32": (8, 64, 64, 130, 32, 64, True, (130, 129, 128, 97, 96, 1, 0, 64)),
    "128_rows_d128": (4, 32, 32, 130, 128, 256, False, (130, 129, 0, 33)),
    "128_rows_d128_causal": (4, 64, 64, 130, 128, 256, True, None),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", MANY_HEADS)
def test_many_heads(cuda, shape, dtype):
    from techjam_amd.kernels import differential_attention

    b, h, hk, s, d, dv, causal, lens = MANY_HEADS[shape]
    q, k, v, lam, dout = inputs(TYPES[dtype], b, h, hk, s, d, dv, seed=8)
    lengths = None if lens is None else lengths_of(*lens)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, lam)]
    out = differential_attention(*leaves, is_causal=causal, valid_len=lengths)
    dq, dk, dvv, dlam = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        plain = differential_attention(q, k, v, lam, is_causal=causal, valid_len=lengths)
    for kv in (0, hk // 2, hk - 1):
        g = h // hk
        heads_of = slice(kv * g, (kv + 1) * g)
        pairs, key_pair = slice(2 * kv * g, 2 * (kv + 1) * g), slice(2 * kv, 2 * kv + 2)
        want = attention(q[:, pairs], k[:, key_pair], v[:, kv:kv + 1], lam[heads_of], causal=causal, lengths=lengths,
                         dout=dout[:, heads_of])
        assert_within(out[:, heads_of], want["out"], "out", FLOOR[q.dtype])
        assert_within(plain[:, heads_of], want["out"], "out without gradients", FLOOR[q.dtype])
        assert_within(dq[:, pairs], want["dq"], "dq", FLOOR[q.dtype])
        assert_within(dk[:, key_pair], want["dk"], "dk", FLOOR[q.dtype])
        assert_within(dvv[:, kv:kv + 1], want["dv"], "dv", FLOOR[q.dtype])
        assert_within(dlam[heads_of], want["dlam"], "dlam", 1e-40)
