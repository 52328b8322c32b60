"""Differential attention and layer norm: calls at the edges of what they allow, without a GPU."""

from __future__ import annotations

import sys

import pytest
import torch
from torch.autograd import forward_ad

from techjam_amd import UnsupportedCaseError
from techjam_amd.kernels import LayerNorm, _lib, differential_attention, differential_attention_cached, layer_norm
from techjam_amd.model import EncoderBlock, TransformerConfig, TransformerEncoder

attention_kernels = sys.modules["techjam_amd.kernels.differential"]
norm_kernels = sys.modules["techjam_amd.kernels.layer_norm"]  # the package's attribute is the function


def attention_inputs(sq=4, sk=4):
    return torch.zeros(1, 4, sq, 32), torch.zeros(1, 4, sk, 32), torch.zeros(1, 2, sk, 64), torch.zeros(2)


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused_and_not_dropped(grad):
    """A dual tensor does not require grad: its output would come without a tangent."""
    lengths = torch.ones(1, dtype=torch.int32)
    norm = (torch.zeros(2, 8), torch.zeros(8), torch.zeros(8))
    module = LayerNorm(8)
    calls = [(layer_norm, norm), (differential_attention, attention_inputs()),
             (lambda *t: differential_attention_cached(*t, lengths), attention_inputs(1, 4)),
             (lambda x: module(x), norm[:1])]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for call, inputs in calls:
            for i, x in enumerate(inputs):
                dual = forward_ad.make_dual(x, torch.ones_like(x))
                with pytest.raises(UnsupportedCaseError, match="forward-mode"):
                    call(*inputs[:i], dual, *inputs[i + 1:])
                with torch.inference_mode(), pytest.raises(UnsupportedCaseError, match="GPU"):
                    call(*inputs[:i], dual, *inputs[i + 1:])  # no derivatives there: the device is what is refused
            with pytest.raises(UnsupportedCaseError, match="GPU"):
                call(*inputs)


@pytest.mark.parametrize("width,row_stride", [(2048, 8192 * 2048), (96, 1 << 40), (8, 3), (1, 1 << 30), (7, 0)])
@pytest.mark.parametrize("ndim", [1, 2, 3])
def test_a_single_row_has_no_row_stride(width, row_stride, ndim):
    """One row counts as contiguous whatever its stride, and the kernels take strides below 2^23."""
    t = torch.arange(width, dtype=torch.float32).as_strided((1,) * (ndim - 1) + (width,), (row_stride,) * (ndim - 1) + (1,))
    rows = norm_kernels._rows(t)
    assert rows.shape == (1, width) and rows.stride() == (width, 1) and rows.data_ptr() == t.data_ptr()
    assert torch.equal(rows[0], torch.arange(width))


def test_rows_far_apart_are_copied():
    two = torch.zeros(2).as_strided((2, 1), (1, 5)).expand(2, 4)
    assert norm_kernels._rows(two).stride() == (4, 1)
    far = torch.empty(1, device="meta").as_strided((2, 4), (1 << 23, 1))
    near = torch.empty(1, device="meta").as_strided((2, 4), ((1 << 23) - 1, 1))
    assert norm_kernels._rows(far).stride() == (4, 1)
    assert norm_kernels._rows(near).stride() == ((1 << 23) - 1, 1)
    assert norm_kernels._rows(torch.zeros(0, 4)).shape == (0, 4)


def _view(shape, strides, offset=0):
    n = offset + sum((a - 1) * b for a, b in zip(shape, strides)) + 1
    return torch.randn(n).half().as_strided(shape, strides, offset)


@pytest.mark.parametrize("shape,strides,in_place", [
    ((1, 1, 1, 64), (1027, 1027, 1027, 1), True),     # one token's value in a projection of odd width
    ((1, 2, 7, 64), (897, 448, 64, 1), True),         # a batch of one
    ((1, 2, 7, 64), (5, 64, 128, 1), True),           # the same, token by token in memory
    ((2, 1, 7, 64), (448, 3, 64, 1), True),           # one key head
    ((2, 2, 1, 64), (128, 64, 1 << 40, 1), True),     # one token
    ((1, 2, 7, 64), (897, 455, 65, 1), False),        # odd rows
    ((1, 1, 2, 64), (1, 1, 65, 1), False),
    ((1, 1, 1, 64), (1, 1, 1, 1), True),
    ((1, 1, 2, 64), (7, 7, 1 << 26, 1), False),       # rows too far apart
    ((0, 2, 1, 64), (3, 64, 7, 1), True),
    ((2, 2, 0, 64), (64, 128, 7, 1), True),           # a cache of no capacity
])
def test_strides_of_dimensions_of_one_do_not_count(shape, strides, in_place):
    if strides[2] == 1 << 26:
        t = torch.empty(1, device="meta").half().as_strided(shape, strides)
    else:
        t = _view(shape, strides) if 0 not in shape else torch.empty(1).half().as_strided(shape, strides)
    got = attention_kernels._rows_view(t)
    assert attention_kernels._readable(got) and got.shape == t.shape
    if t.device.type == "cpu":
        assert torch.equal(got, t)
        assert (got.data_ptr() == t.data_ptr()) == in_place or 0 in shape


def test_misaligned_single_tokens_are_copied():
    t = _view((1, 2, 1, 64), (1, 64, 1, 1), offset=1)
    got = attention_kernels._rows_view(t)
    assert attention_kernels._readable(got) and torch.equal(got, t)


@pytest.mark.parametrize("scale", [1e300, -3.5e38, 2.0 ** 127.5, float("inf"), float("nan")])
def test_scales_past_float32_are_refused(scale):
    """Handed on as a float32, 1e300 would be an infinity and every output NaN."""
    with pytest.raises(ValueError):
        attention_kernels._scale(scale, 64)


@pytest.mark.parametrize("scale", [0.0, -2.0 ** 127, 2.0 ** 127, 1e-300])
def test_scales_of_float32_are_taken(scale):
    assert attention_kernels._scale(scale, 64) == scale


@pytest.mark.parametrize("b,h,hk,sq,sk,fits", [
    (512, 32, 32, 1, 65536, True),       # 137 GB of keys and values at 32 dims in 16 bits
    (1, 64, 64, 1, 1 << 24, True),
    (2048, 8, 1, 1, 1 << 20, True),
    (128, 1, 1, 1, 1 << 29, False),      # more blocks of keys than are counted in 32 bits
    (1, 1, 1, 1, 1 << 30, False),
    (1 << 20, 16, 1, 1, 16, False),      # a workgroup per row: 2^24 of them
])
def test_how_large_caches_may_be(b, h, hk, sq, sk, fits):
    """What a call within the limits lacks here is its workspace; nothing is launched."""
    L = _lib.lib()
    st = (_lib.ctypes.c_int64 * 4)(64, 64, 64, 1)
    p = 4096  # never dereferenced
    code = L.tj_diff_attn_fwd(p, p, p, p, _lib.TJ_F16, b, h, hk, sq, sk, 32, 64, st, st, st, st, 0.125, 1, 1, p, 1, p,
                              None, None, None, 0, None)
    assert code == (_lib.TJ_ERR_WORKSPACE if fits else _lib.TJ_ERR_SHAPE)
    if fits:
        floats = L.tj_diff_attn_workspace_bytes(b, h, hk, sq, sk, 64, 1) // 4
        assert 0 < floats < 1 << 28


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_of_another_type_than_the_cache_are_refused(dtype):
    model = TransformerEncoder(TransformerConfig(2, 8, 16, 2, 32, 1, True, attention="differential"))
    cache = model.new_state(2, 8, dtype).layers[0]
    x = torch.zeros(2, 1, 16)
    lengths, place = torch.ones(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int64)
    attention = model.layers[0].attention
    with pytest.raises(ValueError, match="cache holds"):
        attention.step(x, cache, lengths, place)
    assert not bool(cache.k.any())
    with torch.autocast("cpu", dtype), pytest.raises(UnsupportedCaseError, match="GPU"):
        attention.step(x, cache, lengths, place)  # autocast's type is the cache's


def test_blocks_of_unknown_attention_are_refused():
    """Any word but "differential" would have built softmax attention."""
    with pytest.raises(ValueError, match="attention must be one of"):
        EncoderBlock(16, 2, 32, attention="differental")
    with pytest.raises(ValueError, match="attention must be one of"):
        TransformerEncoder(TransformerConfig(2, 8, 16, 2, 32, 1, True, attention="differental"))
