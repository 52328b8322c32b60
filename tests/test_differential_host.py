"""Refusals of differential attention and layer norm that need no GPU."""

from __future__ import annotations

import pytest
import torch

from techjam_amd import UnsupportedCaseError
from techjam_amd.kernels import LayerNorm, differential_attention, differential_attention_cached, layer_norm


def qkv(b=1, h=2, hk=2, s=8, sk=None, d=32, dv=64, dtype=torch.float32):
    sk = s if sk is None else sk
    return (torch.zeros(b, 2 * h, s, d, dtype=dtype), torch.zeros(b, 2 * hk, sk, d, dtype=dtype),
            torch.zeros(b, hk, sk, dv, dtype=dtype), torch.zeros(h))


def test_there_is_no_cpu_implementation():
    with pytest.raises(UnsupportedCaseError):
        differential_attention(*qkv())
    with pytest.raises(UnsupportedCaseError):
        differential_attention_cached(*qkv(sk=16), torch.ones(1, dtype=torch.int32))
    with pytest.raises(UnsupportedCaseError):
        layer_norm(torch.zeros(2, 8))


@pytest.mark.parametrize("change,error", [
    (dict(d=129), UnsupportedCaseError),
    (dict(dv=257), UnsupportedCaseError),
    (dict(dtype=torch.float64), UnsupportedCaseError),
    (dict(h=3, hk=2), ValueError),
    (dict(sk=9), ValueError),
])
def test_attention_refuses(change, error):
    with pytest.raises(error):
        differential_attention(*qkv(**change))


def test_attention_refuses_shapes_and_weights_that_do_not_fit():
    q, k, v, lam = qkv()
    for bad in ((q[0], k, v, lam), (q[:, :3], k, v, lam), (q, k[:, :2], v, lam), (q, k, v[:, :, :4], lam),
                (q, k.half(), v, lam), (q, k, v, lam[:1].expand(3)), (q, k, v, lam.int()), (q, k, v, 0.5),
                (q[:, :0], k, v, lam[:0]), (q, k[..., :16], v, lam), (q.expand(2, -1, -1, -1), k, v, lam)):
        with pytest.raises(ValueError):
            differential_attention(*bad)


def test_cached_refuses():
    q, k, v, lam = qkv(s=1, sk=16)
    with pytest.raises(ValueError):
        differential_attention_cached(q, k, v, lam, None)


def test_norm_refuses():
    x = torch.zeros(2, 8)
    with pytest.raises(UnsupportedCaseError):
        layer_norm(torch.zeros(2, 16385))
    with pytest.raises(UnsupportedCaseError):
        layer_norm(x.double())
    for bad in (torch.zeros(()), torch.zeros(2, 0)):
        with pytest.raises(ValueError):
            layer_norm(bad)
    with pytest.raises(UnsupportedCaseError):  # the device comes first
        layer_norm(x, norm_dtype=torch.float16)
    with pytest.raises(ValueError):
        LayerNorm((2, 8))
    with pytest.raises(ValueError):
        LayerNorm(8)(torch.zeros(2, 9))


def test_layer_norm_module_has_torchs_parameters():
    own, torchs = LayerNorm(8), torch.nn.LayerNorm(8)
    own.load_state_dict(torchs.state_dict())
    assert isinstance(own, torch.nn.LayerNorm) and own.normalized_shape == (8,)


def test_entry_points_refuse_before_launching():
    from techjam_amd.kernels import _lib

    L = _lib.lib()
    st = (_lib.ctypes.c_int64 * 4)(4 * 64 * 64, 64 * 64, 64, 1)
    p = 4096  # never dereferenced

    def fwd(dtype=_lib.TJ_F16, h=2, hk=2, sq=16, sk=16, d=64, dv=64, cached=0, lengths=None, ws=None, nb=0, b=1):
        return L.tj_diff_attn_fwd(p, p, p, p, dtype, b, h, hk, sq, sk, d, dv, st, st, st, st, 0.125, 1, cached, p, 1,
                                  lengths, None, None, ws, nb, None)

    assert fwd(dtype=9) == _lib.TJ_ERR_DTYPE
    assert fwd(h=3) == _lib.TJ_ERR_SHAPE
    assert fwd(sk=17) == _lib.TJ_ERR_SHAPE
    assert fwd(d=160) == _lib.TJ_ERR_UNSUPPORTED
    assert fwd(d=12) == _lib.TJ_ERR_ALIGN
    assert fwd(sq=1, sk=4096, cached=1) == _lib.TJ_ERR_SHAPE
    assert fwd(sq=1, sk=4096, cached=1, lengths=p) == _lib.TJ_ERR_WORKSPACE
    assert fwd(b=0) == _lib.TJ_OK
    # The workspace covers the parts; whole long sequences over many heads need none.
    assert L.tj_diff_attn_workspace_bytes(1, 2, 2, 1, 4096, 64, 1) > 0
    assert L.tj_diff_attn_workspace_bytes(64, 16, 16, 4096, 4096, 128, 0) == 0
    # existing entry points do not take bfloat16
    assert L.tj_attn_fwd(p, p, p, p, _lib.TJ_BF16, 1, 4, 128, 64, st, st, st, st, 0.125, 1, None, None, None, None) == _lib.TJ_ERR_DTYPE


def test_refused_steps_leave_the_state_as_it_was():
    from techjam_amd.model import TransformerConfig, TransformerEncoder

    def model(layers=2, heads=2):
        return TransformerEncoder(TransformerConfig(2, 8, 16, heads, 32, layers, True, attention="differential"))

    m = model()
    state = m.new_state(2, 8)
    state.lengths.fill_(6)
    state.longest = 6
    for x in (torch.zeros(1, 9, 16), torch.zeros(1, 1, 16), torch.zeros(2, 9, 16), torch.zeros(2, 1, 8), torch.zeros(2, 16)):
        with pytest.raises(ValueError):  # another batch would spread over the caches' rows; 9 exceed the capacity
            m.prefill(x, state)
    for x in (torch.zeros(1, 1, 16), torch.zeros(2, 3, 16), torch.zeros(2, 0, 16)):
        with pytest.raises(ValueError):
            m.step(x, state)
    for other in (model(layers=3), model(heads=4)):
        with pytest.raises(ValueError):
            m.step(torch.zeros(2, 1, 16), other.new_state(2, 8))
    # A call that is refused on its way (here: no kernels for CPU tensors) counts no tokens.
    with pytest.raises(UnsupportedCaseError):
        m.step(torch.zeros(2, 1, 16), state)
    assert state.lengths.tolist() == [6, 6] and state.longest == 6
    with pytest.raises(UnsupportedCaseError):
        m.prefill(torch.zeros(2, 8, 16), state)
    assert state.lengths.tolist() == [0, 0] and state.longest == 0


def test_cache_without_room_is_refused_past_the_grid():
    from techjam_amd.kernels import _lib

    L = _lib.lib()
    st = (_lib.ctypes.c_int64 * 4)(64, 64, 64, 1)
    p, rows = 4096, 1 << 20
    # 2^20 sequences of 16 tokens against caches of no capacity: a workgroup per row, 2^24 of them.
    assert L.tj_diff_attn_fwd(p, p, p, p, _lib.TJ_F16, rows, 1, 1, 16, 0, 64, 64, st, st, st, st, 0.125, 1, 1, p, 1, p,
                              None, None, None, 0, None) == _lib.TJ_ERR_SHAPE
