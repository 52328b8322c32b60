"""Attention with grouped heads where its numbers and memory go wrong first: small values, bad offsets, gradients (GPU)."""

from __future__ import annotations

import pytest
import torch

from grouped_reference import check, packed
from test_grouped_gpu import inputs, norm_of, run_packed
from test_grouped_use_gpu import draft_inputs, run_tree

pytestmark = pytest.mark.gpu


# -- values at the lower end of a type -------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size,loss_scale", [(1e-4, 2.0 ** 13), (1e-5, 2.0 ** 14), (1e-6, 2.0 ** 14)])
def test_gradients_of_small_values(dtype, causal, size, loss_scale):
    """Values that small leave outputs below fp16's smallest normal number, 2^-14, whose own bits (they are multiples
    of 2^-24) are too few for delta = dO . O: with the output alone, or a rest that is lost below 2^-24, delta is off by
    2^-25 an element, which at 1e-5 is 2e-3 of dQ and at 1e-6 2e-2. The gradients themselves are normal numbers,
    as under a scaled loss, and are held to what they are held to elsewhere."""
    q, k, v, dout = inputs(500, 2, 1, 64, 64, dtype, seed=9)
    v, dout = (v.float() * size).to(dtype), (dout.float() * loss_scale).to(dtype)
    got = run_packed(q, k, v, [0, 200, 500], causal, dout)
    for name, (value, bound) in packed(q, k, v, [0, 200, 500], causal, None, None, dout).items():
        # The output of fp16 is as far off as its steps of 2^-24 are wide: check adds them to its bound.
        check(name, got[name], value, bound, None if name == "out" else norm_of(dtype))


# -- strides -----------------------------------------------------------------------

def test_new_tokens_whose_heads_are_far_apart():
    """Heads 2^31 elements apart, and one head with such a stride, give what the same tokens side by side give."""
    b, h, t, d = 2, 2, 3, 64
    q, k, v = draft_inputs(b, h, 1, t, 300, d, torch.float16)
    parents = [[-1, 0, 0]] * b
    want = run_tree(q, k, v, [300, 120], parents)
    big = torch.empty((1 << 31) + 64 + b * t * d, dtype=torch.float16, device="cuda")
    far = big.as_strided((b, h, t, d), (t * d, (1 << 31) + 64, d, 1)).copy_(q)
    assert torch.equal(run_tree(far, k, v, [300, 120], parents), want)
    one = big.as_strided((b, 1, t, d), (t * d, 1 << 33, d, 1))
    assert torch.equal(run_tree(one, k, v, [300, 120], parents), run_tree(q[:, :1].contiguous(), k, v, [300, 120], parents))


# -- states ----------------------------------------------------------------------

def test_accepting_is_not_captured():
    from techjam_amd import UnsupportedCaseError
    from test_grouped_model_gpu import encoder

    model, x, _ = encoder()
    state = model.new_state(3, 12)
    x = x.cuda()
    path, counts = torch.tensor([[0, 1]] * 3).cuda(), torch.tensor([2, 1, 0]).cuda()
    with torch.no_grad():
        model.prefill(x[:, :8], state)
        model.step(x[:, :2], state, torch.tensor([[-1, 0]] * 3, dtype=torch.int32).cuda())
        graph = torch.cuda.CUDAGraph()
        with torch.inference_mode(), torch.cuda.graph(graph), pytest.raises(UnsupportedCaseError, match="captured"):
            state.accept(path, counts)
        assert state.lengths.tolist() == [8, 8, 8] and state.longest == 8 and state.drafts == 2
        state.accept(path, counts)
        assert state.lengths.tolist() == [10, 9, 8] and state.longest == 10 and state.drafts == 0


def test_prompts_are_not_rounded_into_a_cache_of_another_type():
    from test_grouped_model_gpu import encoder

    model, x, lengths = encoder()
    mask = (torch.arange(x.shape[1])[None, :] < lengths[:, None]).cuda()
    with torch.no_grad():
        for dtype in (torch.float16, torch.bfloat16):
            state = model.new_state(3, 50, dtype)
            with pytest.raises(ValueError, match="create the state in that dtype"):
                model.prefill(x.cuda(), state, mask)
            assert not state.lengths.any() and state.longest == 0
            with torch.autocast("cuda", dtype):  # whose projections have that type
                model.prefill(x.cuda(), state, mask)
                assert model.step(x.cuda()[:, :1], state).isfinite().all()
            assert state.lengths.tolist() == [n + 1 for n in lengths.tolist()]
