"""States and arguments of grouped attention that would lose or overwrite what a program holds (no GPU needed)."""

from __future__ import annotations

import random
import sys

import pytest
import torch

from techjam_amd import UnsupportedCaseError
from test_grouped_host import model

kernels = sys.modules["techjam_amd.kernels.grouped"]


# -- what a graph's replay would not count ----------------------------------------

def test_accept_and_recount_are_not_captured(monkeypatch):
    """A replayed accept moves the lengths on the device and not their bound on the host, so that the next step would
    write past a full cache."""
    state = model().new_state(2, 8)
    state.lengths.fill_(4)
    state.longest = 4
    state.drafts = 2
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(UnsupportedCaseError, match="captured"):
        state.accept(torch.zeros(2, 1, dtype=torch.long), torch.ones(2, dtype=torch.long))
    with pytest.raises(UnsupportedCaseError, match="captured"):
        state.recount()
    assert state.lengths.tolist() == [4, 4] and state.longest == 4 and state.drafts == 2
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    state.accept(torch.zeros(2, 1, dtype=torch.long), torch.ones(2, dtype=torch.long))
    state.recount()
    assert state.lengths.tolist() == [5, 5] and state.longest == 5


# -- caches of another type --------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float64])
def test_first_tokens_are_not_rounded_into_a_cache_of_another_type(dtype):
    """The step that follows would be refused, with the prompts already rounded."""
    m = model()
    cache = m.new_state(2, 8, dtype).layers[0]
    cache.k.fill_(7)
    cache.v.fill_(7)
    attention, lengths = m.layers[0].attention, torch.full((2,), 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="create the state in that dtype"):
        attention(torch.randn(2, 4, 32), None, True, lengths, cache)
    with pytest.raises(ValueError, match="create the state in that dtype"):
        attention.step(torch.randn(2, 1, 32), cache, lengths, torch.full((2, 1), 3))
    assert (cache.k == 7).all() and (cache.v == 7).all()


# -- strides past what the kernels multiply ------------------------------------------

def _far(shape, strides):
    n = sum((a - 1) * b for a, b in zip(shape, strides)) + 1
    t = torch.empty(n, dtype=torch.float16).as_strided(shape, strides)  # memory that is never touched takes none
    t.copy_(torch.randn(shape, generator=torch.Generator().manual_seed(0)))
    return t


@pytest.mark.parametrize("shape,strides,in_place", [
    ((2, 4, 3, 64), (768, 64, 256, 1), True),                    # a projection's
    ((1, 2, 3, 64), (64, (1 << 31) + 64, 64, 1), False),         # heads too far apart for 32 bits
    ((1, 2, 3, 64), (64, (1 << 31) - 64, 64, 1), True),
    ((2, 1, 3, 64), (192, (1 << 33) + 1, 64, 1), True),          # one head: its stride is never used
    ((2, 1, 3, 64), (192, 1 << 33, 64, 1), True),
    ((2, 2, 1, 64), ((1 << 31) + 64, 64, 1 << 33, 1), True),     # sequences may be as far apart as they like
])
def test_new_tokens_are_read_in_place_where_they_can_be(shape, strides, in_place):
    t = _far(shape, strides)
    seen = kernels._queries_view(t)
    assert torch.equal(seen, t) and (seen.data_ptr() == t.data_ptr()) == in_place
    sb, sh, ss, sd = seen.stride()
    assert sd == 1 and not (sb | sh | ss) % 8 and seen.data_ptr() % 16 == 0 and sh < 1 << 31 and ss * 64 * 2 < 1 << 31


# -- packed prompts ------------------------------------------------------------------

@pytest.mark.parametrize("offsets", [
    torch.tensor([0, 3, 8]),                                    # int64
    torch.tensor([0.0, 3.0, 8.0]), torch.tensor([0, 9, 3, 9, 8, 9], dtype=torch.int32)[::2], [0, 3, 8], None])
def test_offsets_of_another_kind_leave_the_state_as_it_was(offsets):
    """They are refused before the state is emptied, as offsets of the wrong values are."""
    m = model()
    state = m.new_state(2, 8)
    state.lengths.fill_(6)
    state.longest, state.drafts = 6, 2
    with pytest.raises(ValueError, match="offsets"):
        m.prefill_packed(torch.zeros(8, 32), offsets, state)
    assert state.lengths.tolist() == [6, 6] and state.longest == 6 and state.drafts == 2
    with pytest.raises(ValueError, match="offsets"):
        m.forward_packed(torch.zeros(8, 32), offsets)


@pytest.mark.parametrize("offsets", [torch.zeros(0, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32),
                                     torch.tensor(0, dtype=torch.int32), torch.zeros(3, dtype=torch.int32, device="meta")])
def test_offsets_of_another_shape_or_place_are_refused(offsets):
    for m in (model(), model(layers=0)):
        with pytest.raises(ValueError, match="offsets"):
            m.forward_packed(torch.zeros(8, 32), offsets)


# -- operands ------------------------------------------------------------------------

def test_fp16_operands_are_refused_everywhere():
    """They are the fused softmax encoder's; the padded forward pass says so, and the others would take float32."""
    m = model()
    state = m.new_state(2, 8)
    state.lengths.fill_(6)
    state.longest, state.drafts = 6, 2
    m.gemm_operands = "fp16"
    offsets = torch.tensor([0, 3, 8], dtype=torch.int32)
    for call in (lambda: m(torch.zeros(2, 8, 32)), lambda: m.forward_packed(torch.zeros(8, 32), offsets),
                 lambda: m.prefill_packed(torch.zeros(8, 32), offsets, state), lambda: m.prefill(torch.zeros(2, 4, 32), state),
                 lambda: m.step(torch.zeros(2, 1, 32), state),
                 lambda: m.step(torch.zeros(2, 1, 32), state, torch.full((2, 1), -1, dtype=torch.int32))):
        with pytest.raises(UnsupportedCaseError, match="fp16 GEMM operands"):
            call()
    assert state.lengths.tolist() == [6, 6] and state.longest == 6 and state.drafts == 2
    m.gemm_operands = "bf16"
    with pytest.raises(ValueError, match="gemm_operands"):
        m.forward_packed(torch.zeros(8, 32), offsets)


# -- offsets out of order ----------------------------------------------------------------

def test_offsets_out_of_order_reach_nothing_outside():
    """Whatever region and tile a workgroup finds: with offsets clipped to 0 .. T and the tile's rows checked against the
    region's, as the kernels do both, its rows, their numbers and their peaks lie within what is allocated."""
    rng = random.Random(2)
    lists = [[0, 500, 100, 200], [-50, 20, 10, 1 << 30], [150, 100, 50, 0], [(1 << 31) - 1, -(1 << 31), 7] * 30]
    lists += [[rng.randint(-300, 700) for _ in range(rng.randint(1, 60))] for _ in range(200)]
    for offsets in lists:
        t, n = rng.choice((1, 63, 64, 200, 500)), len(offsets) - 1
        edges = [0] + [min(t, max(0, x)) for x in offsets] + [t]
        for j in range(n + 2):
            start, rows = edges[j], max(0, edges[j + 1] - edges[j])
            assert 0 <= start and start + rows <= t
            for unit in (32, 64):  # the numbers of 32 tokens, the peaks of 64
                assert rows == 0 or start // unit + j + (rows - 1) // unit < t // unit + n + 2
            for per, unit in ((1, 64), (2, 32), (3, 128), (8, 64)):
                for tile in range(-(-rows * per // unit)):  # those that there() lets through
                    first, last = tile * unit // per, min(rows * per, (tile + 1) * unit) - 1
                    assert first < rows and last // per < rows
