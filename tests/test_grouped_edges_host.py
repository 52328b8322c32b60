"""States and arguments of grouped attention that would lose or overwrite what a program holds (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from techjam_amd import UnsupportedCaseError
from test_grouped_host import model


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
