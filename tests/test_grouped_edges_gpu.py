"""Attention with grouped heads where its numbers and memory go wrong first: small values, bad offsets, gradients (GPU)."""

from __future__ import annotations

import pytest
import torch

from grouped_reference import check, packed
from test_grouped_gpu import inputs, norm_of, run_packed

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
