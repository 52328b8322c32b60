"""Differential attention and layer norm: calls at the edges of what they allow, on the kernels (GPU)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_the_last_token_of_a_long_sequence(cuda, dtype):
    """One row whose stride is the whole sequence's, forward and backward: a compact row's bits."""
    from techjam_amd.kernels import layer_norm

    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.empty(1, 32768, 1024, dtype=dtype, device="cuda")[:, -1] for _ in range(2))
    x.normal_(generator=g)
    dy.normal_(generator=g)
    assert x.stride(0) == 1 << 25 and dy.stride(0) == 1 << 25
    w, b = torch.randn(1024, generator=g, device="cuda"), torch.randn(1024, generator=g, device="cuda")

    def run(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    for got, want in zip(run(x, dy), run(x.clone(memory_format=torch.contiguous_format), dy.clone())):
        assert torch.equal(got, want)
