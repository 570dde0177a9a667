"""Pairs without a slot take nothing from the expert rows that they do not have (CPU; on a GPU: the kernels)."""
import math

import pytest
import torch

from distdl_b200.ops import moe


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_that_are_no_numbers_stay_with_their_tokens(device):
    T, E, k, C, d = 4, 2, 2, 4, 8
    logits = torch.tensor([[2.0, 1.0], [1.0, -math.inf], [-math.inf, -math.inf], [0.0, 3.0]], device=device)
    logits.requires_grad_()
    w, _, ids, slot, _ = moe.route(logits, E, k, C)
    x = torch.ones(T, d, device=device, dtype=torch.bfloat16)
    x[0] = math.nan                                           # the first row of both experts
    y = moe.combine(moe.dispatch(x, ids, slot, E, C, k), w, ids, slot, T, k)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all() and (y[2] == 0).all()
    assert torch.allclose(y[[1, 3]].float(), torch.ones(2, d, device=device), atol=2.0 ** -8)
    d, = torch.autograd.grad(y[1:].float().sum(), logits)
    assert torch.isfinite(d[1:]).all() and (d[2] == 0).all()
