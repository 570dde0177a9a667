"""Gradients below the smallest normal number count in the norm and are scaled as any others."""
import math

import pytest
import torch

from distdl_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [7, 1 << 20])
@pytest.mark.parametrize("dtype,value", [(torch.float32, 1e-39), (torch.bfloat16, 1e-39), (torch.float16, 6e-7),
                                         (torch.float32, 1e-44), (torch.bfloat16, 2.0 ** -133)])
def test_small_gradients(dtype, value, n):
    g = torch.full((n,), value, device="cuda", dtype=dtype)
    want = math.sqrt(g.double().square().sum().item())
    assert 0 < want and abs(ops.grad_norm([g], squared=True).item() - want * want) <= 2.0 ** -40 * want * want
    # one rounding to fp32: half a step, below 2^-126 that of 2^-149
    assert abs(ops.grad_norm([g]).item() - want) <= max(2.0 ** -24 * want, 2.0 ** -150) * (1 + 1e-6)
    big = torch.full((4,), 2.0, device="cuda")
    kept = g.double()
    norm = ops.clip_grad_norm_([g, big], 3.0)
    scale = 3.0 / (norm.item() + 1e-6)
    # the factor and the product rounded to fp32, then to the type
    step = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    err = (g.double() - kept * scale).abs().max().item()
    assert err <= kept.max().item() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22) + 0.5 * step + 2.0 ** -149
    # a largest norm below the normal numbers
    ops.clip_grad_norm_([big], 1e-39)
    assert abs(big[0].item() - 0.5e-39) <= 0.5e-39 * 2.0 ** -7
