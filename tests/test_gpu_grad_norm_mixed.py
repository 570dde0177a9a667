"""Gradients that the kernels do not take among others that they do."""
import math

import pytest
import torch

from distdl_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("odd", ["fp64", "holes"])
def test_one_odd_tensor_among_many(odd, first):
    torch.manual_seed(0)
    g = [torch.randn(1 << 25, device="cuda"), torch.randn(1000, device="cuda").to(torch.bfloat16),
         torch.randn(77, device="cuda").to(torch.float16)]
    one = torch.randn(500, device="cuda", dtype=torch.float64) if odd == "fp64" else torch.randn(50, 20, device="cuda")[:, ::2]
    g.insert(0 if first else 2, one)
    before = [t.double().clone() for t in g]
    want = math.sqrt(sum(t.square().sum().item() for t in before))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    norm = ops.grad_norm(g)
    squared = ops.grad_norm(g, squared=True)
    clipped = ops.clip_grad_norm_(g, 0.25 * want)
    again = ops.clip_grad_norm_(g, 0.125 * want, norm=torch.full((), 0.25 * want, device="cuda"))
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held < 1 << 24         # (128 MB of gradients: no copies of them)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want and torch.equal(norm, clipped) and again.dtype == torch.float32
    assert abs(squared.item() - want * want) <= 2.0 ** -40 * want * want
    for t, b in zip(g, before):
        ref = b * (0.25 * want / (norm.item() + 1e-6)) * (0.125 * want / (torch.tensor(0.25 * want).item() + 1e-6))
        # twice a factor, a product and a rounding to the type
        bound = 2 * (torch.finfo(t.dtype).eps / 2 + 2.0 ** -22) * ref.abs() + (2.0 ** -24 if t.dtype == torch.float16 else 1e-37)
        assert ((t.double() - ref).abs() <= bound).all()
