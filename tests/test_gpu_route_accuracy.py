"""Softmax weights, probabilities and gradients of the routing kernels far below the token's largest logit, against 64 bits."""
import pytest
import torch

from distdl_b200.ops import moe

pytestmark = pytest.mark.gpu

# exponential 2^-21 in the term and in the sum, 13 additions and a product of fp32, a division within 2^-22
REL = 2.0 ** -19


@pytest.mark.parametrize("how", [dict(), dict(renormalize=False), dict(bias="zero")], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k", [(65, 8), (128, 32), (256, 8), (512, 32)])
def test_small_probabilities_are_as_exact_as_large_ones(E, k, dtype, how):
    g = torch.Generator().manual_seed(E)
    how = dict(how)
    if "bias" in how:
        how["bias"] = torch.zeros(E, device="cuda")
    seen = 0.0
    for _ in range(8):
        # (eighths: their differences are exact)
        l = (torch.randn(1, E, generator=g) * 80).round().div(8).to(torch.bfloat16).to(dtype).cuda().requires_grad_()
        w, p, ids, _, _ = moe.route(l, E, k, 9, **how)
        l64 = l.detach().double().requires_grad_()
        p64 = torch.softmax(l64, -1)[0]
        w64 = p64[ids.long()]
        w64 = w64 / w64.sum() if how.get("renormalize", True) else w64
        assert ((p.double() - p64).abs() <= REL * p64 + 1e-37).all()
        assert ((w[0].double() - w64).abs() <= REL * w64 + 1e-37).all()
        seen = max(seen, (l64.max() - l64.min()).item())
        q = torch.randn(E, generator=g).cuda()
        d, = torch.autograd.grad(p, l, q)
        want = (p64 * (q.double() - (p64 * q).sum())).detach()
        size = p64.detach() * 2 * q.abs().max()
        # (both of p's errors, and a sum of products over the experts: 13 additions)
        assert ((d[0].double() - want).abs() <= (torch.finfo(dtype).eps / 2) * want.abs() + 4 * REL * size + 1e-37).all()
    assert seen > 40
