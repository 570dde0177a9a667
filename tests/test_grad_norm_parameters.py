"""Clipping by parameters: frozen ones stay as they are, and None is passed over."""
import pytest
import torch

from distdl_b200 import ops, parallel


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("clip", [ops.clip_grad_norm_, parallel.clip_grad_norm_])
def test_frozen_parameters_are_no_gradients(clip, device):
    model = torch.nn.Sequential(torch.nn.Linear(4, 3), torch.nn.Linear(3, 2)).to(device)
    model[0].requires_grad_(False)
    model(torch.randn(5, 4, device=device)).square().sum().backward()
    frozen = [p.detach().clone() for p in model[0].parameters()]
    grads = [p.grad.clone() for p in model[1].parameters()]
    want = torch.cat([g.flatten() for g in grads]).double().norm()
    norm = clip([None, *model.parameters(), None], 1e-3)
    assert torch.allclose(norm.double(), want)
    assert all(torch.equal(p, f) for p, f in zip(model[0].parameters(), frozen))
    assert all(torch.allclose(p.grad, g * (1e-3 / (norm + 1e-6))) for p, g in zip(model[1].parameters(), grads))
    # one that has a gradient from before it was frozen: that one
    model[1].requires_grad_(False)
    again = clip(model.parameters(), 1e9)
    assert torch.allclose(again, torch.tensor(1e-3, device=device), rtol=2e-3)
    assert clip([None], 1.0).item() == 0.0 and clip(model[0].parameters(), 1.0).item() == 0.0
    # gradients as they are
    g = torch.full((4,), 2.0, device=device)
    assert clip(g, 1.0).item() == 4.0 and torch.allclose(g, torch.full_like(g, 0.5))
