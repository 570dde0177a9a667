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


class _Elsewhere(torch.Tensor):
    """A tensor whose elements are those of another one, doubled."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.copy_.default and isinstance(args[0], cls):
            args[0].inner.copy_(args[1] / 2)
            return args[0]
        return func(*[a.inner * 2 if isinstance(a, cls) else a for a in args], **(kwargs or {}))


@pytest.mark.parametrize("place", [0, 1, 2])
def test_a_subclass_is_not_taken_by_its_address_wherever_it_stands(place, monkeypatch):
    from distdl_b200.ops import optim
    tensors = [torch.ones(3), torch.ones(2), torch.ones(4)]
    inner = tensors[place].clone()
    tensors[place] = _Elsewhere(inner)
    n = inner.numel()
    want = torch.tensor(9.0 - n + 4.0 * n).sqrt()
    assert torch.allclose(ops.grad_norm(tensors), want)
    assert torch.allclose(ops.clip_grad_norm_(tensors, 1.0), want) and torch.allclose(inner, torch.ones(n) / want)
    monkeypatch.setattr(optim, "use_native", lambda t: True)
    assert optim._tensors(tensors) is None
    tensors[place] = inner
    assert optim._tensors(tensors) is not None
