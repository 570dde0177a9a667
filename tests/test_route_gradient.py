"""The gradient of the routing kernels where nothing arrives (CPU: the launches are not reached)."""
import torch

from distdl_b200.ops import moe


class _Nothing(torch.autograd.Function):
    """A consumer that has no gradient for its input."""

    @staticmethod
    def forward(ctx, w, p):
        return w.sum() + p.sum()

    @staticmethod
    def backward(ctx, d):
        return None, None


def test_no_gradient_arrives(monkeypatch):
    def forward(logits, E, k, capacity, how):
        T = logits.shape[0]
        ids = torch.zeros(T * k, dtype=torch.int32)
        return torch.zeros(T, k), torch.zeros(E), ids, ids.clone(), torch.zeros(E, dtype=torch.int32)

    monkeypatch.setattr(moe, "_route_forward", forward)
    how = ("sigmoid", None, 1, 1, "max", True, 1.0)
    for create_graph in (False, True):
        logits = torch.randn(5, 8, requires_grad=True)
        w, p = moe._RouteFn.apply(logits, 8, 2, 4, how)[:2]
        d, = torch.autograd.grad(_Nothing.apply(w, p), logits, create_graph=create_graph, allow_unused=True)
        assert d is None
