"""Operands that are no plain tensors: the kernels are not handed their addresses (CPU, the launches stubbed)."""
import torch

from distdl_b200 import ops
from distdl_b200.ops import moe, optim, rotary


class Named(torch.Tensor):
    """A subclass, as far as the calls can see."""


def named(t):
    return t.as_subclass(Named)


def test_weights_positions_biases_and_norms(monkeypatch):
    def refuse(*a, **k):
        raise AssertionError("a kernel was launched")

    for module in (rotary, moe, optim):
        monkeypatch.setattr(module, "use_native", lambda *t: True)
        monkeypatch.setattr(module, "call_on", refuse)
    x, w, pos, r = torch.randn(6, 4, 16), torch.ones(16), torch.arange(6), ops.Rotary()
    kernels = []
    for call in (lambda f: ops.rope(x, 6, 3, rotary=r, positions=f(pos)),
                 lambda f: ops.rope_(x.clone(), 6, 3, rotary=r, positions=f(pos)),
                 lambda f: ops.qk_norm_rope(x, 6, 2, 1, f(w), w),
                 lambda f: ops.qk_norm_rope(x, 6, 2, 1, None, f(w)),
                 lambda f: ops.qk_norm_rope(x, 6, 2, 1, rotary=r, positions=f(pos)),
                 lambda f: moe.route(x[0], 16, 2, 9, score="sigmoid", bias=f(torch.zeros(16))),
                 lambda f: ops.clip_grad_norm_([x.clone()], 1.0, norm=f(torch.tensor(2.0)))):
        call(named)
        try:
            call(lambda t: t)
        except (AssertionError, RuntimeError):                # (the kernels' way: the stub, or no device to ask)
            kernels.append(call)
    assert len(kernels) == 7
