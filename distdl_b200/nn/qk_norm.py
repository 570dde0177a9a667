"""Norms of the query and key heads with the rotary positions in the same pass.  New relative to the reference, which has
no attention code; the weights are sharded and gathered as those of its ZeRO norm layers
(``src/distdl/nn/rmsnorm_zero.py:22-347``)."""
import torch

from .. import ops
from .module import Module
from .rmsnorm_zero import DistributedRMSNormZero


class DistributedQKNormRope(Module):
    r"""``forward(qkv, seq, hq, hkv)``: the RMS norm of every one of the ``hq`` query heads (weight ``q_norm.weight``) and
    ``hkv`` key heads (``k_norm.weight``) of ``qkv [tokens, heads, head_dim]``, turned by their positions as ``rotary`` (an
    ``ops.Rotary``, or None: no rotation) says; the heads behind, the values, are passed on.  One weight of ``head_dim``
    values serves all query heads of all workers, another all key heads: both are split evenly over the workers of ``P_x``
    and gathered on use, and their gradients are summed over them.  Positions as for ``ops.rope``: ``offset``, ``ranges`` or
    ``positions``.

    A new tensor while gradients are recorded; otherwise ``qkv`` itself, changed in place, is returned.  ``q_norm`` and
    ``k_norm`` hold the weights and are not called themselves: hooks belong on this layer."""

    def __init__(self, P_x, head_dim, rotary=None, eps=1e-6, collect_state=False, device=None, dtype=None,
                 scale_backward=None, auto_clear_buffer=True):
        super().__init__()
        self.P_x, self.head_dim, self.rotary, self.eps = P_x, int(head_dim), rotary, eps
        if not P_x.active:
            return
        if rotary is not None:
            rotary.rotated(self.head_dim)                     # (refuses settings that do not fit the heads)
        settings = dict(eps=eps, collect_state=collect_state, device=device, dtype=dtype, scale_backward=scale_backward,
                        auto_clear_buffer=auto_clear_buffer)
        self.q_norm = DistributedRMSNormZero(P_x, self.head_dim, **settings)
        self.k_norm = DistributedRMSNormZero(P_x, self.head_dim, **settings)

    def extra_repr(self):
        return f"head_dim={self.head_dim}, rotary={self.rotary}"

    def forward(self, qkv, seq, hq, hkv, offset=0, ranges=None, positions=None):
        if not self.P_x.active:
            return qkv
        wq, wk = self.q_norm._gathered()[0], self.k_norm._gathered()[0]
        run = ops.qk_norm_rope if torch.is_grad_enabled() else ops.qk_norm_rope_
        return run(qkv, seq, hq, hkv, wq, wk, rotary=self.rotary, offset=offset, ranges=ranges, positions=positions,
                   eps=self.eps)
