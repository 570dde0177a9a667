"""Gradient clipping over all workers, for optimizers other than :class:`~distdl_b200.parallel.FlatAdamW` (which clips
for itself).  New relative to the reference, which leaves the optimizer to the user."""
from __future__ import annotations

import torch
import torch.distributed as dist

from .. import ops
from ..ops.optim import gradients_of


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scales the gradients of ``parameters`` (this worker's; gradients themselves are taken too, None is passed over) in
    place so that the norm of the gradients of ALL workers together is at most ``max_norm``, and returns that norm (an fp32
    scalar on the gradients' device).  Every element of a distributed layer's parameters lives on exactly one worker, so that
    the workers' sums of squares add up.  Collective over all processes; a worker without gradients takes part."""
    grads = gradients_of(parameters)
    if not dist.is_initialized() or dist.get_world_size() == 1:
        return ops.clip_grad_norm_(grads, max_norm)
    total = ops.grad_norm(grads, squared=True)
    if not grads and torch.cuda.is_available():
        total = total.cuda()                                  # (where the others' sums are)
    dist.all_reduce(total)
    return ops.clip_grad_norm_(grads, max_norm, norm=total.sqrt().float())
