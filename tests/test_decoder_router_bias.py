"""The routers' biases in checkpoints in the serial layout: present, and absent (CPU ranks)."""
import pytest
import torch

from dist_harness import run_ranks
from test_decoder_options import options


def body(rank, world):
    from distdl_b200 import models

    def make():
        torch.manual_seed(3)
        return models.Decoder(options("moe"), models.ParallelLayout(world, 1))

    a, b = make(), make()
    biases = lambda m: [x.mlp.router_bias for x in m.blocks]                # noqa: E731
    for i, t in enumerate(biases(a)):
        t.copy_(torch.arange(t.numel()) * 0.5 + i)
    for p in a.parameters():
        p.data.mul_(2.0)
    serial = a.state_dict()
    b.load_state_dict(serial if rank == 0 else {})
    assert all(torch.equal(x, y) for x, y in zip(biases(a), biases(b)))
    without = {k: v for k, v in serial.items() if not k.endswith("router_bias")}
    c = make()
    for t in biases(c):
        t.fill_(7.0)
    with pytest.raises(RuntimeError, match="router_bias"):    # on every worker, none is left waiting
        c.load_state_dict(dict(without))
    missing = c.load_state_dict(dict(without), strict=False).missing_keys
    assert sum(k.endswith("router_bias") for k in missing) == 2
    assert all((t == 7.0).all() for t in biases(c))
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), c.parameters()))
    return True


@pytest.mark.parametrize("world", [1, 2])
def test_checkpoints_with_and_without_the_biases(world):
    assert all(run_ranks("test_decoder_router_bias", "body", world, timeout=120))
