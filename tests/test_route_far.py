"""Sigmoid scores that 64 bits no longer tell apart keep the order of their logits wherever they are chosen one by one, and biases of
+inf are all alike (CPU; on a GPU: the kernels)."""
import math

import pytest
import torch

from distdl_b200.ops import moe

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("E,groups,top_groups,by", [(12, 1, 1, "max"), (12, 3, 3, "top2"), (12, 12, 12, "top2"), (12, 12, 9, "top2"),
                                                    (12, 3, 3, "max"), (96, 8, 8, "top2"), (96, 96 // 3, 32, "top2")])
def test_saturated_scores(E, groups, top_groups, by, device):
    g = torch.Generator().manual_seed(E + groups)
    logits = 40.0 + torch.stack([torch.randperm(E, generator=g) for _ in range(20)]).float()
    ids = moe.route(logits.to(device), E, 5, 20, score="sigmoid", groups=groups, top_groups=top_groups, group_score=by)[2]
    assert torch.equal(ids.cpu().view(20, 5).long(), logits.argsort(1, descending=True)[:, :5])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(12, 3), (64, 8), (60, 6), (256, 4)])
def test_biases_of_infinity_are_alike(E, groups, score, device):
    size = E // groups
    bias = torch.zeros(E)
    bias[size + 1] = math.inf                                 # one in the second group, two in the third
    bias[2 * size:2 * size + 2] = math.inf
    logits = torch.randn(9, E, generator=torch.Generator().manual_seed(0))
    how = dict(score=score, bias=bias.to(device), groups=groups, top_groups=1, group_score="top2")
    ids = moe.route(logits.to(device), E, 2, 9, **how)[2].cpu().view(9, 2)
    assert (ids[:, 0] == size + 1).all() and (ids // size == 1).all()
    ids = moe.route(logits.to(device), E, 3, 9, **dict(how, top_groups=2))[2].cpu().view(9, 3)
    assert (ids == torch.tensor([size + 1, 2 * size, 2 * size + 1])).all()
    # a NaN is ahead of them
    logits[:, E - 1] = math.nan
    ids = moe.route(logits.to(device), E, 2, 9, **how)[2].cpu().view(9, 2)
    assert (ids[:, 0] == E - 1).all() and (ids // size == groups - 1).all()
