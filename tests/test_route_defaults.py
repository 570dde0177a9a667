"""Routing with all settings at their defaults: masked experts, padding tokens, numbers that are none, ties (CPU)."""
import math

import pytest
import torch

from distdl_b200.ops import moe


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("E", [4, 64, 65, 128])
def test_masked_experts_and_padding_tokens(E, dtype):
    logits = torch.full((4, E + 3), -math.inf, dtype=dtype)
    logits[:, E:] = 50.0                                      # padding columns are not looked at
    logits[0, [0, 2, 3]] = torch.tensor([1.0, 3.0, 2.0], dtype=dtype)
    logits[2, 1] = 0.5
    logits[3, :4] = torch.tensor([0.0, -200.0, -math.inf, -400.0], dtype=dtype)     # (its other scores are 0 in fp32)
    logits.requires_grad_()
    w, prob, ids, slot, counts = moe.route(logits, E, 2, 2)
    assert ids.tolist() == [2, 3, -1, -1, 1, -1, 0, 1]
    assert slot.tolist() == [0, 0, -1, -1, 0, -1, 0, 1]
    assert counts.tolist()[:4] == [1, 2, 1, 1] and counts.sum() == 5
    first = torch.softmax(torch.tensor([3.0, 2.0]), 0)
    assert torch.allclose(w, torch.stack([first, torch.zeros(2), torch.tensor([1.0, 0.0]), torch.tensor([1.0, 0.0])]))
    assert torch.isfinite(prob).all() and abs(prob.sum().item() - 3.0) < 1e-5
    d, = torch.autograd.grad((w * torch.arange(8.0).reshape(4, 2)).sum() + (prob * torch.arange(E)).sum(), logits)
    assert torch.isfinite(d).all() and (d[1] == 0).all() and (d[:, E:] == 0).all() and d[0, 2] != 0


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("E", [8, 80])
def test_what_is_no_number_shows_in_its_token_alone(E, bad):
    torch.manual_seed(0)
    logits = torch.randn(5, E)
    logits[1, 3] = bad
    logits[3] = bad
    logits.requires_grad_()
    w, prob, ids, slot, counts = moe.route(logits, E, 2, 9)
    assert torch.isnan(w).all(-1).tolist() == [False, True, False, True, False] and not torch.isnan(w[::2]).any()
    assert ids.reshape(5, 2)[1, 0] == 3 and ids.reshape(5, 2)[3].tolist() == [0, 1] and torch.isnan(prob).all()
    assert ((ids >= 0) & (ids < E)).all() and counts.sum() == 10
    d, = torch.autograd.grad(w[::2].square().sum(), logits)
    assert torch.isfinite(d[::2]).all()


@pytest.mark.parametrize("E", [8, 80])
def test_ties_and_near_ties(E):
    logits = torch.zeros(2, E)
    logits[1, 5], logits[1, 2] = 2e-9, 1e-9                   # no difference of scores in fp32
    _, _, ids, _, _ = moe.route(logits, E, 3, 9)
    assert ids.tolist() == [0, 1, 2, 5, 2, 0]


@pytest.mark.parametrize("E", [8, 80])
def test_no_tokens(E):
    w, prob, ids, slot, counts = moe.route(torch.zeros(0, E), E, 3, 9)
    assert w.shape == (0, 3) and ids.numel() == slot.numel() == 0 and (prob == 0).all() and (counts == 0).all()


@pytest.mark.parametrize("how", [dict(bias=torch.zeros(8)), dict(bias=torch.zeros(8), groups=2, top_groups=1, group_score="top2"),
                                 dict(groups=4, top_groups=2, group_score="top2"), dict(scale=1.5)], ids=lambda h: str(len(h)))
def test_softmax_of_infinity_still_chooses_k_experts(how):
    logits = torch.tensor([[0.0, 3.0, 1.0, math.inf, 2.0, -1.0, 5.0, 4.0], [0.0, 3.0, 1.0, 2.5, 2.0, -1.0, math.inf, math.inf]])
    w, _, ids, slot, counts = moe.route(logits, 8, 3, 9, **how)
    ids = ids.reshape(2, 3)
    # (half of the experts: the ones beside the infinite)
    assert ids.tolist() == ([[3, 1, 2], [6, 7, 4]] if how.get("groups") == 2 else [[3, 6, 7], [6, 7, 1]])
    assert torch.isnan(w).all() and counts.sum() == 6 and (slot >= 0).all()
