"""Choices among scores that fp32 does not tell apart, behind experts that are alike, and far below the best."""
import pytest
import torch

from test_gpu_route import BF16, FP32, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", [dict(), dict(score="sigmoid"), dict(score="softmax", renormalize=False)], ids=str)
@pytest.mark.parametrize("bias", [None, "zero", "one step"])
@pytest.mark.parametrize("E,k", [(72, 2), (128, 3), (256, 8), (512, 31)])
def test_the_better_one_lies_behind_some_that_are_alike(E, k, bias, how):
    g = torch.Generator().manual_seed(E + k)
    logits = torch.randn(60, E, generator=g) - 6.0
    b = None if bias is None else torch.zeros(E)
    for t in range(60):
        alike = min(E - 1, k + t % 9)                         # as many as are chosen, and more
        place = torch.randperm(E, generator=g)[:alike + 1].sort().values
        logits[t, place[:-1]] = 1.0
        logits[t, place[-1]] = 1.0 if bias == "one step" and t % 2 else 1.0 + 2.0 ** -23
    if bias == "one step":
        b[E // 2:] = 2.0 ** -25
    check(logits.cuda(), E, k, 60, grads=False, bias=None if b is None else b.cuda(), **how)


@pytest.mark.parametrize("E", [72, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_all_alike_but_for_one_far_above(E, bias):
    """What lies far below the largest is told apart all the same."""
    logits = torch.zeros(40, E)
    logits[:, 7] = 200.0
    for t in range(40):
        logits[t, 10 + t:13 + t] = torch.tensor([3.0, 5.0, 4.0])
    if bias:
        check(torch.zeros(40, E).cuda(), E, 3, 40, grads=False, score="sigmoid", bias=logits[0].cuda())
    else:
        check(logits.cuda(), E, 3, 40, grads=False)
        check(logits.to(BF16).cuda(), E, 3, 40, grads=False)
        check(logits.cuda(), E, 4, 40, grads=False, groups=8, top_groups=2)


def test_biases_a_step_apart_on_few_values():
    g = torch.Generator().manual_seed(3)
    for E, dtype in ((96, BF16), (256, FP32)):
        logits = torch.randint(-2, 3, (200, E), generator=g).to(dtype).cuda()
        bias = (torch.randint(0, 3, (E,), generator=g) * 2.0 ** -25).cuda()
        for score in ("softmax", "sigmoid"):
            check(logits, E, 6, 30, grads=False, score=score, bias=bias)
            check(logits, E, 6, 30, grads=False, score=score, bias=bias, groups=8, top_groups=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(64, 8), (256, 8), (60, 6), (512, 4), (16, 8)])
def test_group_sums_of_experts_far_below_the_best(E, groups, score):
    """Of a group's two best the second may lie far below all others, and still decides."""
    g = torch.Generator().manual_seed(E)
    size = E // groups
    logits = torch.randn(50, E, generator=g)
    bias = -200.0 - 100.0 * torch.rand(E, generator=g)
    place = torch.randperm(groups, generator=g)
    for i, (best, second) in enumerate([(0.5, -100.0), (-0.5, -50.0), (0.25, -75.0), (-9.0, -12.0)]):
        bias[place[i] * size + torch.randperm(size, generator=g)[:2]] = torch.tensor([best, second])
    how = dict(score=score, groups=groups, group_score="top2", bias=bias.cuda())
    for top_groups in (1, 2, 3):
        check(logits.cuda(), E, 2, 50, grads=False, top_groups=top_groups, **how)
    masked = logits.clone()
    masked[torch.rand(50, E, generator=g) < 0.3] = -float("inf")
    check(masked.cuda(), E, 2, 50, grads=False, top_groups=2, **how)
