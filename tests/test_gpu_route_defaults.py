"""Routing with all settings at their defaults on the GPU, against the definition in 64 bits: every type, masked experts, padding
tokens, numbers that are none, ties."""
import math

import pytest
import torch

from distdl_b200.ops import moe
from test_gpu_route import BF16, FP16, FP32, check

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (6, 8, 1), (8, 8, 2), (8, 8, 8), (16, 17, 4), (33, 40, 8), (60, 64, 4), (64, 64, 8), (64, 64, 12), (65, 65, 3),
         (128, 136, 8)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("E,width,k", SIZES)
def test_defaults_match_the_definition(E, width, k, dtype):
    torch.manual_seed(E + k)
    logits = (torch.randn(70, width, device="cuda") * 2).to(dtype)
    check(logits, E, k, 6)
    check(logits[:1], E, k, 6)
    check(logits.T.contiguous().T, E, k, 6)                   # strided


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("E,width,k", SIZES)
def test_masked_experts_and_padding_tokens(E, width, k, dtype):
    torch.manual_seed(E + k + 1)
    logits = torch.randn(70, width, device="cuda").to(dtype)
    logits[torch.rand(70, width, device="cuda") < 0.7] = -math.inf
    logits[7] = -math.inf
    logits[9, :E] = -math.inf
    logits[11] = -math.inf
    logits[11, E // 2] = 2.0
    w, prob, ids, slot, counts = check(logits, E, k, 9)
    ids, slot = ids.reshape(70, k), slot.reshape(70, k)
    assert (ids[[7, 9]] == -1).all() and (slot[[7, 9]] == -1).all() and (w[[7, 9]] == 0).all()
    assert ids[11, 0] == E // 2 and (ids[11, 1:] == -1).all() and w[11, 0] == 1
    assert counts.sum() == (ids >= 0).sum()
    kept = slot >= 0                                          # no slot is given twice
    assert (ids.long() * 1000 + slot.long())[kept].unique().numel() == kept.sum()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("E,k", [(8, 2), (64, 8), (80, 3)])
def test_what_is_no_number_shows_in_its_token_alone(E, k, bad, dtype):
    torch.manual_seed(2)
    logits = torch.randn(300, E, device="cuda").to(dtype)
    logits[4, 3] = bad
    logits[299] = bad
    logits[5, 1:] = -math.inf
    logits.requires_grad_()
    w, prob, ids, slot, counts = moe.route(logits, E, k, 300)
    host = moe.route(logits.detach().cpu(), E, k, 300)
    for a, b in zip((ids, slot, counts), host[2:]):
        assert torch.equal(a.cpu(), b)
    rows = torch.isnan(w).any(-1).nonzero().flatten().tolist()
    assert rows == [4, 299] and torch.isnan(w[4]).all() and torch.isnan(prob).all()
    assert ids.reshape(300, k)[4, 0] == 3 and ids.reshape(300, k)[299].tolist() == list(range(k))
    assert w[5, 0] == 1 and (w[5, 1:] == 0).all()
    d, = torch.autograd.grad((w[:4].square().sum(), w[5:299].square().sum()), logits)
    good = torch.ones(300, dtype=torch.bool)
    good[[4, 299]] = False
    assert torch.isfinite(d[good]).all() and torch.isnan(d[~good]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_ties_and_scores_that_fp32_does_not_tell_apart(dtype):
    logits = torch.zeros(40, 24, device="cuda", dtype=dtype)
    logits[1, 5], logits[1, 2] = 2e-9, 1e-9
    logits[2, 7], logits[2, 3:6] = 200.0, torch.tensor([3.0, 5.0, 4.0])
    _, _, ids, _, _ = check(logits, 24, 3, 40, grads=False)
    assert ids.reshape(40, 3)[:3].tolist() == [[0, 1, 2], [5, 2, 0], [7, 4, 5]]


def test_no_tokens():
    for dtype in (BF16, FP32):
        w, prob, ids, slot, counts = moe.route(torch.zeros(0, 8, device="cuda", dtype=dtype), 8, 3, 9)
        assert w.shape == (0, 3) and ids.numel() == slot.numel() == 0 and (prob == 0).all() and (counts == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(24, 1), (64, 8), (256, 8), (60, 6), (512, 16), (10, 5)])
def test_the_kernels_choose_as_the_path_without_them(E, groups, score, dtype):
    """Tokens with several logits that are no numbers, and with infinities."""
    g = torch.Generator().manual_seed(E)
    logits = torch.randn(200, E, generator=g).to(dtype)
    for value in (math.nan, math.inf, -math.inf):
        logits[torch.rand(200, E, generator=g) < 1.5 / E] = value
    bias = torch.randn(E, generator=g) * 0.1
    for by in ("max", "top2"):
        for b in (None, bias):
            how = dict(score=score, groups=groups, top_groups=(groups + 1) // 2, group_score=by)
            got = moe.route(logits.cuda(), E, 4, 20, bias=None if b is None else b.cuda(), **how)
            want = moe.route(logits, E, 4, 20, bias=b, **how)
            for x, y in zip(got[2:], want[2:]):
                assert torch.equal(x.cpu(), y)
            assert torch.equal(torch.isnan(got[0]).cpu(), torch.isnan(want[0]))
            assert torch.allclose(got[0].cpu(), want[0], rtol=1e-5, atol=1e-30, equal_nan=True)
