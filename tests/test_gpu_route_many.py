"""Routing of as many tokens as training has (several per warp, chunks of every size, further rounds of the backward pass), against
the definition in 64 bits, all tokens at once."""
import math

import pytest
import torch

from distdl_b200.ops import moe

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def chosen(l, k, score, bias, groups, top_groups, group_score):
    """The experts [tokens, k] for logits in 64 bits, -1 where there is none."""
    T, E = l.shape
    none = l == -math.inf
    if bias is None and (groups == 1 or group_score == "max"):
        c = l.clone()
    else:
        c = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l.masked_fill(none.all(1, keepdim=True), 0.0), 1)
        c = c if bias is None else c + bias.double()
    c[none] = -math.inf
    if groups > 1:
        two = c.view(T, groups, -1).topk(min(2, E // groups), dim=2).values
        value = two[..., 0].clone()
        if group_score == "top2" and two.shape[2] > 1:
            value += two[..., 1].masked_fill(two[..., 1] == -math.inf, 0.0)
        order = torch.argsort(value, dim=1, descending=True, stable=True)
        out = torch.ones(T, groups, dtype=torch.bool, device=l.device).scatter_(1, order[:, :top_groups], False)
        c.view(T, groups, -1).masked_fill_(out.unsqueeze(2), -math.inf)
    order = torch.argsort(c, dim=1, descending=True, stable=True)[:, :k]
    return order.masked_fill(c.gather(1, order) == -math.inf, -1)


def placed(ids, E, capacity):
    """(slots, counts): ranks in pair order."""
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=E)
    order = torch.argsort(torch.where(flat >= 0, flat, E), stable=True)
    start = torch.cat([counts.cumsum(0) - counts, counts.sum().reshape(1)])
    rank = torch.empty_like(flat)
    rank[order] = torch.arange(flat.numel(), device=flat.device) - start[torch.where(flat >= 0, flat, E)[order]]
    return torch.where((flat >= 0) & (rank < capacity), rank, -1), counts


def outputs(l, ids, score, renormalize, scale):
    """(weights, sums of probabilities) in 64 bits, differentiable."""
    none = (l == -math.inf).all(1, keepdim=True)
    l = l.masked_fill(none, 0.0)
    log_s = l if score == "softmax" else torch.nn.functional.logsigmoid(l)
    p = torch.softmax(log_s, 1).masked_fill(none, 0.0)
    here, at = ids >= 0, ids.clamp(min=0)
    if renormalize:
        picked = log_s.gather(1, at).masked_fill(~here, -math.inf).masked_fill(~here.any(1, keepdim=True), 0.0)
        w = torch.softmax(picked, 1)
    else:
        w = (p if score == "softmax" else torch.sigmoid(l)).gather(1, at)
    return (scale * w).masked_fill(~here, 0.0), p.sum(0)


def check(T, E, width, k, dtype, capacity, score="softmax", bias=None, groups=1, top_groups=1, group_score="max",
          renormalize=True, scale=1.0, masked=False):
    g = torch.Generator("cuda").manual_seed(T + E)
    logits = torch.randn(T, width, generator=g, device="cuda").to(dtype)
    if masked:
        logits[torch.rand(T, width, generator=g, device="cuda") < 0.3] = -math.inf
        logits[torch.rand(T, generator=g, device="cuda") < 0.1] = -math.inf
    logits.requires_grad_()
    bias = torch.randn(E, generator=g, device="cuda") * 0.05 if bias else None
    how = dict(score=score, bias=bias, groups=groups, top_groups=top_groups, group_score=group_score, renormalize=renormalize,
               scale=scale)
    w, prob, ids, slot, counts = moe.route(logits, E, k, capacity, **how)
    l64 = logits.detach()[:, :E].double().requires_grad_()
    want = chosen(l64.detach(), k, score, bias, groups, top_groups, group_score)
    assert torch.equal(ids.view(T, k).long(), want)
    s6, c6 = placed(want, E, capacity)
    assert torch.equal(slot.long(), s6) and torch.equal(counts.long(), c6)
    assert masked or (slot == -1).any()                       # (the capacity drops some)
    w6, p6 = outputs(l64, want, score, renormalize, scale)
    # exponentials of differences d up to 12: 2^-22 + d 2^-23 in the term and in sums of k or of all experts; some additions and divisions
    rel = 2.0 ** -18
    assert ((w.double() - w6).abs() <= rel * w6.abs() + 1e-30).all()
    # sums over tokens: at most 32 in a warp, 8 warps, the chunks over 32 lanes and those (at most 64 + 5 additions), 2^-24 each
    assert ((prob.double() - p6).abs() <= (rel + 109 * 2.0 ** -24) * p6 + 1e-30).all()
    dw, dp = torch.randn(T, k, generator=g, device="cuda"), torch.randn(E, generator=g, device="cuda")
    got, = torch.autograd.grad((w, prob), logits, (dw, dp))
    d6, = torch.autograd.grad((w6, p6), l64, (dw.double(), dp.double()))
    assert (got[:, E:] == 0).all()
    # a sum of two parts, each a difference of terms of at most this size
    size = 2 * dw.abs().amax(1, keepdim=True) * w6.detach().sum(1, keepdim=True) + 2 * dp.abs().max()
    bound = torch.finfo(dtype).eps / 2 * d6.abs() + rel * size + (2.0 ** -25 if dtype == FP16 else 0.0)
    err = (got[:, :E].double() - d6).abs()
    assert (err <= bound).all(), (err - bound).max().item()


@pytest.mark.parametrize("T", [3552, 3553, 7105, 16385, 70001])
@pytest.mark.parametrize("E,width,groups,how", [
    (256, 256, 8, dict(score="sigmoid", bias=True, group_score="top2", scale=2.5)),
    (512, 512, 16, dict(score="softmax", bias=True)),
    (510, 512, 6, dict(score="sigmoid", group_score="top2", renormalize=False)),
    (250, 250, 5, dict(score="softmax", masked=True, renormalize=False)),
    (128, 128, 1, dict()),
    (60, 64, 1, dict(score="sigmoid", masked=True)),
    (8, 8, 1, dict()),
], ids=str)
def test_many_tokens(T, E, width, groups, how):
    dtype = (BF16, FP32, FP16)[(T + E) % 3]
    k = min(8, E // 2)
    check(T, E, width, k, dtype, capacity=max(1, T * k // E), groups=groups, top_groups=max(1, groups // 2), **how)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T,E,k", [(262145, 64, 4), (300000, 16, 2), (131073, 256, 8)])
def test_chunks_of_the_largest_size(T, E, k, dtype):
    check(T, E, E, k, dtype, capacity=T * k // E)
    check(T, E, E, k, dtype, capacity=T * k // E, score="sigmoid", bias=True)
