"""Routing to experts in its general form on the GPU, against the definition in 64 bits."""
import math

import pytest
import torch

from distdl_b200.ops import moe

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def definition(logits, E, k, capacity, score="softmax", bias=None, groups=1, top_groups=None, group_score="max",
               renormalize=True, scale=1.0):
    """(weights, prob_sum, ids, slot, counts) token by token, on the CPU in 64 bits; differentiable in ``logits``."""
    T = logits.shape[0]
    l = logits[:, :E]
    weights = torch.zeros(T, k, dtype=torch.float64)
    rows, probs = [], []
    for t in range(T):
        live = torch.isfinite(l[t].detach())
        if not live.any():
            rows.append([])
            probs.append(torch.zeros(E, dtype=torch.float64))
            continue
        lt = torch.where(live, l[t], torch.full_like(l[t], -math.inf))
        s = torch.softmax(lt, 0) if score == "softmax" else torch.sigmoid(lt)
        ratio = torch.softmax(lt if score == "softmax" else torch.nn.functional.logsigmoid(lt), 0)
        c = s.detach() + (0.0 if bias is None else bias.double())
        # (without a bias and sums the logits' order: scores of 64 bits are no longer apart far from zero)
        if bias is None and (groups == 1 or group_score == "max"):
            c = lt.detach().clone()
        c[~live] = -math.inf
        if groups > 1:
            by = c.reshape(groups, -1)
            best = by.sort(dim=1, descending=True).values
            value = best[:, 0].clone()
            if group_score == "top2" and best.shape[1] > 1:
                value += torch.where(best[:, 1] > -math.inf, best[:, 1], torch.zeros_like(value))
            order = sorted(range(groups), key=lambda g: (-value[g].item(), g))
            for g in order[top_groups if top_groups else groups:]:
                by[g] = -math.inf
            c = by.reshape(-1)
        order = [e for e in sorted(range(E), key=lambda e: (-c[e].item(), e)) if c[e] > -math.inf][:k]
        rows.append(order)
        probs.append(ratio)
        if order:
            if renormalize:
                from_l = lt[order] if score == "softmax" else torch.nn.functional.logsigmoid(lt[order])
                w = torch.softmax(from_l, 0)
            else:
                w = s[order]
            weights = weights.index_put((torch.full((len(order),), t), torch.arange(len(order))), scale * w)
    ids = torch.full((T, k), -1)
    for t, order in enumerate(rows):
        ids[t, :len(order)] = torch.tensor(order, dtype=torch.long) if order else ids[t, :0]
    slot, counts = torch.full((T * k,), -1), torch.zeros(E, dtype=torch.long)
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if e >= 0:
            if counts[e] < capacity:
                slot[p] = counts[e]
            counts[e] += 1
    return weights, torch.stack(probs).sum(0), ids.reshape(-1), slot, counts


def check(logits, E, k, capacity, grads=True, **how):
    logits = logits.detach().requires_grad_()
    w, prob, ids, slot, counts = moe.route(logits, E, k, capacity, **how)
    l64 = logits.detach().double().cpu().requires_grad_()
    host = dict(how, bias=None if how.get("bias") is None else how["bias"].cpu())
    w6, p6, i6, s6, c6 = definition(l64, E, k, capacity, **host)
    assert torch.equal(ids.cpu().long(), i6), (ids.cpu().long() != i6).nonzero()[:5]
    assert torch.equal(slot.cpu().long(), s6) and torch.equal(counts.cpu().long(), c6)
    # fp32: exponentials of differences up to |d| (relative 2^-22 + |d| 2^-23), sums of k and of the experts, divisions
    spread = l64.detach()[:, :E]
    spread = torch.where(torch.isfinite(spread), spread, torch.zeros_like(spread)).abs().max().item()
    rel = 2.0 ** -19 + 2 * spread * 2.0 ** -23
    assert ((w.detach().cpu().double() - w6.detach()).abs() <= rel * w6.detach().abs() + 1e-30).all()
    assert ((prob.detach().cpu().double() - p6.detach()).abs() <= 2 * rel * p6.detach().abs() + 1e-30).all()
    if not grads:
        return w, prob, ids, slot, counts
    g = torch.Generator().manual_seed(1)
    dw, dp = torch.randn(w6.shape, generator=g, dtype=torch.float64), torch.randn(E, generator=g, dtype=torch.float64)
    for use in ((dw, dp), (dw, None), (None, dp)):
        outs = [(o, o6, d) for o, o6, d in zip((w, prob), (w6, p6), use) if d is not None]
        got, = torch.autograd.grad([o[0] for o in outs], logits, [o[2].float().cuda() for o in outs], retain_graph=True)
        want, = torch.autograd.grad([o[1] for o in outs], l64, [o[2].float().double() for o in outs], retain_graph=True)
        got = got.cpu().double()
        assert (got[:, E:] == 0).all()
        # a sum of two parts, each a difference of terms of at most this size
        size = how.get("scale", 1.0) * 2 * dw.abs().amax(-1, keepdim=True) * w6.detach().sum(-1, keepdim=True) / max(
            how.get("scale", 1.0), 1e-30) + 2 * dp.abs().max()
        bound = (torch.finfo(logits.dtype).eps / 2) * want.abs() + rel * size + (2.0 ** -25 if logits.dtype == FP16 else 0)
        assert got.shape == want.shape and ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max()
    return w, prob, ids, slot, counts


HOW = [
    dict(score="softmax", renormalize=False),
    dict(score="softmax", scale=2.5),
    dict(score="sigmoid"),
    dict(score="sigmoid", renormalize=False, scale=16.0),
]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("how", HOW, ids=lambda h: "-".join(map(str, h.values())))
@pytest.mark.parametrize("E,width,k,groups,top_groups", [(1, 1, 1, 1, 1), (2, 8, 1, 1, 1), (8, 8, 8, 1, 1), (60, 64, 4, 1, 1),
                                                         (33, 35, 5, 3, 2), (64, 64, 6, 8, 3), (70, 70, 3, 7, 1),
                                                         (256, 256, 8, 8, 4), (160, 160, 6, 16, 5), (96, 104, 32, 32, 20),
                                                         (512, 512, 10, 1, 1), (510, 512, 12, 2, 1), (500, 500, 7, 4, 2)])
def test_route_matches_the_definition(E, width, k, groups, top_groups, how, bias):
    torch.manual_seed(E + k)
    dtype = (BF16, FP16, FP32)[E % 3]
    logits = (torch.randn(45, width, device="cuda") * 2).to(dtype)
    for by in ("max", "top2") if groups > 1 else ("max",):
        check(logits, E, k, 6, groups=groups, top_groups=top_groups, group_score=by,
              bias=torch.randn(E, device="cuda") * 0.1 if bias else None, **how)


@pytest.mark.parametrize("T", [1, 31, 32, 33, 255, 256, 257, 700])
def test_slots_over_chunks(T):
    torch.manual_seed(T)
    logits = (torch.randn(T, 40, device="cuda") + 2 * torch.randn(1, 40, device="cuda")).to(BF16)
    check(logits, 40, 5, max(1, T // 9), grads=T < 300, score="sigmoid")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
def test_ties_go_to_the_lowest(score, group_score, bias):
    """Logits of few values: most experts of a token are equal, and most groups."""
    torch.manual_seed(3)
    logits = torch.randint(-1, 2, (120, 48), device="cuda").to(BF16)
    logits[:3] = 0.0
    b = None if bias is None else torch.zeros(48, device="cuda") if bias == "zero" else \
        torch.randint(0, 2, (48,), device="cuda") * 0.25
    check(logits, 48, 6, 10, grads=False, score=score, group_score=group_score, groups=6, top_groups=3, bias=b)
    check(logits, 48, 6, 10, grads=False, score=score, bias=b, renormalize=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_nearly_equal_scores_are_told_apart(score):
    """Scores that differ by less than fp32 computes them to: the bias undoes the logits' differences but for some 2^-26."""
    torch.manual_seed(4)
    T, E = 400, 64
    logits = torch.randn(T, E, device="cuda")
    s = torch.softmax(logits[:1].double(), -1) if score == "softmax" else torch.sigmoid(logits[:1].double())
    bias = (0.5 - s[0]).float()
    logits = logits[:1] + torch.randn(T, E, device="cuda") * 1e-7
    check(logits, E, 8, T, grads=False, score=score, bias=bias)
    check(logits, E, 8, T, grads=False, score=score, bias=bias, groups=8, top_groups=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [1, 2, 8, 31, 32])
def test_the_first_left_out_is_told_apart(score, k):
    # k - 1 experts far above the others; of two that are an ulp of fp32 apart the later is the better one
    g = torch.Generator().manual_seed(k)
    logits = torch.randn(32, 80, generator=g)
    place = torch.stack([torch.randperm(80, generator=g) for _ in range(32)])
    two = place[:, k - 1:k + 1].sort(1).values
    logits.scatter_(1, place[:, :k - 1], 6.0 + torch.rand(32, k - 1, generator=g))
    logits.scatter_(1, two, torch.tensor([4.0, 4.0 + 2.0 ** -21]).expand(32, 2))
    check(logits.cuda(), 80, k, 32, grads=False, score=score, bias=torch.zeros(80).cuda())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts_and_padding_tokens(score, grouped, bias):
    torch.manual_seed(5)
    logits = torch.randn(50, 36, device="cuda")
    logits[torch.rand(50, 36, device="cuda") < 0.6] = -math.inf
    logits[7] = -math.inf                                    # a padding token
    logits[11] = -math.inf
    logits[11, 30] = 2.0                                     # one expert left
    logits[12] = torch.finfo(FP32).min                       # the lowest value is a value
    how = dict(groups=6, top_groups=4, group_score="top2") if grouped else {}
    b = torch.randn(36, device="cuda") * 0.1 if bias else None
    # (its differences reach 3e38: exponentials of them are exactly 0 or 1, and the tolerance's |d| does not apply)
    keep = [t for t in range(50) if t != 12]
    for renormalize in (True, False):                        # (a scale: the general form, which knows masked experts)
        w, prob, ids, slot, _ = check(logits[keep], 36, 5, 9, score=score, bias=b, renormalize=renormalize, scale=1.5, **how)
        assert (ids[7 * 5:8 * 5] == -1).all() and (slot[7 * 5:8 * 5] == -1).all() and (w[7] == 0).all()
        assert ids[11 * 5] == 30 and (ids[11 * 5 + 1:12 * 5] == -1).all()
    w, prob, ids, slot, _ = moe.route(logits[12:13], 36, 5, 9, score=score, bias=b, scale=1.5, **how)
    assert torch.allclose(w, torch.full_like(w, 0.3)) and (ids >= 0).all() and torch.isfinite(prob).all()


def test_far_logits():
    """Weights of tokens whose scores underflow, and saturated sigmoids in the logits' order."""
    logits = torch.tensor([[-200.0, -201.0, -199.5, -300.0], [200.0, 201.0, 90.0, 200.5], [-1e30, 1e30, 0.0, 5.0]],
                          device="cuda")
    w, _, ids, _, _ = moe.route(logits, 4, 2, 9, score="sigmoid")
    assert ids.tolist() == [2, 0, 1, 3, 1, 3]
    want = torch.softmax(torch.tensor([-199.5, -200.0], dtype=torch.float64), 0)
    assert torch.allclose(w[0].double().cpu(), want, rtol=1e-5)
    assert torch.allclose(w[1:], torch.full((2, 2), 0.5, device="cuda"), atol=4e-3)
    w, prob, ids, _, _ = moe.route(logits, 4, 2, 9, score="softmax", scale=3.0)
    assert ids.tolist() == [2, 0, 1, 3, 1, 3] and torch.isfinite(w).all() and torch.isfinite(prob).all()


def test_biases_that_take_experts_out():
    """-inf takes an expert out; a bias far below the others' leaves it to the end, and leaves the others told apart."""
    torch.manual_seed(14)
    logits = torch.randn(200, 40, device="cuda")
    for low in (-math.inf, -1e9, -1e30):
        bias = torch.randn(40, device="cuda") * 0.1
        bias[::3] = low
        for how in (dict(score="sigmoid"), dict(score="softmax", groups=8, top_groups=5, group_score="top2")):
            host = dict(how, bias=bias.cpu())
            ids = moe.route(logits, 40, 8, 200, bias=bias, **how)[2].cpu().long()
            # (bias -inf: as the definition with the logit -inf)
            l64 = logits.double().cpu()
            want = definition(l64, 40, 8, 200, **host)[2] if low > -math.inf else None
            assert want is None or torch.equal(ids, want)
            assert low > -math.inf or not (ids[ids >= 0] % 3 == 0).any()
    ids = moe.route(logits, 40, 30, 200, bias=bias, score="sigmoid")[2].reshape(200, 30)
    assert (ids[:, :26] % 3 != 0).all() and (ids[:, 26:] % 3 == 0).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_nan_shows_in_its_token_alone(score):
    logits = torch.randn(9, 24, device="cuda")
    logits[4, 3] = math.nan
    logits[6] = math.nan
    logits.requires_grad_()
    for groups in (1, 4):
        w, prob, ids, slot, counts = moe.route(logits, 24, 3, 50, score=score, groups=groups, top_groups=max(1, groups - 1),
                                               bias=torch.zeros(24, device="cuda"))
        bad = torch.isnan(w).all(-1)
        assert bad.tolist() == [t in (4, 6) for t in range(9)] and not torch.isnan(w[~bad]).any()
        assert (ids >= 0).all() and (ids < 24).all() and counts.sum() == 27
        d, = torch.autograd.grad(w[:4].sum(), logits)
        assert not torch.isnan(d[~bad]).any()


def test_padding_columns_views_and_addresses():
    torch.manual_seed(8)
    for make in (lambda: torch.randn(40, 100, device="cuda")[:, :70], lambda: torch.randn(70, 40, device="cuda").T,
                 lambda: torch.randn(40 * 70 + 1, device="cuda")[1:].view(40, 70),
                 lambda: torch.randn(40, 2000, device="cuda")):
        for dt in (BF16, FP32):
            x = make().to(dt)
            x = x if dt == FP32 else make().to(dt)
            if x.shape[1] > 70:
                x[:, 61:] = math.nan                          # padding is not looked at
            check(x, 61, 4, 20, score="sigmoid")
    odd = torch.randn(40 * 72 + 1, device="cuda").to(BF16)[1:].view(40, 72)
    check(odd, 61, 4, 20, score="sigmoid")


def test_no_room_and_all_experts():
    torch.manual_seed(15)
    logits = torch.randn(20, 12, device="cuda")
    w, prob, ids, slot, counts = moe.route(logits, 12, 12, 0, score="sigmoid")
    assert (slot == -1).all() and (counts == 20).all() and (ids.reshape(20, 12).sort(1).values == torch.arange(
        12, device="cuda")).all()
    check(logits, 12, 12, 1 << 40, score="sigmoid")
    with torch.inference_mode():
        moe.route(torch.randn(20, 12, device="cuda"), 12, 3, 4, score="sigmoid")


def test_results_changed_in_place_do_not_disturb_the_gradient():
    logits = torch.randn(20, 12, device="cuda", requires_grad=True)
    w, prob, ids, slot, counts = moe.route(logits, 12, 3, 4, score="sigmoid")
    want, = torch.autograd.grad(w.square().sum(), logits, retain_graph=True)
    counts += 1
    slot.fill_(-1)
    assert torch.equal(torch.autograd.grad(w.square().sum(), logits, retain_graph=True)[0], want)
    ids += 1                                                  # (these the gradient needs)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(w.square().sum(), logits)


def test_no_tokens():
    w, prob, ids, slot, counts = moe.route(torch.zeros(0, 128, device="cuda"), 128, 4, 8, score="sigmoid")
    assert w.shape == (0, 4) and ids.numel() == 0 and (prob == 0).all() and (counts == 0).all()


def test_outputs_do_not_depend_on_the_run():
    torch.manual_seed(9)
    logits = torch.randn(6000, 256, device="cuda", requires_grad=True)
    bias = torch.randn(256, device="cuda") * 0.05

    def once():
        w, prob, ids, slot, counts = moe.route(logits, 256, 8, 200, score="sigmoid", bias=bias, groups=8, top_groups=4,
                                               group_score="top2")
        return [w, prob, ids, slot, counts, *torch.autograd.grad((w.sum(), prob.square().sum()), logits)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_more_experts_than_64_without_settings():
    torch.manual_seed(10)
    check(torch.randn(70, 128, device="cuda").to(BF16), 128, 4, 5)


def test_gradient_against_differences():
    torch.manual_seed(11)
    for how in HOW:
        logits = torch.randn(6, 20, device="cuda", requires_grad=True)
        dw, dp = torch.randn(6, 4, device="cuda"), torch.randn(20, device="cuda")
        bias = torch.linspace(0, 9, 20, device="cuda")         # the choice does not change along the way
        loss = lambda x: sum((o.double() * d.double()).sum() for o, d in                                  # noqa: E731
                             zip(moe.route(x, 20, 4, 9, bias=bias, **how)[:2], (dw, dp)))
        d, = torch.autograd.grad(loss(logits), logits)
        v = torch.randn_like(logits)
        h = 2.0 ** -7
        with torch.no_grad():
            want = ((loss(logits + h * v) - loss(logits - h * v)) / (2 * h)).item()
        # third derivatives of softmax and sigmoid are below 1 in size; fp32 noise 1e-6 over the step
        assert abs((d.double() * v.double()).sum().item() - want) <= how.get("scale", 1.0) * 5e-3 * max(1.0, abs(want))


def test_captured_twice_and_on_another_stream():
    torch.manual_seed(12)
    logits = torch.randn(500, 128, device="cuda", requires_grad=True)
    dw = torch.randn(500, 6, device="cuda")

    def once():
        w, prob, ids, slot, counts = moe.route(logits, 128, 6, 30, score="sigmoid")
        return [w.detach(), prob.detach(), ids, slot, counts, *torch.autograd.grad(w, logits, dw)]

    once()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once()
        graphs.append((g, out, torch.cuda.Stream()))
    with torch.no_grad():
        logits.copy_(torch.randn_like(logits))
    want = once()
    for g, _, s in graphs:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_routed_rows_reach_their_experts_and_come_back():
    """route, dispatch, experts, combine as the expert layer runs them, with padding tokens and dropped pairs."""
    torch.manual_seed(13)
    T, E, k, d, C = 90, 80, 4, 64, 6
    logits = torch.randn(T, E, device="cuda")
    logits[80:] = -math.inf
    x = torch.randn(T, d, device="cuda", dtype=BF16, requires_grad=True)
    logits = logits.requires_grad_()
    w, prob, ids, slot, counts = moe.route(logits, E, k, C, score="sigmoid", scale=2.0)
    y = moe.combine(moe.dispatch(x, ids, slot, E, C, k) * 3, w, ids, slot, T, k)
    kept = (slot.reshape(T, k) >= 0).float() * w
    assert torch.allclose(y.float(), 3 * kept.sum(-1, keepdim=True) * x.float(), rtol=2e-2, atol=2e-2)
    assert (y[80:] == 0).all()
    dx, dl = torch.autograd.grad(y, (x, logits), torch.randn_like(y))
    assert (dx[80:] == 0).all() and (dl[80:] == 0).all() and torch.isfinite(dl).all()
