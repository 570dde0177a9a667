"""Routing settings: the plain path, what is refused, the balancing bias (CPU)."""
import math

import pytest
import torch

from distdl_b200 import ops
from distdl_b200.ops import moe


def test_defaults_and_the_general_form_agree():
    torch.manual_seed(0)
    logits = torch.randn(37, 12, requires_grad=True)
    a = moe.route(logits, 10, 3, 6)
    b = moe.route(logits, 10, 3, 6, bias=torch.zeros(10))
    for x, y in zip(a, b):
        assert torch.allclose(x.float(), y.float(), atol=1e-6)
    ga, = torch.autograd.grad(a[0].square().sum() + a[1].square().sum(), logits)
    gb, = torch.autograd.grad(b[0].square().sum() + b[1].square().sum(), logits)
    assert torch.allclose(ga, gb, atol=1e-5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradients_of_the_plain_path(score, renormalize):
    torch.manual_seed(1)
    logits = torch.randn(5, 8, dtype=torch.float64, requires_grad=True)
    bias = torch.linspace(0, 7, 8)

    def both(x):
        w, p = moe._route_weights(x, 8, moe._choose(x, 8, 3, (score, bias, 1, 1, "max", renormalize, 2.0)),
                                  (score, bias, 1, 1, "max", renormalize, 2.0))
        return w.double(), p.double()

    grads = torch.autograd.grad(sum((o * torch.arange(1, o.numel() + 1).reshape(o.shape)).sum() for o in both(logits)), logits)
    h, want = 1e-2, torch.zeros_like(logits)
    with torch.no_grad():
        for i in range(logits.numel()):
            e = torch.zeros(logits.numel(), dtype=torch.float64)
            e[i] = h
            up, down = (sum((o * torch.arange(1, o.numel() + 1).reshape(o.shape)).sum() for o in both(logits + s * e.view(5, 8)))
                        for s in (1, -1))
            want.view(-1)[i] = (up - down) / (2 * h)
    # outputs are rounded to fp32 (sums up to 200: 2e-5 each over the step), third derivatives times h^2 / 6
    assert torch.allclose(grads[0], want, atol=2e-2)


def test_masked_experts_and_padding_tokens():
    logits = torch.tensor([[1.0, -math.inf, 3.0, 2.0], [-math.inf] * 4, [-math.inf, 0.5, -math.inf, -math.inf]])
    for score in ("softmax", "sigmoid"):
        w, prob, ids, slot, counts = moe.route(logits, 4, 2, 1, score=score, scale=2.0)
        assert ids.tolist() == [2, 3, -1, -1, 1, -1]
        assert slot.tolist() == [0, 0, -1, -1, 0, -1] and counts.tolist() == [0, 1, 1, 1]
        assert (w[1] == 0).all() and w[2].tolist() == [2.0, 0.0] and torch.isfinite(prob).all()


def test_groups():
    logits = torch.tensor([[3.0, 0.0, 2.0, 2.0, 1.0, 1.0]])
    assert moe.route(logits, 6, 2, 9, groups=3, top_groups=1, scale=2.0)[2].tolist() == [0, 1]
    assert moe.route(logits, 6, 2, 9, groups=3, top_groups=1, group_score="top2", score="sigmoid")[2].tolist() == [2, 3]
    # sums of two: 1.45, 1.76 and 1.46, so that the best expert's group is left out
    assert moe.route(logits, 6, 2, 9, groups=3, top_groups=2, group_score="top2", score="sigmoid")[2].tolist() == [2, 3]
    assert moe.route(logits, 6, 2, 9, groups=3, top_groups=2, score="sigmoid")[2].tolist() == [0, 2]


def test_balance_bias():
    bias = torch.zeros(4)
    moe.balance_bias_(bias, torch.tensor([1, 5, 3, 3], dtype=torch.int32), 0.5)
    assert bias.tolist() == [0.5, -0.5, 0.0, 0.0]
    with pytest.raises(ValueError):
        moe.balance_bias_(bias, torch.zeros(3), 0.5)


def test_calls_that_are_refused():
    x = torch.randn(5, 12)
    for args, how in (((13, 2, 4), {}), ((0, 1, 4), {}), ((12, 0, 4), {}), ((12, 13, 4), {}), ((12, 2, 4), dict(score="tanh")),
                      ((12, 2, 4), dict(group_score="mean", groups=2)), ((12, 2, 4), dict(groups=5)),
                      ((12, 2, 4), dict(groups=0)), ((12, 2, 4), dict(groups=4, top_groups=5)),
                      ((12, 2, 4), dict(groups=4, top_groups=0)), ((12, 4, 4), dict(groups=4, top_groups=1)),
                      ((12, 2, 4), dict(scale=0.0)), ((12, 2, 4), dict(scale=math.inf)),
                      ((12, 2, 4), dict(bias=torch.zeros(11))), ((12, 2, 4), dict(bias=torch.zeros(12, dtype=torch.int32)))):
        with pytest.raises(ValueError):
            moe.route(x, *args, **dict(dict(renormalize=False), **how))
    with pytest.raises(ValueError):
        ops.moe.route(x[0], 12, 2, 4, score="sigmoid")
    with pytest.raises(ValueError):
        ops.moe.route(x.long(), 12, 2, 4, score="sigmoid")


def test_native_entry_points_refuse_bad_sizes_without_a_launch():
    from distdl_b200 import _native
    if not _native.available():
        pytest.skip("the native library is not built")
    lib = _native.lib()

    def forward(ld=16, dtype=0, tokens=4, E=16, k=2, groups=1, top=1, words=1 << 20, scratch=256, logits=256, size=None):
        packed = moe._ROUTE_CALL.pack(logits, 0, 256, 256, 256, 256, 256, scratch, words, ld, dtype, tokens, E, k, 8, groups,
                                      top, 0, 0, 1, 1.0)
        return lib.dd_route_fwd(packed, len(packed) if size is None else size, None)

    assert forward(size=16) == 1001 and lib.dd_route_fwd(None, 120, None) == 1001
    assert forward(E=513, ld=600) == 1001 and forward(k=33, E=64, ld=64) == 1001 and forward(k=17) == 1001
    assert forward(ld=15) == 1001 and forward(dtype=3) == 1001 and forward(groups=3, top=1) == 1001
    assert forward(groups=4, top=5) == 1001 and forward(words=31) == 1001 and forward(scratch=260) == 1002
    assert forward(logits=0) == 1001 and forward(tokens=0) == 1001 and forward(tokens=1 << 30, k=2) == 1001
    assert lib.dd_route_bwd(256, 16, 0, 4, 16, 2, 0, 1, 1.0, 256, 256, None, None, 264, None) == 1002
    assert lib.dd_route_bwd(256, 16, 0, 4, 16, 2, 0, 1, 1.0, None, 256, None, None, 256, None) == 1001
