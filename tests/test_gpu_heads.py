"""Rotary positions and the norm of query and key heads on the GPU, against the definition in 64 bits."""
import math

import pytest
import torch

from distdl_b200 import ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    """The largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def frequencies(r, head_dim):
    return torch.tensor(r.frequencies(head_dim), dtype=torch.float64, device="cuda")


def angles(r, head_dim, pos):
    return torch.polar(torch.tensor(r.scale, dtype=torch.float64, device="cuda"),
                       pos.double().unsqueeze(1) * frequencies(r, head_dim)).unsqueeze(1)


def turn(x, z, r):
    """fp64 heads turned by complex numbers ``z [tokens, 1, pairs]``."""
    n = r.rotated(x.shape[-1])
    if n == 0:
        return x
    lead = x[..., :n]
    p = lead.unflatten(-1, (n // 2, 2)) if r.interleaved else lead.unflatten(-1, (2, n // 2)).transpose(-1, -2)
    t = torch.view_as_real(torch.view_as_complex(p.contiguous()) * z)
    t = t if r.interleaved else t.transpose(-1, -2)
    return torch.cat([t.flatten(-2), x[..., n:]], dim=-1)


def assert_turned(y, x, z, r, nheads, dtype):
    """One rounding to ``dtype``, and of a pair (a, b) four roundings to fp32 of products and sums, cosine and sine within two
    units of fp32: below 2^-20 of |a| + |b|, times the magnitude."""
    ref = turn(x[:, :nheads].double(), z, r)
    size = z.abs().max().item() if z.numel() else 1.0
    bound = (half_step(dtype) + 1e-12) * ref.abs() + 2.0 ** -20 * max(size, 1.0) * 2 * x[:, :nheads].double().abs().amax(
        dim=-1, keepdim=True) + (2.0 ** -25 if dtype == FP16 else 0.0)
    err = (y[:, :nheads].double() - ref).abs()
    assert (err <= bound).all(), (err - bound).max().item()
    assert torch.equal(y[:, nheads:], x[:, nheads:])


SHAPES = [
    # head_dim, dim, interleaved
    (128, 128, False), (128, 128, True), (64, 64, False), (64, 16, True), (128, 32, False), (80, 80, False), (80, 34, False),
    (96, 96, True), (256, 256, False), (192, 64, False), (40, 26, True), (24, 24, False), (8, 8, False), (512, 512, False),
    (100, 50, False), (100, 100, True), (33, 32, False), (7, 6, True), (2, 2, False), (1, 0, False), (512, 2, True),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hd,dim,near", SHAPES)
def test_rope_matches_the_definition(hd, dim, near, dtype):
    torch.manual_seed(hd + dim)
    r = ops.Rotary(theta=10000.0, dim=dim, interleaved=near)
    x = torch.randn(2 * 19, 5, hd, device="cuda").to(dtype).requires_grad_()
    y = ops.rope(x, 19, 3, rotary=r, offset=11)
    pos = torch.arange(38, device="cuda") % 19 + 11
    z = angles(r, hd, pos)
    assert_turned(y, x, z, r, 3, dtype)
    dy = torch.randn_like(y)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert_turned(dx, dy, z.conj(), r, 3, dtype)


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 40), (3, 7), (257, 3), (5000, 9), (64, 150)])
def test_rope_sizes(tokens, heads):
    r = ops.Rotary(scaling="yarn", factor=8.0, original=512)
    x = torch.randn(tokens, heads, 128, device="cuda", dtype=BF16)
    nh = (heads + 1) // 2
    z = angles(r, 128, torch.arange(tokens, device="cuda"))
    assert_turned(ops.rope(x, tokens, nh, rotary=r), x, z, r, nh, BF16)
    keep = x.clone()
    y = ops.rope_(x, tokens, nh, rotary=r)
    assert y.data_ptr() == x.data_ptr()
    assert_turned(x, keep, z, r, nh, BF16)
    assert ops.rope(x[:0], 4, nh, rotary=r).shape == (0, heads, 128)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn", "bands"])
def test_rope_at_far_positions(scaling):
    """Angles of positions up to 2^31 - 1, where 32 bits are off by whole turns."""
    r = ops.Rotary(scaling=scaling, factor=16.0, original=4096)
    pos = torch.tensor([0, 1, 77777, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -5], device="cuda")
    x = torch.randn(7, 2, 128, device="cuda")
    for p in (pos, pos.to(torch.int32)):
        assert_turned(ops.rope(x, 7, 2, rotary=r, positions=p), x, angles(r, 128, pos), r, 2, FP32)


def test_positions_per_place_per_token_and_from_ranges():
    r = ops.Rotary(theta=1000.0)
    x = torch.randn(12, 4, 64, device="cuda", dtype=BF16)
    place = torch.tensor([9, 2, 2, 100], device="cuda")
    a = ops.rope(x, 4, 4, rotary=r, positions=place)
    assert torch.equal(a, ops.rope(x, 4, 4, rotary=r, positions=place.repeat(3).reshape(3, 4)))
    assert torch.equal(a, ops.rope(x, 4, 4, rotary=r, positions=torch.stack([place, place], 1)[:, 0]))
    assert_turned(a, x, angles(r, 64, place.repeat(3)), r, 4, BF16)
    b = ops.rope(x, 6, 4, rotary=r, ranges=((3, 2), (50, 4)))
    assert_turned(b, x, angles(r, 64, torch.tensor([3, 4, 50, 51, 52, 53] * 2, device="cuda")), r, 4, BF16)
    assert torch.equal(ops.rope(x, 4, 4, rotary=r, offset=7), ops.rope(x, 4, 4, rotary=r, ranges=((7, 4),)))


def _strided(dtype, hd, how):
    if how == "tokens apart":
        return torch.randn(9, 2, 6, hd, device="cuda").to(dtype)[:, 1]
    if how == "heads first":
        return torch.randn(6, 9, hd, device="cuda").to(dtype).transpose(0, 1)
    if how == "odd address":
        return torch.randn(9 * 6 * hd + 1, device="cuda").to(dtype)[1:].view(9, 6, hd)
    if how == "part of a wider head":
        return torch.randn(9, 6, hd + 1, device="cuda").to(dtype)[..., :hd]
    return torch.randn(9, 6, 2 * hd, device="cuda").to(dtype)[..., ::2]          # components apart


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("hd", [128, 40])
@pytest.mark.parametrize("how", ["tokens apart", "heads first", "odd address", "part of a wider head", "components apart"])
def test_rope_of_views(how, hd, dtype):
    torch.manual_seed(1)
    r = ops.Rotary(theta=10000.0)
    x = _strided(dtype, hd, how)
    z = angles(r, hd, torch.arange(9, device="cuda"))
    assert_turned(ops.rope(x, 9, 4, rotary=r), x, z, r, 4, dtype)
    xq = x.detach().clone(memory_format=torch.preserve_format).requires_grad_()
    run_norm(x.detach(), None, None, 3, 2, r, 9)
    g = torch.randn(9, 6, 1, device="cuda").to(dtype).expand(9, 6, hd)               # an expanded gradient
    (d,) = torch.autograd.grad(ops.rope(xq, 9, 4, rotary=r), xq, g)
    assert_turned(d, g.contiguous(), z.conj(), r, 4, dtype)
    if how == "components apart":
        with pytest.raises(ValueError):
            ops.rope_(x, 9, 4, rotary=r)
    else:
        keep = x.clone()
        ops.rope_(x, 9, 4, rotary=r)
        assert_turned(x, keep, z, r, 4, dtype)


def test_in_place_leaves_the_neighbourhood_alone():
    r = ops.Rotary(dim=48)
    big = torch.randn(20, 10, 64, device="cuda", dtype=BF16)
    keep = big.clone()
    ops.rope_(big[4:12, 2:7], 8, 4, rotary=r)
    ops.qk_norm_rope_(big[14:16, 1:6], 2, 2, 2, rotary=r)
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[4:12, 2:6, :48] = False
    mask[14:16, 1:5] = False
    assert torch.equal(big[mask], keep[mask])


def test_rope_in_place_carries_gradients_and_leaves_the_callers_gradient_alone():
    r = ops.Rotary(theta=10000.0, interleaved=True)
    x = torch.randn(8, 6 * 64, device="cuda", dtype=BF16, requires_grad=True)
    y = ops.rope_(x * 1, 4, 5, layout=(8, 6, 64), rotary=r)
    g = torch.randn_like(y)
    keep = g.clone()
    (d,) = torch.autograd.grad(y, x, g)
    assert torch.equal(g, keep)
    z = angles(r, 64, torch.arange(8, device="cuda") % 4)
    assert_turned(y.view(8, 6, 64), x.detach().view(8, 6, 64), z, r, 5, BF16)
    assert_turned(d.view(8, 6, 64), g.view(8, 6, 64), z.conj(), r, 5, BF16)


def test_the_gradient_of_the_gradient_is_the_rotation():
    r = ops.Rotary(theta=100.0)
    x = torch.randn(4, 2, 32, device="cuda", requires_grad=True)
    y = ops.rope(x, 4, 2, rotary=r)
    g = torch.randn_like(y, requires_grad=True)
    (d,) = torch.autograd.grad(y, x, g, create_graph=True)
    (h,) = torch.autograd.grad(d, g, x.detach())
    assert torch.allclose(h, y, atol=1e-6)


# --------------------------------------------------------------------------------------- norm of the heads
def reference(x, wq, wk, hq, hkv, r, pos, eps):
    h = x[:, :hq + hkv]
    u = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    one = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda")
    y = torch.cat([u[:, :hq] * (one if wq is None else wq), u[:, hq:] * (one if wk is None else wk)], dim=1)
    if r is not None:
        y = turn(y, angles(r, x.shape[-1], pos), r)
    return torch.cat([y, x[:, hq + hkv:]], dim=1)


def run_norm(x, wq, wk, hq, hkv, r, seq, eps=1e-6, offset=0):
    """Outputs and gradients of the kernel and of the definition, with the bounds of their differences."""
    dt = x.dtype
    pos = torch.arange(x.shape[0], device="cuda") % seq + offset
    leaves = [t for t in (x, wq, wk) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = ops.qk_norm_rope(x, seq, hq, hkv, wq, wk, rotary=r, eps=eps, offset=offset)
    dy = torch.randn(y.shape, device="cuda").to(dt)
    got = torch.autograd.grad(y, leaves, dy)
    wide = [None if t is None else t.detach().double().requires_grad_() for t in (x, wq, wk)]
    ref = reference(wide[0], wide[1], wide[2], hq, hkv, r, pos, eps)
    want = torch.autograd.grad(ref, [t for t in wide if t is not None], dy.double())
    nh, mag = hq + hkv, 1.0 if r is None else max(1.0, r.scale)
    x64, g64 = wide[0].detach()[:, :nh], dy.double()[:, :nh]
    rr = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
    top_w = max([1.0] + [t.detach().abs().max().item() for t in (wq, wk) if t is not None])
    u = (x64 * rr).abs()
    half = half_step(dt)
    # fp32: the mean of head_dim squares, its root, three products and the rotation, each within a few 2^-24 of its terms
    ty = half * ref.detach().abs()
    ty[:, :nh] += 2.0 ** -18 * mag * top_w * u.amax(-1, keepdim=True)
    tx = half * want[0].abs()
    gw = mag * top_w * 2 * g64.abs().amax(-1, keepdim=True)
    tx[:, :nh] += 2.0 ** -18 * rr * (gw + u * (gw * u).mean(-1, keepdim=True))
    small = 2.0 ** -25 if dt == FP16 else 0.0
    assert ((y.double() - ref).abs() <= ty + small).all(), ((y.double() - ref).abs() - ty).max().item()
    assert ((got[0].double() - want[0]).abs() <= tx + small).all(), ((got[0].double() - want[0]).abs() - tx).max().item()
    k = 1
    for w, rows in ((wq, slice(0, hq)), (wk, slice(hq, nh))):
        if w is None:
            continue
        # a sum of tokens * heads terms in chains of some hundred: 2^-15 of the sum of their sizes
        size = (u[:, rows].amax(-1, keepdim=True) * mag * 2 * g64[:, rows].abs().amax(-1, keepdim=True)).sum((0, 1))
        bound = half_step(w.dtype) * want[k].abs() + 2.0 ** -15 * size
        err = (got[k].double() - want[k]).abs()
        assert got[k].dtype == w.dtype and got[k].shape == w.shape
        assert (err <= bound).all(), (err - bound).max().item()
        k += 1
    return y.detach(), got


@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("hd,dim,near", SHAPES)
def test_qk_norm_rope_matches_the_definition(hd, dim, near, dtype, wdtype):
    torch.manual_seed(hd * 3 + dim)
    x = (torch.randn(2 * 17, 6, hd, device="cuda") * 3).to(dtype)
    wq, wk = ((1 + 0.2 * torch.randn(hd, device="cuda")).to(wdtype) for _ in range(2))
    run_norm(x, wq, wk, 3, 2, ops.Rotary(theta=10000.0, dim=dim, interleaved=near), 17, eps=1e-5, offset=3)


@pytest.mark.parametrize("tokens,hq,hkv,rest", [(1, 1, 1, 0), (1, 16, 4, 4), (3, 0, 2, 1), (3, 2, 0, 5), (2000, 8, 1, 1),
                                                (700, 25, 25, 25), (9000, 4, 2, 2), (2, 100, 20, 20)])
def test_qk_norm_rope_sizes(tokens, hq, hkv, rest):
    torch.manual_seed(tokens)
    x = torch.randn(tokens, hq + hkv + rest, 128, device="cuda").to(BF16)
    w = [(1 + 0.2 * torch.randn(128, device="cuda")).to(BF16) for _ in range(2)]
    run_norm(x, w[0], w[1], hq, hkv, ops.Rotary(scaling="bands", factor=8.0, original=512), tokens)


@pytest.mark.parametrize("which", ["none", "query", "key"])
def test_qk_norm_without_a_weight_or_a_rotation(which):
    x = torch.randn(50, 7, 64, device="cuda").to(BF16)
    w = (1 + 0.2 * torch.randn(64, device="cuda")).to(BF16)
    run_norm(x, w if which == "query" else None, w.clone() if which == "key" else None, 4, 2, None, 50)
    run_norm(x.detach(), w.detach() if which == "query" else None, w.detach().clone() if which == "key" else None, 4, 2,
             ops.Rotary(), 25)


def test_heads_of_zeros_and_of_huge_values():
    """A head of zeros stays one (eps keeps the root finite) and so does its gradient; squares up to 1e38 are no trouble."""
    x = torch.zeros(4, 3, 128, device="cuda")
    x[1] = 1e17
    x[2] = 1e-20
    r = ops.Rotary()
    w = torch.ones(128, device="cuda")
    y, got = run_norm(x, w, w.clone(), 1, 1, r, 4)
    assert torch.isfinite(y).all() and torch.isfinite(got[0]).all() and (y[0, :2] == 0).all()


def test_nothing_but_the_head_itself_sees_a_nan():
    x = torch.randn(5, 4, 128, device="cuda", dtype=BF16)
    x[2, 1, 77] = float("nan")
    y = ops.qk_norm_rope(x, 5, 2, 1, rotary=ops.Rotary())
    bad = torch.isnan(y).any(-1)
    assert bad.sum() == 1 and bad[2, 1]


def test_qk_norm_in_place_equals_the_new_tensor():
    r = ops.Rotary(theta=10000.0)
    for dt, hd in ((BF16, 128), (FP32, 48), (BF16, 37)):
        r = ops.Rotary(theta=10000.0, dim=hd // 2 * 2)
        x = torch.randn(30, 9, hd, device="cuda").to(dt)
        w = (1 + 0.2 * torch.randn(hd, device="cuda")).to(dt)
        y = ops.qk_norm_rope(x, 15, 5, 2, w, w, rotary=r)
        version = x._version
        assert ops.qk_norm_rope_(x, 15, 5, 2, w, w, rotary=r) is x and x._version > version
        assert torch.equal(x, y)


def test_the_gradients_do_not_depend_on_the_run():
    torch.manual_seed(5)
    x = torch.randn(3000, 12, 128, device="cuda", dtype=BF16, requires_grad=True)
    w = [torch.randn(128, device="cuda", requires_grad=True) for _ in range(2)]
    dy = torch.randn_like(x)
    runs = [torch.autograd.grad(ops.qk_norm_rope(x, 1000, 8, 2, *w, rotary=ops.Rotary()), (x, *w), dy) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_gradient_against_differences():
    torch.manual_seed(6)
    r = ops.Rotary(theta=50.0, dim=24)
    x = torch.randn(3, 4, 32, device="cuda", requires_grad=True)
    w = [(1 + 0.2 * torch.randn(32, device="cuda")).requires_grad_() for _ in range(2)]
    dy = torch.randn(3, 4, 32, device="cuda")
    loss = lambda *t: (ops.qk_norm_rope(t[0], 3, 2, 1, t[1], t[2], rotary=r).double() * dy.double()).sum()   # noqa: E731
    grads = torch.autograd.grad(loss(x, *w), (x, *w))
    for k, t in enumerate((x, *w)):
        direction = torch.randn_like(t)
        step = 2.0 ** -7
        with torch.no_grad():
            args = [x, *w]
            args[k] = t + step * direction
            up = loss(*args)
            args[k] = t - step * direction
            down = loss(*args)
        want = ((up - down) / (2 * step)).item()
        have = (grads[k].double() * direction.double()).sum().item()
        # the third derivative along a unit-sized direction times step^2 / 6, and fp32 noise over the step
        assert abs(have - want) <= 2e-3 * max(1.0, grads[k].norm().item() * direction.norm().item())


def test_gathered_weights_collect_their_gradient_beside_them():
    x = torch.randn(64, 6, 128, device="cuda", dtype=BF16, requires_grad=True)
    w = [torch.ones(128, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2)]
    dy = torch.randn_like(x)
    plain = torch.autograd.grad(ops.qk_norm_rope(x, 64, 3, 2, *w, rotary=ops.Rotary()), w, dy)
    for t in w:
        t.main_grad = torch.full((128,), 2.0, device="cuda")
    ops.qk_norm_rope(x, 64, 3, 2, *w, rotary=ops.Rotary()).backward(dy)
    for t, p in zip(w, plain):
        assert t.grad is None
        assert torch.allclose(t.main_grad - 2.0, p.float(), rtol=2.0 ** -8, atol=1e-4)


def test_on_another_stream_and_captured_in_graphs():
    r = ops.Rotary(theta=10000.0)
    x = torch.randn(40, 6, 128, device="cuda", dtype=BF16, requires_grad=True)
    w = [torch.ones(128, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2)]
    dy = torch.randn_like(x)

    def step():
        y = ops.qk_norm_rope(x, 20, 3, 2, *w, rotary=r)
        z = ops.rope(y, 20, 5, rotary=r)
        return [y.detach(), z.detach(), *torch.autograd.grad(z, (x, *w), dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graphs = []
    for _ in range(2):                                       # two graphs of the same leaves, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    want = step()
    streams = [torch.cuda.Stream() for _ in graphs]
    for s, (graph, _) in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_one_weight_for_queries_and_keys():
    """Its gradient is the sum of both, also where it is collected beside the weight."""
    x = torch.randn(200, 6, 128, device="cuda", dtype=BF16)
    w = torch.ones(128, device="cuda", requires_grad=True)
    dy = torch.randn_like(x)
    both = [torch.ones(128, device="cuda", requires_grad=True) for _ in range(2)]
    want = sum(torch.autograd.grad(ops.qk_norm_rope(x, 200, 3, 3, *both, rotary=ops.Rotary()), both, dy))
    assert torch.equal(torch.autograd.grad(ops.qk_norm_rope(x, 200, 3, 3, w, w, rotary=ops.Rotary()), w, dy)[0], want)
    w.main_grad = torch.zeros(128, device="cuda")
    ops.qk_norm_rope(x, 200, 3, 3, w, w, rotary=ops.Rotary()).backward(dy)
    assert torch.equal(w.grad + w.main_grad, want)


def test_differentiated_twice_and_forwards():
    """The gradient of a gradient, and forward-mode derivatives, by elementary operations."""
    torch.manual_seed(7)
    r = ops.Rotary(theta=100.0)
    x = torch.randn(3, 3, 16, device="cuda", dtype=torch.float32, requires_grad=True)
    w = (1 + 0.1 * torch.randn(16, device="cuda")).requires_grad_()
    dy = torch.randn(3, 3, 16, device="cuda")

    def twice(x, w):
        y = ops.qk_norm_rope(x, 3, 2, 1, w, w, rotary=r)
        g, = torch.autograd.grad(y, x, dy.to(y.dtype), create_graph=True)
        return torch.autograd.grad(g.square().sum(), (x, w))

    wide = twice(x.detach().double().requires_grad_(), w.detach().double().requires_grad_())
    for a, b in zip(twice(x, w), wide):
        assert torch.allclose(a.double(), b, rtol=1e-4, atol=1e-4 * b.abs().max().item())
    import torch.autograd.forward_ad as fwd
    t = torch.randn_like(x)
    with torch.no_grad(), fwd.dual_level():
        out = fwd.unpack_dual(ops.rope(fwd.make_dual(x.detach(), t), 3, 3, rotary=r))
        assert torch.allclose(out.tangent, ops.rope(t, 3, 3, rotary=r), atol=1e-5)
    many = torch.func.vmap(lambda z: ops.rope(z, 3, 3, rotary=r))(torch.stack([x.detach(), t]))
    assert torch.allclose(many[1], ops.rope(t, 3, 3, rotary=r), atol=1e-5)


def test_in_inference_mode_and_without_heads_to_turn():
    r = ops.Rotary(theta=10000.0)
    with torch.inference_mode():
        x = torch.randn(6, 5, 64, device="cuda", dtype=BF16)
        y = ops.qk_norm_rope(x, 6, 3, 1, rotary=r)
        z = ops.rope(x, 6, 4, rotary=r)
        assert torch.equal(ops.rope_(x.clone(), 6, 4, rotary=r), z)
        assert torch.equal(ops.qk_norm_rope_(x, 6, 3, 1, rotary=r), y)
    x = torch.randn(6, 5, 64, device="cuda", dtype=BF16, requires_grad=True)
    w = [torch.ones(64, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2)]
    y = ops.qk_norm_rope(x, 6, 0, 0, *w, rotary=r)
    dy = torch.randn_like(y)
    grads = torch.autograd.grad(y, (x, *w), dy)
    assert torch.equal(y, x) and torch.equal(grads[0], dy) and not grads[1].any() and not grads[2].any()
    empty = ops.qk_norm_rope(x[:0], 6, 3, 1, *w, rotary=r)
    grads = torch.autograd.grad(empty, (x, *w), empty.detach(), allow_unused=True)
    assert empty.shape == (0, 5, 64) and not grads[0].any() and not grads[1].any() and not grads[2].any()
    assert torch.equal(ops.rope_(x.detach(), 6, 5, rotary=ops.Rotary(dim=0)), x)


def test_only_what_is_asked_for_gets_a_gradient():
    r = ops.Rotary()
    x = torch.randn(30, 6, 128, device="cuda", dtype=BF16, requires_grad=True)
    wq, wk = (torch.ones(128, device="cuda", dtype=BF16) for _ in range(2))
    dy = torch.randn_like(x)
    dx, = torch.autograd.grad(ops.qk_norm_rope(x, 30, 3, 2, wq, wk, rotary=r), x, dy)
    wk.requires_grad_()
    only, = torch.autograd.grad(ops.qk_norm_rope(x.detach(), 30, 3, 2, wq, wk, rotary=r), wk, dy)
    every = torch.autograd.grad(ops.qk_norm_rope(x, 30, 3, 2, wq.requires_grad_(), wk, rotary=r), (x, wq, wk), dy)
    assert torch.equal(every[0], dx) and torch.equal(every[2], only)


def test_positions_changed_before_the_backward_pass_are_noticed():
    x = torch.randn(4, 2, 64, device="cuda", requires_grad=True)
    pos = torch.arange(4, device="cuda")
    for y in (ops.rope(x, 4, 2, rotary=ops.Rotary(), positions=pos),
              ops.qk_norm_rope(x, 4, 1, 1, rotary=ops.Rotary(), positions=pos)):
        pos += 1
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_a_leaf_is_not_turned_in_place():
    x = torch.randn(4, 3, 64, device="cuda", requires_grad=True)
    keep = x.detach().clone()
    with pytest.raises(RuntimeError):
        ops.rope_(x, 4, 3, rotary=ops.Rotary())
    assert torch.equal(x, keep)


def test_ranges_first_met_in_a_graph():
    x = torch.randn(7, 2, 64, device="cuda")
    ranges = ((11, 3), (501, 4))
    r = ops.Rotary()
    ops.rope(x, 7, 2, rotary=r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rope(x, 7, 2, rotary=r, ranges=ranges)
    eager = ops.rope(x, 7, 2, rotary=r, ranges=ranges)
    graph.replay()
    assert torch.equal(y, eager)


def test_offsets_beyond_32_bits():
    """Tokens whose elements lie more than 2^31 apart."""
    big = torch.empty((1 << 31) + (1 << 12), device="cuda", dtype=BF16)
    x = big.as_strided((2, 3, 128), ((1 << 31) + 8, 128, 1))
    x.copy_(torch.randn(2, 3, 128, device="cuda"))
    r = ops.Rotary()
    keep = x.clone()
    assert_turned(ops.rope(x, 2, 2, rotary=r), keep, angles(r, 128, torch.arange(2, device="cuda")), r, 2, BF16)
    y = ops.qk_norm_rope(keep, 2, 1, 1, rotary=r)
    ops.qk_norm_rope_(x, 2, 1, 1, rotary=r)
    assert torch.equal(x, y)


HALVES = [(128, 50), (128, 2), (128, 126), (64, 34), (256, 24), (512, 510), (512, 4), (40, 38), (8, 6), (16, 10), (24, 4)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hd,dim", HALVES)
def test_halves_that_are_not_whole_vectors(hd, dim, dtype):
    if dtype == FP32 and hd == 512:
        hd, dim = 256, dim // 4 * 2                           # (the most that a warp holds as vectors)
    torch.manual_seed(hd + dim)
    r = ops.Rotary(theta=10000.0, dim=dim)
    x = torch.randn(70, 9, hd, device="cuda").to(dtype).requires_grad_()
    z = angles(r, hd, torch.arange(70, device="cuda") % 35 + 5)
    y = ops.rope(x, 35, 7, rotary=r, offset=5)
    assert_turned(y, x, z, r, 7, dtype)
    dy = torch.randn_like(y)
    assert_turned(torch.autograd.grad(y, x, dy)[0], dy, z.conj(), r, 7, dtype)
    flat = x.detach().clone()
    assert torch.equal(ops.rope_(flat, 35, 7, rotary=r, offset=5), y)
    w = [(1 + 0.2 * torch.randn(hd, device="cuda")).to(dtype) for _ in range(2)]
    y, _ = run_norm(x.detach() * 2, *w, 4, 3, r, 35, offset=5)
    flat = x.detach() * 2
    assert torch.equal(ops.qk_norm_rope_(flat, 35, 4, 3, *[t.detach() for t in w], rotary=r, offset=5), y)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_many_heads_with_halves_that_are_not_whole_vectors(dtype):
    torch.manual_seed(2)
    r = ops.Rotary(dim=50)
    x = torch.randn(900, 30, 128, device="cuda").to(dtype)
    assert_turned(ops.rope(x, 900, 29, rotary=r), x, angles(r, 128, torch.arange(900, device="cuda")), r, 29, dtype)
    w = [(1 + 0.2 * torch.randn(128, device="cuda")).to(dtype) for _ in range(2)]
    run_norm(x, *w, 19, 5, r, 300)


@pytest.mark.parametrize("dim", [50, 32])
def test_what_stays_is_a_copy_whatever_it_is(dim):
    x = torch.randn(11, 5, 128, device="cuda", dtype=BF16)
    r = ops.Rotary(dim=dim)
    clean = ops.rope(x, 11, 4, rotary=r)
    for k, v in enumerate((float("inf"), float("nan"), -float("inf"))):
        x[:, :, dim + k::7] = v
    for y in (ops.rope(x, 11, 4, rotary=r), ops.rope_(x.clone(), 11, 4, rotary=r)):
        assert torch.equal(y[..., :dim], torch.cat([clean[:, :4], x[:, 4:]], 1)[..., :dim])
        # (of a NaN the bits behind its first are not kept by a conversion)
        torch.testing.assert_close(y[..., dim:], x[..., dim:], rtol=0.0, atol=0.0, equal_nan=True)
