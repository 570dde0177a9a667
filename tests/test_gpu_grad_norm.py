"""The norm of many gradients and their clipping on the GPU, against sums in 64 bits."""
import math

import pytest
import torch

from distdl_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float16, torch.float32)


def exact_norm(tensors):
    return math.sqrt(sum(t.double().square().sum().item() for t in tensors))


def check(tensors, max_norm, given=None):
    before = [t.clone() for t in tensors]
    want = exact_norm(before)
    keep = ops.grad_norm(tensors)
    squared = ops.grad_norm(tensors, squared=True)
    assert keep.dtype == torch.float32 and keep.shape == () and squared.dtype == torch.float64
    # one rounding of the result; the squares and sums are within 2^-40
    assert abs(keep.item() - want) <= 2.0 ** -23 * want
    assert abs(squared.item() - want * want) <= 2.0 ** -40 * want * want + 1e-300
    norm = ops.clip_grad_norm_(tensors, max_norm, norm=given)
    assert (norm is given) if given is not None else torch.equal(norm, keep)
    n = norm.item()
    scale = min(1.0, max_norm / (n + 1e-6)) if n == n else n
    for t, b in zip(tensors, before):
        ref = b.double() * scale
        # fp32: the quotient and the product, then one rounding to the type
        tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[t.dtype]
        bound = (torch.finfo(t.dtype).eps / 2 + 2.0 ** -22) * ref.abs() + tiny
        assert ((t.double() - ref).abs() <= bound).all()
        if scale == 1.0:
            assert torch.equal(t, b)
    return norm


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1,), (7, 0, 1), (8, 16, 24), (32768, 32769, 32767), (1000003,), (5,) * 500,
                                   (300, 1 << 20, 17, 65536 * 3)])
def test_norm_and_clipping(sizes, dtype):
    torch.manual_seed(sum(sizes))
    make = lambda: [(torch.randn(n, device="cuda") * 0.3).to(dtype) for n in sizes]      # noqa: E731
    size = math.sqrt(sum(sizes)) * 0.3
    check(make(), 0.5 * size + 1e-3)
    check(make(), 10 * size + 10)                            # nothing to clip
    check(make(), 0.0)


def test_mixed_types_and_shapes():
    torch.manual_seed(1)
    g = [torch.randn(13 + k, 7, device="cuda").to(TYPES[k % 3]) for k in range(40)]
    g.append(torch.randn(6, 10, 4, device="cuda").permute(2, 0, 1))              # dense in another order
    g.append(torch.zeros(0, 5, device="cuda"))
    g.append(torch.randn((), device="cuda"))
    check(g, 3.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_addresses_that_are_not_whole_vectors(dtype):
    torch.manual_seed(2)
    big = torch.randn(400000, device="cuda").to(dtype)
    keep = big.clone()
    cuts = [(1, 40001), (40003, 40004), (40006, 40013), (50001, 150000), (150000, 150001), (200007, 399999)]
    check([big[a:b] for a, b in cuts], 20.0)
    outside = torch.ones_like(big, dtype=torch.bool)
    for a, b in cuts:
        outside[a:b] = False
    assert torch.equal(big[outside], keep[outside])


def test_views_with_holes():
    torch.manual_seed(3)
    big = torch.randn(50, 40, device="cuda")
    keep = big.clone()
    check([big[:, 3:17], torch.randn(30, device="cuda")], 2.0)
    assert torch.equal(big[:, 17:], keep[:, 17:])


def test_extreme_values():
    """Squares that fp32 cannot hold, and values whose squares it loses."""
    for value in (3e25, 1e-25):
        g = [torch.full((1000,), value, device="cuda"), torch.full((3,), value, device="cuda", dtype=torch.bfloat16)]
        want = exact_norm(g)
        assert abs(ops.grad_norm(g).item() - want) <= 2.0 ** -23 * want
    g = [torch.full((1000,), 3e25, device="cuda")]
    ops.clip_grad_norm_(g, 2.0)
    assert abs(exact_norm(g) - 2.0) <= 1e-5
    for bad in (math.nan, math.inf):
        g = [torch.ones(100, device="cuda"), torch.ones(70000, device="cuda")]
        g[1][69999] = bad
        norm = ops.clip_grad_norm_(g, 1.0)
        want = torch.nn.Parameter(torch.ones(100, device="cuda")), torch.nn.Parameter(torch.ones(70000, device="cuda"))
        want[0].grad, want[1].grad = torch.ones(100, device="cuda"), torch.ones(70000, device="cuda")
        want[1].grad[69999] = bad
        torch.nn.utils.clip_grad_norm_(want, 1.0)
        assert math.isnan(norm.item()) == math.isnan(bad) and not math.isfinite(norm.item())
        assert all(torch.equal(a.isnan(), b.grad.isnan()) for a, b in zip(g, want))


def test_parameters_and_a_given_norm():
    torch.manual_seed(4)
    p = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (10, 200, 3)]
    for t in p[:2]:
        t.grad = torch.randn_like(t)
    keep = [t.grad.clone() for t in p[:2]]
    value = [t.detach().clone() for t in p]
    version = p[0].grad._version
    norm = ops.clip_grad_norm_(iter(p), 1.0)
    assert p[0].grad._version > version and all(torch.equal(a, b) for a, b in zip(p, value))
    ref = exact_norm(keep)
    assert all(torch.allclose(t.grad, k / (ref + 1e-6)) for t, k in zip(p, keep)) and abs(norm.item() - ref) < 1e-5
    check([torch.randn(1000, device="cuda") for _ in range(300)], 5.0, given=torch.tensor(17.0, device="cuda"))
    assert ops.clip_grad_norm_(p[2:], 1.0).item() == 0.0


def test_memory_that_is_shared_is_refused():
    from distdl_b200 import _native
    g = torch.randn(100, device="cuda")
    keep = g.clone()
    for pair in ([g, g], [g, g[50:]], [g[:51], g[50:]]):
        with pytest.raises(_native.NativeError):
            ops.clip_grad_norm_(pair, 1.0)
    assert torch.equal(g, keep)
    check([g[:50], g[50:]], 1.0)
    assert abs(ops.grad_norm([g, g]).item() - math.sqrt(2) * exact_norm([g])) < 1e-5


def test_the_same_in_every_run_on_streams_and_in_graphs():
    torch.manual_seed(5)
    g = [torch.randn(n, device="cuda") for n in (100000, 33, 1 << 21, 4097)]
    first = ops.grad_norm(g)
    for _ in range(3):
        assert torch.equal(first, ops.grad_norm(g))
    work = [t.clone() for t in g]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = ops.grad_norm(g)
            both = ops.clip_grad_norm_([t.clone() for t in g], 3.0)
        graphs.append((graph, norm, both, torch.cuda.Stream()))
    for graph, _, _, s in graphs:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for _, norm, both, _ in graphs:
        assert torch.equal(norm, first) and torch.equal(both, first)
    assert all(torch.equal(a, b) for a, b in zip(g, work))


def test_a_tensor_of_more_than_32_bits():
    g = torch.zeros((1 << 31) + 100, device="cuda", dtype=torch.bfloat16)
    g[-50:] = 2.0
    g[:7] = 1.0
    want = math.sqrt(50 * 4 + 7)
    assert abs(ops.clip_grad_norm_([g], 1.0).item() - want) < 1e-5
    assert abs(g[-1].item() - 2 / want) <= 2.0 ** -8 * 2 / want and g[1 << 30] == 0


def test_gradients_of_inference_mode_among_others():
    ours = torch.randn(1000, device="cuda")
    keep = ours.clone()
    with torch.inference_mode():
        other = torch.randn(77, device="cuda")
        want = math.sqrt(ours.double().square().sum().item() + other.double().square().sum().item())
        assert abs(ops.clip_grad_norm_([other, ours], 1.0).item() - want) <= 2.0 ** -23 * want
    version = ours._version
    ops.clip_grad_norm_([other, ours], 0.5)
    assert ours._version > version
    assert torch.allclose(ours, keep * (0.5 / want), rtol=1e-5, atol=0)
