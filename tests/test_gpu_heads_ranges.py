"""Positions from several ranges on the GPU: first met in inference mode, on another stream and in a graph."""
import pytest
import torch

from distdl_b200 import ops

pytestmark = pytest.mark.gpu

RANGES = [((3, 70),), ((0, 30), (400, 40)), ((400, 40), (3, 30)), ((8, 20), (0, 20), (200, 30)), ((1 << 30, 1), (7, 69))]


def listed(ranges):
    return torch.cat([torch.arange(a, a + n, device="cuda") for a, n in ranges])


def results(x, dy, w, r, **how):
    a = ops.rope(x, 70, 3, rotary=r, **how)
    b = ops.qk_norm_rope(x, 70, 2, 1, w, w, rotary=r, **how)
    grads = torch.autograd.grad((a, b), (x, w), (dy, dy)) if torch.is_grad_enabled() else ()
    return [a, ops.rope_(x * 1, 70, 3, rotary=r, **how), b, *grads]


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (50, torch.float16), (128, torch.float32)])
@pytest.mark.parametrize("where", ["inference mode", "another stream", "graph"])
@pytest.mark.parametrize("ranges", RANGES, ids=str)
def test_ranges_are_the_positions_that_they_list(ranges, where, hd, dtype):
    torch.manual_seed(0)
    # (positions met in no other case)
    shift = 10000 * (1 + ["inference mode", "another stream", "graph"].index(where)) + hd
    ranges = tuple((a + shift, n) for a, n in ranges)
    r = ops.Rotary(dim=hd // 4 * 2)
    x = torch.randn(140, 4, hd, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(140, 4, hd, device="cuda").to(dtype)
    w = torch.randn(hd, device="cuda").to(dtype).requires_grad_()
    want = results(x, dy, w, r, positions=listed(ranges))
    if where == "inference mode":
        with torch.inference_mode():
            results(x.detach(), dy, w.detach(), r, ranges=ranges)
        got = results(x, dy, w, r, ranges=ranges)
    elif where == "another stream":
        side = torch.cuda.Stream()
        busy = torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy = busy @ busy * 1e-3                     # what the first call queues is far from done
            with torch.no_grad():
                results(x, dy, w, r, ranges=ranges)
        got = results(x, dy, w, r, ranges=ranges)
        torch.cuda.synchronize()
    else:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            held = results(x, dy, w, r, ranges=ranges)
        got = results(x, dy, w, r, ranges=ranges)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("where", ["another stream", "graph"])
def test_tables_of_ranges_first_met_elsewhere(where):
    theta, ranges = (811.0, ((4, 30), (500, 40))) if where == "graph" else (812.0, ((4, 30), (500, 40)))
    x = torch.randn(140, 4, 64, device="cuda", dtype=torch.bfloat16)
    rotary = ops.Rotary(theta=theta)
    want = ops.rope(x, 70, 3, rotary=rotary, positions=listed(ranges))
    if where == "graph":
        ops.rope_(x.clone(), 70, 3, theta=theta, offset=470)      # (the table that holds these positions)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.rope_(x.clone(), 70, 3, theta=theta, ranges=ranges)
        got = ops.rope_(x.clone(), 70, 3, theta=theta, ranges=ranges)
        graph.replay()
        assert torch.equal(held, got)
    else:
        side = torch.cuda.Stream()
        busy = torch.randn(4096, 4096, device="cuda")
        y = x.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy = busy @ busy * 1e-3
            ops.rope_(y, 70, 3, theta=theta, ranges=ranges)
        got = ops.rope_(x.clone(), 70, 3, theta=theta, ranges=ranges)
        torch.cuda.synchronize()
    # one rounding to bf16 of either, and a table of fp32 (2^-24) against angles of 64 bits
    assert ((got.float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 2.0 ** -16 * x.float().abs().max()).all()
