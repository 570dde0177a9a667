"""The norm of many gradients and their clipping: plain path, refusals, and over workers (CPU)."""
import math

import pytest
import torch

from distdl_b200 import ops
from dist_harness import run_ranks


def test_plain_path_against_torch():
    torch.manual_seed(0)
    p = [torch.nn.Parameter(torch.randn(n)) for n in (3, 40, 5)]
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    for a, b in zip(p[:2], q):
        a.grad = torch.randn_like(a)
        b.grad = a.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(q, 0.5)
    assert torch.allclose(ops.grad_norm(t.grad for t in p), want)
    assert torch.allclose(ops.grad_norm([t.grad for t in p], squared=True), want.double().square())
    assert torch.allclose(ops.clip_grad_norm_(p, 0.5), want)
    assert all(torch.allclose(a.grad, b.grad) for a, b in zip(p[:2], q))
    keep = [t.grad.clone() for t in p[:2]]
    assert ops.clip_grad_norm_(p, 0.25, norm=torch.tensor(1.0)).item() == 1.0
    assert all(torch.allclose(t.grad, 0.25 * k) for t, k in zip(p, keep))
    assert ops.grad_norm([]).item() == 0.0 and ops.grad_norm(torch.full((4,), 2.0)).item() == 4.0


def test_calls_that_are_refused():
    g = torch.randn(5)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([g], bad)
    for norm in (torch.zeros(2), torch.zeros((), dtype=torch.float64)):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([g], 1.0, norm=norm)
    with pytest.raises(ValueError):
        ops.grad_norm([g, torch.arange(3)])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.randn(4, 4).to_sparse()])
    with pytest.raises(RuntimeError):
        ops.clip_grad_norm_([torch.ones(1).expand(5)], 1.0)                    # elements that share memory


def test_native_entry_point_refuses_without_a_launch():
    import array

    from distdl_b200 import _native
    if not _native.available():
        pytest.skip("the native library is not built")
    lib = _native.lib()

    def call(p, n, code, count=None, clip=1, given=1, norm=64, scratch=None, parts=0):
        p, n, code = array.array("Q", p), array.array("q", n), array.array("B", code)
        return lib.dd_grad_norm(p.buffer_info()[0], n.buffer_info()[0], code.buffer_info()[0],
                                len(p) if count is None else count, scratch, parts, norm, None, 1.0, given, clip, None)

    assert call([256, 512], [10, 10], [2, 3]) == 1001                         # an unknown type
    assert call([258], [10], [2]) == 1002                                     # fp32 at an address of halves
    assert call([256, 280], [10, 10], [2, 2]) == 1001                         # they overlap
    assert call([256, 256], [10, 10], [2, 2]) == 1001
    assert call([0], [10], [2]) == 1001
    assert call([256], [-1], [2]) == 1001
    assert call([256], [10], [2], norm=None) == 1001
    assert call([256], [10], [2], given=1, clip=0) == 1001
    assert call([256], [10], [2], given=0, scratch=None) == 1001
    assert call([256], [1 << 50], [2]) == 1003
    assert call([256], [10], [2], count=-1) == 1001


def body_clip_over_workers(rank, world):
    from distdl_b200 import parallel
    torch.manual_seed(0)
    full = [torch.randn(world, 6), torch.randn(world, 3)]
    p = [torch.nn.Parameter(torch.zeros(6)), torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(0))]
    for t, f in zip(p, full):
        t.grad = f[rank].clone()
    if rank == 1:
        p = p[:1] + p[2:]                                     # workers need not hold the same tensors
        full[1][1] = 0.0
    norm = parallel.clip_grad_norm_(p, 0.5)
    want = math.sqrt(sum(f.double().square().sum().item() for f in full)) if rank == 1 else None
    assert torch.allclose(p[0].grad, full[0][rank] * (0.5 / (norm + 1e-6)))
    return norm.item(), want


def test_clipping_over_workers():
    out = run_ranks("test_grad_norm", "body_clip_over_workers", 2, timeout=120)
    assert out[0][0] == out[1][0] and math.isclose(out[1][0], out[1][1], rel_tol=1e-6)
