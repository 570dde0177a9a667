"""Positions from several ranges: the same as the positions listed, and nothing of one call is left for the next (CPU)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from distdl_b200 import ops
from distdl_b200.ops import rotary as rotary_module

RANGES = [((3, 7),), ((0, 3), (40, 4)), ((40, 4), (3, 3)), ((5, 4), (9, 3)), ((2, 0), (9, 3), (1, 4)), ((8, 2), (0, 2), (20, 3)),
          ((-4, 2), (1 << 20, 5))]


def listed(ranges):
    return torch.cat([torch.arange(a, a + n) for a, n in ranges])


@pytest.mark.parametrize("ranges", RANGES, ids=str)
def test_ranges_are_the_positions_that_they_list(ranges):
    torch.manual_seed(0)
    x = torch.randn(14, 4, 16, dtype=torch.float64)
    r = ops.Rotary(dim=12, interleaved=True)
    assert torch.equal(ops.rope(x, 7, 3, rotary=r, ranges=ranges), ops.rope(x, 7, 3, rotary=r, positions=listed(ranges)))
    assert torch.equal(ops.qk_norm_rope(x, 7, 2, 1, rotary=r, ranges=ranges),
                       ops.qk_norm_rope(x, 7, 2, 1, rotary=r, positions=listed(ranges)))


@pytest.mark.parametrize("ranges", RANGES, ids=str)
def test_ranges_first_met_in_inference_mode(ranges, monkeypatch):
    """What a gradient keeps of the positions is not what a call in inference mode has made (the launches themselves stubbed)."""
    ranges = tuple((a + 1000, n) for a, n in ranges)           # (met nowhere else)
    monkeypatch.setattr(rotary_module, "_native_ok", lambda *t: True)
    monkeypatch.setattr(rotary_module, "_call", lambda *a, **k: None)
    monkeypatch.setattr(rotary_module, "_parts", lambda d: 1)
    r, x = ops.Rotary(), torch.randn(14, 4, 16)
    w = torch.ones(16, requires_grad=True)
    calls = (lambda t: ops.rope(t, 7, 3, rotary=r, ranges=ranges),
             lambda t: ops.rope_(t * 1, 7, 3, rotary=r, ranges=ranges),
             lambda t: ops.qk_norm_rope(t, 7, 2, 1, w, w, rotary=r, ranges=ranges))
    for call in calls:
        with torch.inference_mode():
            call(x)
        call(x.clone().requires_grad_()).sum().backward()


@pytest.mark.parametrize("ranges", RANGES, ids=str)
def test_ranges_first_met_under_fake_tensors(ranges):
    r = ops.Rotary()
    ranges = tuple((a + 2000, n) for a, n in ranges)           # (met nowhere else)
    with FakeTensorMode():
        ops.rope(torch.randn(14, 4, 16), 7, 3, rotary=r, ranges=ranges)
    x = torch.randn(14, 4, 16)
    assert torch.equal(ops.rope(x, 7, 3, rotary=r, ranges=ranges), ops.rope(x, 7, 3, rotary=r, positions=listed(ranges)))


@pytest.mark.parametrize("place", [dict(), dict(offset=3), dict(ranges=((0, 3), (40, 4)))], ids=str)
def test_tables_first_made_under_fake_tensors_or_in_inference_mode(place):
    x = torch.randn(14, 4, 16)
    for theta, mode in ((701.0, FakeTensorMode()), (702.0, torch.inference_mode())):
        with mode:
            ops.rope_(torch.randn(14, 4, 16), 7, 3, theta=theta, **place)
        y = x.clone().requires_grad_()
        out = ops.rope_(y * 1, 7, 3, theta=theta, **place)
        out.sum().backward()
        assert torch.allclose(out, ops.rope(x, 7, 3, rotary=ops.Rotary(theta=theta), **place), atol=1e-5)
        with FakeTensorMode():
            ops.rope_(torch.randn(14, 4, 16), 7, 3, theta=theta, **place)


def test_tables_are_kept_under_modes_whose_tensors_are_none_of_their_own():
    from torch.utils.flop_counter import FlopCounterMode

    from distdl_b200.ops.activation import rope_table, rope_table_ranges
    with FlopCounterMode(display=False):
        a, b = rope_table(7, 16, 703.0, "cpu"), rope_table_ranges(((1, 3), (9, 2)), 16, 703.0, "cpu")
    assert rope_table(7, 16, 703.0, "cpu") is a and rope_table_ranges(((1, 3), (9, 2)), 16, 703.0, "cpu") is b
    with FlopCounterMode(display=False):
        assert rope_table(7, 16, 703.0, "cpu") is a


def test_ranges_that_are_refused():
    x, r = torch.randn(14, 4, 16), ops.Rotary()
    for ranges, tokens in ((((0, 6),), 14), (((0, 8), (3, -1)), 14), (((0, 7),), 13), ((), 14)):
        with pytest.raises(ValueError):
            ops.rope(x[:tokens], 7, 3, rotary=r, ranges=ranges)
    with pytest.raises(ValueError):
        ops.rope(x, 7, 3, rotary=r, ranges=((0, 7),), offset=1)
    assert ops.rope(x[:0], 7, 3, rotary=r, ranges=((0, 7),)).shape == (0, 4, 16)
    assert ops.rope(x[:0], 0, 3, rotary=r, ranges=((0, 0),)).shape == (0, 4, 16)


def test_the_native_entry_point_refuses_a_second_range_before_the_first():
    from distdl_b200 import _native
    if not _native.available():
        pytest.skip("the native library is not built")
    lib = _native.lib()
    call = rotary_module._CALL.pack(64, 0, 128, 0, 0, 0, 0, 0, 0, 0, 32, 16, 32, 16, 32, 16, 0, 0, 4, 0, 0, 2, 0, 0, 16, 0, 0, 0,
                                    0, 0, 1.0, 1.0, 1e-6)
    for split, want in ((3, 0), (1 << 40, 0), (-1, 1001)):
        two = call + rotary_module._SECOND.pack(split, 5)
        assert lib.dd_heads(two, len(two), None) == want          # (no tokens: nothing is launched)
    assert lib.dd_heads(call + b"12345678", len(call) + 8, None) == 1001
