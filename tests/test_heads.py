"""Rotary settings, the plain path of the rotations and of the heads' norm, and what they refuse (CPU)."""
import math

import pytest
import torch

from distdl_b200 import ops


def test_the_default_settings_are_those_of_the_in_place_rotation():
    x = torch.randn(6, 3, 16, dtype=torch.float32)
    a = ops.rope_(x.clone(), 3, 2, theta=777.0)
    b = ops.rope(x, 3, 2, rotary=ops.Rotary(theta=777.0))
    assert torch.allclose(a, b, atol=1e-6)
    assert torch.equal(b, ops.rope_(x.clone(), 3, 2, rotary=ops.Rotary(theta=777.0)))
    assert torch.equal(b, ops.rope_(x.clone(), 3, 2, theta=777.0, positions=torch.arange(6) % 3))
    c = ops.rope_(x.clone().reshape(6, 48), 3, 2, layout=(6, 3, 16), rotary=ops.Rotary(theta=777.0))
    assert torch.equal(c, b.reshape(6, 48))


def test_frequencies():
    base = ops.Rotary(theta=10000.0, dim=8).frequencies(16)
    assert base == tuple(10000.0 ** (-2 * i / 8) for i in range(4))
    linear = ops.Rotary(theta=10000.0, dim=8, scaling="linear", factor=4.0).frequencies(16)
    assert linear == tuple(f / 4 for f in base)
    ntk = ops.Rotary(theta=10000.0, dim=8, scaling="ntk", factor=4.0).frequencies(8)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], base[-1] / 4)          # the slowest pair is stretched by the factor
    for how, kept, slowed in (("bands", 4.0, 1.0), ("yarn", 32.0, 1.0)):
        f = ops.Rotary(theta=10000.0, scaling=how, factor=8.0, original=4096).frequencies(128)
        plain = ops.Rotary(theta=10000.0).frequencies(128)
        for a, b in zip(f, plain):
            turns = 4096 * b / (2 * math.pi)
            assert b / 8 * (1 - 1e-12) <= a <= b * (1 + 1e-12)
            if turns > 1.3 * kept:
                assert math.isclose(a, b)
            if turns < slowed / 1.3:
                assert math.isclose(a, b / 8)
    assert math.isclose(ops.Rotary(scaling="yarn", factor=4.0, original=64).scale, 0.1 * math.log(4) + 1)
    assert ops.Rotary(scaling="yarn", factor=4.0, original=64, magnitude=1.0).scale == 1.0
    assert ops.Rotary(dim=0).frequencies(64) == ()


@pytest.mark.parametrize("rotary", [None, ops.Rotary(), ops.Rotary(dim=6, interleaved=True),
                                    ops.Rotary(dim=8, scaling="yarn", factor=4.0, original=64)])
def test_gradients_of_the_plain_path(rotary):
    torch.manual_seed(0)
    x = torch.randn(6, 5, 16, dtype=torch.float64, requires_grad=True)
    w = torch.randn(16, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: ops.qk_norm_rope(a, 3, 3, 1, b, 2 * b, rotary=rotary), (x, w))
    if rotary is not None:
        assert torch.autograd.gradcheck(lambda a: ops.rope(a, 3, 4, rotary=rotary, offset=5), (x,))


def test_in_place_norm_writes_in_place():
    x = torch.randn(6, 5, 16)
    y = ops.qk_norm_rope(x, 3, 3, 1, rotary=ops.Rotary())
    assert ops.qk_norm_rope_(x, 3, 3, 1, rotary=ops.Rotary()) is x
    assert torch.equal(x, y)


@pytest.mark.parametrize("settings", [dict(theta=1.0), dict(theta=float("inf")), dict(dim=3), dict(dim=-2),
                                      dict(scaling="cubic"), dict(scaling="linear", factor=0.5),
                                      dict(scaling="linear", factor=float("nan")), dict(scaling="yarn", factor=2.0),
                                      dict(scaling="bands", factor=2.0, original=0),
                                      dict(scaling="bands", factor=2.0, original=8, low=4.0, high=4.0),
                                      dict(scaling="yarn", factor=2.0, original=8, slow=40.0),
                                      dict(magnitude=float("nan"))])
def test_settings_that_are_refused(settings):
    with pytest.raises(ValueError):
        ops.Rotary(**settings)


def test_calls_that_are_refused():
    x, r = torch.randn(6, 4, 16), ops.Rotary()
    pos = torch.arange(6)
    bad = [
        lambda: ops.rope(x, 3, 5, rotary=r),                                    # more heads than there are
        lambda: ops.rope(x, 3, -1, rotary=r),
        lambda: ops.rope(x, 0, 2, rotary=r),
        lambda: ops.rope(x, 3, 2, rotary=None),
        lambda: ops.rope(x[0], 3, 2, rotary=r),
        lambda: ops.rope(x.long(), 3, 2, rotary=r),
        lambda: ops.rope(x, 3, 2, rotary=ops.Rotary(dim=18)),
        lambda: ops.rope(x[..., :15], 3, 2, rotary=r),                          # an odd head without dim
        lambda: ops.rope(x, 3, 2, rotary=ops.Rotary(dim=2, scaling="ntk", factor=2.0)),
        lambda: ops.rope(x, 3, 2, rotary=r, positions=pos[:4]),
        lambda: ops.rope(x, 3, 2, rotary=r, positions=pos[:0]),
        lambda: ops.rope(x, 3, 2, rotary=r, positions=pos, offset=1),
        lambda: ops.rope(x, 3, 2, rotary=r, positions=pos, ranges=((0, 3),)),
        lambda: ops.rope(x, 3, 2, rotary=r, ranges=((0, 2),)),
        lambda: ops.rope_(x, 3, 2, rotary=r, layout=(6, 4, 15)),
        lambda: ops.qk_norm_rope(x, 3, 3, 2, rotary=r),
        lambda: ops.qk_norm_rope(x, 3, -1, 2, rotary=r),
        lambda: ops.qk_norm_rope(x, 3, 2, 1, torch.ones(15), rotary=r),
        lambda: ops.qk_norm_rope_(x[:, :1].expand(6, 4, 16), 3, 2, 1, rotary=r),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.rope(x, 3, 2, rotary="yarn")
    with pytest.raises(TypeError):
        ops.rope(x, 3, 2, rotary=r, positions=pos.float())
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope_(x.clone().requires_grad_(), 3, 2, 1, rotary=r)


def test_native_entry_points_refuse_bad_sizes_without_a_launch():
    from distdl_b200 import _native
    if not _native.available():
        pytest.skip("the native library is not built")
    from distdl_b200.ops.rotary import _CALL
    lib = _native.lib()

    def call(kind=0, tokens=4, hq=2, hk=0, rest=0, hd=16, dim=16, x=64, dy=0, out=128, turns=0, seq=4, dtype=0, dwq=0,
             size=None):
        packed = _CALL.pack(x, dy, out, 0, 0, dwq, 0, 0, 0, turns, 32, 16, 32, 16, 32, 16, tokens, 0, seq, kind, dtype, hq, hk,
                            rest, hd, dim, 0, 0, 0, 0, 1.0, 1.0, 1e-6)
        return lib.dd_heads(packed, len(packed) if size is None else size, None)

    assert call() == 1001                         # frequencies are missing
    assert call(dim=0, kind=3) == 1001 and call(dim=0, size=100) == 1001 and lib.dd_heads(None, 208, None) == 1001
    assert call(dim=0, hk=1) == 1001              # a rotation of heads of two kinds
    assert call(dim=0, hq=-1) == 1001 and call(dim=0, rest=-1) == 1001
    assert call(dim=0, hd=600) == 1003
    assert call(dim=3, turns=64) == 1001 and call(dim=18, turns=64) == 1001 and call(dim=4, turns=64, seq=0) == 1001
    assert call(tokens=-1, dim=0) == 1001
    assert call(tokens=1 << 40, dim=0) == 1003
    assert call(dim=0, dtype=3) == 1001
    assert call(dim=0, x=0) == 1001 and call(dim=0, out=0) == 1001 and call(dim=0, kind=2) == 1001
    assert call(dim=0, kind=2, dy=64, dwq=64) == 1001         # no room for the sums
    assert call(tokens=0, dim=0) == 0
