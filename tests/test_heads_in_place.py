"""``ops.rope_`` with a ``Rotary`` or positions works in place wherever it runs (CPU; on a GPU: the elementary path)."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.flop_counter import FlopCounterMode

from distdl_b200 import ops
from dist_harness import run_ranks

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
R = ops.Rotary(theta=1000.0, dim=12)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("how", [dict(rotary=R), dict(positions=torch.tensor([5, 0, 2])), dict(rotary=R, ranges=((4, 1), (9, 2)))],
                         ids=lambda h: "-".join(h))
def test_the_tensor_itself_is_turned(how, dtype, device):
    torch.manual_seed(0)
    how = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in how.items()}
    x = torch.randn(6, 4, 16, device=device, dtype=dtype)
    for mode in (None, FlopCounterMode(display=False), torch.inference_mode()):
        y, z, flat = x.clone(), torch.zeros(6, 9, 16, device=device, dtype=dtype), x.clone().reshape(6, 64)
        z[:, 2:6] = x
        if mode is not None:
            mode.__enter__()
        try:
            # (under the mode: kernels and elementary operations round differently)
            want = ops.rope(x, 3, 3, **dict(dict(rotary=ops.Rotary()), **how))
            version = y._version if type(mode) is not torch.inference_mode else -1
            assert ops.rope_(y, 3, 3, **how) is y
            assert version < 0 or y._version > version
            ops.rope_(z[:, 2:6], 3, 3, **how)
            assert ops.rope_(flat, 3, 3, layout=(6, 4, 16), **how) is flat
        finally:
            if mode is not None:
                mode.__exit__(None, None, None)
        assert torch.equal(y, want) and torch.equal(z[:, 2:6], want) and torch.equal(flat, want.reshape(6, 64))
        assert (z[:, :2] == 0).all() and (z[:, 6:] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_heads_of_more_components_than_the_kernels_take(device):
    x = torch.randn(6, 2, 520, device=device)
    want = ops.rope(x, 6, 2, rotary=ops.Rotary())
    ops.rope_(x, 6, 2, rotary=ops.Rotary())
    assert torch.equal(x, want)


def test_its_gradient_and_forward_derivative():
    x = torch.randn(6, 4, 16, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: ops.rope_(t * 1, 3, 3, rotary=R), (x,), check_forward_ad=True)
    y = x * 1
    ops.rope_(y, 3, 3, rotary=R)                              # (the returned tensor is not looked at)
    d, = torch.autograd.grad(y, x, torch.ones_like(y))
    e, = torch.autograd.grad(ops.rope(x, 3, 3, rotary=R), x, torch.ones_like(y))
    assert torch.equal(d, e)
    with forward_ad.dual_level():
        t = forward_ad.make_dual(x.detach().float(), torch.ones(6, 4, 16))
        z = t * 1
        ops.rope_(z, 3, 3, rotary=R)
        assert torch.allclose(forward_ad.unpack_dual(z).tangent, ops.rope(torch.ones(6, 4, 16), 3, 3, rotary=R))


@pytest.mark.parametrize("device", DEVICES)
def test_what_cannot_be_turned_in_place_is_refused(device):
    x = torch.randn(6, 4, 16, device=device)
    with pytest.raises(RuntimeError):
        ops.rope_(x.clone().requires_grad_(), 3, 3, rotary=R)
    with pytest.raises(ValueError):
        ops.rope_(x[:, :1].expand(6, 4, 16), 3, 3, rotary=R)
    with pytest.raises(ValueError):
        ops.rope_(x.transpose(0, 1), 3, 3, rotary=R, layout=(6, 4, 16))
    with torch.no_grad():
        y = x.clone().requires_grad_()
        ops.rope_(y, 3, 3, rotary=R)
    assert torch.equal(y.detach(), ops.rope(x, 3, 3, rotary=R))


def body_decoder(rank, world, dp, tp, cp, mode, tokens):
    from distdl_b200 import models
    losses = []
    for rotary in (None, ops.Rotary(theta=1000.0)):
        cfg = models.llama_tiny(dtype=torch.float32, max_seq=16, vocab_size=100, d_model=64, ffn_dim=96)
        cfg.n_layers, cfg.n_heads, cfg.n_kv_heads, cfg.rope_theta = 2, 4, 2, 1000.0
        cfg.cp_mode, cfg.rotary = mode, rotary
        torch.manual_seed(5 + rank)
        model = models.Decoder(cfg, models.ParallelLayout(dp, tp, cp=cp))
        loss = model.loss(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        losses.append([loss.item()] + [p.grad.norm().item() for p in model.parameters() if p.grad is not None])
    return losses


@pytest.mark.parametrize("dp,tp,cp,mode", [(1, 1, 1, "ring"), (2, 1, 1, "ring"), (1, 2, 1, "ring"), (1, 1, 2, "ring"),
                                           (1, 1, 2, "zigzag"), (1, 1, 2, "a2a")])
def test_a_decoder_with_a_rotary_is_the_one_with_its_theta(dp, tp, cp, mode):
    tokens = torch.randint(0, 100, (2, 17), generator=torch.Generator().manual_seed(0))
    for a, b in run_ranks("test_heads_in_place", "body_decoder", dp * tp * cp, args=(dp, tp, cp, mode, tokens), timeout=300):
        # (fp32, tables of cosines against angles of 64 bits)
        assert len(a) == len(b) > 6 and all(abs(x - y) <= 1e-5 * max(1.0, abs(x)) for x, y in zip(a, b))
