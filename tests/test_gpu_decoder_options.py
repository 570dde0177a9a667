"""Decoders with norms of query and key heads, other rotations and other routers on one GPU: the kernels together against the
library's operators, in training and in generation."""
import math

import pytest
import torch

from distdl_b200 import models, ops, parallel

pytestmark = pytest.mark.gpu


def decoder(family):
    make = models.mixtral_tiny if family == "moe" else models.llama_tiny
    cfg = make(max_seq=256, vocab_size=1000, d_model=512, ffn_dim=512)
    cfg.n_heads, cfg.n_kv_heads, cfg.qk_norm = 4, 2, True
    cfg.rotary = ops.Rotary(theta=10000.0, dim=64, interleaved=True, scaling="yarn", factor=4.0, original=128) \
        if family == "part" else ops.Rotary(theta=10000.0, scaling="bands", factor=4.0, original=128)
    if family == "moe":
        cfg.n_experts, cfg.top_k, cfg.capacity_factor = 80, 4, 2.0
        cfg.router_score, cfg.router_bias, cfg.router_scale = "sigmoid", True, 2.0
        cfg.router_groups, cfg.router_top_groups, cfg.router_group_score = 8, 4, "top2"
    torch.manual_seed(0)
    return models.Decoder(cfg, models.ParallelLayout(1, 1)).cuda()


@pytest.mark.parametrize("family", ["whole", "part"])
def test_kernels_against_the_librarys_operators(family, monkeypatch):
    """Loss and gradient norm: both sides round every activation to bf16 (2^-8 each, some twenty in a row, independent)."""
    model = decoder(family)
    tokens = torch.randint(0, 1000, (3, 257), device="cuda")
    seen = []
    for force in ("1", "0"):
        monkeypatch.setenv("DISTDL_FORCE_TORCH", force)
        loss = model.loss(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        model.release_gathered()
        seen.append((loss.item(), parallel.clip_grad_norm_(model.parameters(), 1e9).item()))
        model.zero_grad(set_to_none=True)
    (a, na), (b, nb) = seen
    assert abs(a - b) <= 1e-2 * a and abs(na - nb) <= 3e-2 * na, seen


@pytest.mark.parametrize("family", ["whole", "part", "moe"])
def test_training_step_with_an_optimizer_of_torchs(family):
    """Rotation, norms, routing, clipping and an optimizer other than the package's, as they run together."""
    model = decoder(family)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-2)       # (steps that a bf16 weight of 1 can take)
    tokens = torch.randint(0, 1000, (2, 257), device="cuda")
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for _ in range(3):
        loss = model.loss(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        model.release_gathered()
        norm = parallel.clip_grad_norm_(model.parameters(), 0.5)
        left = math.sqrt(sum(p.grad.double().square().sum().item() for p in model.parameters() if p.grad is not None))
        assert torch.isfinite(norm) and left <= 0.5 * (1 + 2.0 ** -7)          # one rounding per element
        opt.step()
        opt.zero_grad()
        model.balance_routers(0.01)
    assert math.isfinite(loss.item())
    moved = [n for n, p in model.named_parameters() if not torch.equal(p, before[n])]
    assert any("q_norm" in n for n in moved) and any("k_norm" in n for n in moved)
    if family == "moe":
        mlp = model.blocks[0].mlp
        assert any("router" in n for n in moved) and mlp.router_bias.abs().max() > 0
        assert int(mlp.last_dropped) >= 0 and torch.isfinite(mlp.aux_loss)


def test_recomputed_blocks_give_the_same_gradients():
    """A block that recomputes its forward pass works on the same values: the same kernels, the same order of sums."""
    tokens = torch.randint(0, 1000, (2, 257), device="cuda")
    seen = []
    for policy in ("none", "full"):
        model = decoder("whole")
        model.cfg.activation_policy = policy
        model.loss(tokens[:, :-1], tokens[:, 1:]).backward()
        model.release_gathered()
        seen.append({n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None})
    assert seen[0].keys() == seen[1].keys() and any("q_norm" in n for n in seen[0])
    for n in seen[0]:
        if "embed" not in n:                                  # (its rows are added by atomics)
            assert torch.equal(seen[0][n], seen[1][n]), n


def test_trainer_and_generation():
    from distdl_b200.parallel import SyntheticTokens, Trainer
    model = decoder("moe")
    trainer = Trainer(model, global_tokens_per_step=2 * 256, micro_batch=1, lr=1e-3, warmup_steps=0, max_grad_norm=1.0)
    block = SyntheticTokens(2, 256, 1000).next()
    assert all(math.isfinite(trainer.step(block).item()) for _ in range(2))
    out = model.generate(torch.randint(0, 1000, (2, 9), device="cuda"), 2)
    assert out.shape == (2, 11)
