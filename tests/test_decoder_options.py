"""Decoders with norms of query and key heads, other rotations and other routers on CPU ranks: the same loss and the same
gradient norm on every worker grid from one checkpoint, and what the options refuse."""
import math

import pytest
import torch

from distdl_b200 import ops
from dist_harness import run_ranks


def options(family):
    from distdl_b200 import models
    make = models.mixtral_tiny if family == "moe" else models.llama_tiny
    cfg = make(dtype=torch.float32, max_seq=16, vocab_size=100, d_model=64, ffn_dim=96)
    cfg.n_layers, cfg.collect_state = 2, True
    cfg.n_heads, cfg.n_kv_heads = 4, 2
    cfg.qk_norm = True
    cfg.rotary = ops.Rotary(theta=1000.0, dim=12, interleaved=True, scaling="yarn", factor=4.0, original=8)
    if family == "norm only":
        cfg.rotary = ops.Rotary(theta=1000.0, scaling="bands", factor=4.0, original=8)
    if family == "moe":
        cfg.n_experts, cfg.top_k, cfg.capacity_factor = 8, 2, 16.0      # no token is dropped, whatever the grid
        cfg.router_score, cfg.router_bias, cfg.router_scale = "sigmoid", True, 2.0
        cfg.router_groups, cfg.router_top_groups, cfg.router_group_score = 4, 2, "top2"
    return cfg


def body_loss_and_gradient(rank, world, family, dp, tp, cp, mode, serial, tokens):
    import torch.distributed as dist

    from distdl_b200 import models, parallel
    cfg = options(family)
    cfg.cp_mode = mode
    torch.manual_seed(rank)
    layout = models.ParallelLayout(dp, tp, cp=cp)
    model = models.Decoder(cfg, layout)
    if serial is None:
        with torch.no_grad():
            for n, p in model.named_parameters():
                if "_norm" in n:
                    p.add_(0.2 * torch.randn(p.shape))
    else:
        model.load_state_dict(serial if rank == 0 else {})
    mine = tokens[layout.dp_index * len(tokens) // dp:(layout.dp_index + 1) * len(tokens) // dp]
    loss = model.loss(mine[:, :-1], mine[:, 1:], scale=1.0 / (len(tokens) * 16))
    loss.backward()
    model.release_gathered()
    norms = {n: p.grad for n, p in model.named_parameters() if p.grad is not None}
    assert any("q_norm" in n for n in norms) and any("k_norm" in n for n in norms)
    norm = parallel.clip_grad_norm_(model.parameters(), 0.01)
    after = parallel.clip_grad_norm_(model.parameters(), 1e9)
    model.balance_routers(0.125)
    biases = [m.router_bias.tolist() for m in model.modules() if getattr(m, "router_bias", None) is not None]
    total = loss.detach().clone()
    dist.all_reduce(total)
    sd = model.state_dict()
    assert rank == 0 or len(sd) == 0, list(sd)[:4]
    return float(total), float(norm), float(after), biases, ({k: v.clone() for k, v in sd.items()} if rank == 0 else None)


GRIDS = [(2, 1, 1, "ring"), (1, 2, 1, "ring"), (1, 1, 2, "ring"), (1, 1, 2, "zigzag"), (1, 1, 2, "a2a")]


@pytest.mark.parametrize("family", ["heads", "norm only", "moe"])
def test_worker_grids_agree(family):
    torch.manual_seed(0)
    tokens = torch.randint(0, 100, (2, 17))
    first = run_ranks("test_decoder_options", "body_loss_and_gradient", 1, args=(family, 1, 1, 1, "ring", None, tokens),
                      timeout=300)[0]
    assert math.isfinite(first[0]) and abs(first[2] - 0.01) < 1e-4
    serial = {k: v for k, v in first[4].items()}
    for k in serial:
        if k.endswith("router_bias"):
            assert serial[k].abs().max() == 0.125
            serial[k] = torch.zeros_like(serial[k])
    if family == "moe":
        assert sum(k.endswith("router_bias") for k in serial) == 2
        assert all(set(b) <= {-0.125, 0.0, 0.125} and any(b) for b in first[3])
    for dp, tp, cp, mode in GRIDS:
        if family == "moe" and tp > 1:
            continue
        out = run_ranks("test_decoder_options", "body_loss_and_gradient", 2, args=(family, dp, tp, cp, mode, serial, tokens),
                        timeout=300)
        for loss, norm, after, biases, _ in out:
            assert abs(loss - first[0]) < 1e-5 * abs(first[0]), (dp, tp, cp, mode, loss, first[0])
            assert abs(norm - first[1]) < 1e-4 * first[1], (dp, tp, cp, mode, norm, first[1])
            assert abs(after - 0.01) < 1e-4
            assert biases == first[3]


def body_checkpoint(rank, world, tmp):
    from distdl_b200 import models
    from distdl_b200.parallel import SyntheticTokens, Trainer
    cfg = options("moe")
    cfg.collect_state = False

    def make():
        torch.manual_seed(0)
        return Trainer(models.Decoder(cfg, models.ParallelLayout(world, 1)), global_tokens_per_step=2 * world * 16,
                       micro_batch=1, lr=1e-3, warmup_steps=0, max_grad_norm=1.0)

    a = make()
    block = SyntheticTokens(2, 16, 100, dp_index=rank).next()
    for _ in range(2):
        a.step(block)
        a.model.balance_routers(0.1)
    a.save_checkpoint(tmp)
    b = make()
    manifest = b.load_checkpoint(tmp)
    assert "Rotary" in str(manifest["model"]["rotary"])
    mine, other = (t.model.blocks[0].mlp.router_bias for t in (a, b))
    assert torch.equal(mine, other) and mine.abs().max() > 0
    return abs(a.step(block).item() - b.step(block).item())


def test_checkpoints_keep_the_routers_bias(tmp_path):
    assert max(run_ranks("test_decoder_options", "body_checkpoint", 2, args=(str(tmp_path),), timeout=300)) < 1e-6


def body_generate(rank, world):
    from distdl_b200 import models
    torch.manual_seed(0)
    model = models.Decoder(options("heads"), models.ParallelLayout(1, 1))
    tokens = torch.randint(0, 100, (2, 5))
    out = model.generate(tokens, 3)
    model.train()
    assert out.shape == (2, 8) and torch.equal(out[:, :5], tokens)
    return out.tolist()


def test_generate_works_in_place():
    run_ranks("test_decoder_options", "body_generate", 1, timeout=200)


def test_options_that_do_not_fit_are_refused():
    from distdl_b200 import models
    cfg = options("heads")
    cfg.rotary = ops.Rotary(dim=64)
    with pytest.raises(ValueError):
        models.Decoder(cfg, models.ParallelLayout(1, 1))
    assert models.DecoderConfig(qk_norm=True).num_parameters() - models.DecoderConfig().num_parameters() == 32 * 2 * 128
