"""The routed pairs of an expert layer count in a captured and replayed step as in an eager one."""
import pytest
import torch

from test_gpu_decoder_options import decoder

pytestmark = pytest.mark.gpu


def test_counts_of_replays_add_up():
    model = decoder("moe")
    model.train()
    mlp = model.blocks[0].mlp
    x = torch.randn(2, 64, model.cfg.d_model, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        mlp(x)
        mlp.take_routed()
        assert mlp.take_routed().sum() == 0
        mlp(x)
        want = mlp.take_routed()
        assert want.sum() == 2 * 64 * model.cfg.top_k
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            mlp(x)
        torch.cuda.current_stream().wait_stream(side)
        mlp.take_routed()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mlp(x)
    assert mlp.take_routed().sum() == 0
    for _ in range(3):
        graph.replay()
    assert (mlp.take_routed() == 3 * want).all()
    graph.replay()
    assert (mlp.take_routed() == want).all()
    assert not any("_routed" in k for k in model.state_dict())
