"""GPU: what the streaming aggregator's blocks see: the frame blocks their own frame with its positions, the global
blocks the earlier frames of their own stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _config(depth=1):
    from qvggt_b200.aggregator import AggConfig
    return AggConfig(depth=depth, tokens_per_frame=25, grid_w=5)


def _blocks(cfg, dev, kind="w4", layer_scale=None):
    from qvggt_b200.synthetic import random_block
    gen = torch.Generator(device=dev).manual_seed(5)
    return [[random_block(cfg, gen, dev, kind, layer_scale) for _ in range(cfg.depth)] for _ in range(2)]


@pytest.mark.parametrize("kind", ["w4", "w8"])
def test_time_axis_leaves_the_frame_blocks_their_positions(kind):
    """A frame block attends within its frame, where all tokens have one time: the first frame block's output is the
    aggregator's, bit for bit, whatever the global blocks turn by."""
    from qvggt_b200.aggregator import AggregatorRunner
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = _blocks(cfg, dev, kind)
    x = torch.randn(2, cfg.tokens_per_frame, cfg.dim, generator=torch.Generator().manual_seed(1)).half().to(dev)
    want = AggregatorRunner(cfg, *blocks, 2, dev).forward(x.clone())[-1][0]
    outs = [StreamingRunner(cfg, *blocks, 2, 2, dev, time_axis=t, block_size=32).step(x.clone())[-1]
            for t in (False, True)]
    for frame_out, _ in outs:
        assert torch.equal(frame_out, want)
    assert not torch.equal(outs[0][1], outs[1][1])       # (the global blocks do turn by something else)
