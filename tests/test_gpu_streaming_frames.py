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


@pytest.mark.parametrize("time_axis", [False, True])
@pytest.mark.parametrize("per_step", [1, 2])
def test_attention_of_each_frame_over_its_own_stream(time_axis, per_step):
    """The attention's output itself, of two streams, against 64 bits over the unquantised keys and values of the same
    stream's frames so far.  A code is off by half of amax / 127, once more when its block's scale grows: about 1 % of a
    K or V element, so a score by 0.01 and the output by about 1 % and 1 % again; a key too many or too few, or of the
    other stream, changes it by its whole weight (1 / 150 at the least, of rows that are all different)."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    S, P, H, C = 6, cfg.tokens_per_frame, cfg.heads, cfg.dim
    x = torch.randn(S, 2, P, C, generator=torch.Generator().manual_seed(3)).half().to(dev)
    run = StreamingRunner(cfg, *_blocks(cfg, dev, layer_scale=1.0), per_step, S, dev, streams=2, time_axis=time_axis,
                          block_size=32)
    keys, values = [], []
    for i in range(0, S, per_step):
        run.step(x[i:i + per_step].transpose(0, 1).reshape(2 * per_step, P, C).contiguous())
        q, k, v = (t.double().view(2, per_step * P, H, 64).transpose(1, 2)
                   for t in (run.ws.q.view(run.T, C), run.ws.kv_local[:, :C], run.ws.kv_local[:, C:2 * C]))
        keys.append(k)
        values.append(v)
        k, v = torch.cat(keys, 2), torch.cat(values, 2)
        frame = torch.arange(k.shape[2], device=dev) // P
        s = (q @ k.transpose(-1, -2) / 8).masked_fill(frame[i * P:, None] < frame, -torch.inf)
        want = (s.softmax(-1) @ v).transpose(1, 2).reshape(run.T, C)
        got = run.ws.attn.view(run.T, C).double()
        for a, b in zip(got.view(-1, P, C), want.view(-1, P, C)):
            assert (a - b).norm() <= 3e-2 * b.norm()


@pytest.mark.parametrize("changed", [0, 1])
def test_a_stream_sees_nothing_of_the_other(changed):
    """With other frames in one stream the other stream's outputs keep their bits, and its own change from the first
    frame on."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config(2)
    blocks = _blocks(cfg, dev, layer_scale=1.0)
    P = cfg.tokens_per_frame
    x = torch.randn(3, 2, P, cfg.dim, generator=torch.Generator().manual_seed(4)).half().to(dev)
    y = x.clone()
    y[:, changed] = y[:, changed].flip(1)
    outs = []
    for z in (x, y):
        run = StreamingRunner(cfg, *blocks, 1, 3, dev, streams=2, time_axis=True, block_size=32)
        outs.append([run.step(f.clone())[-1][1].view(2, P, -1) for f in z])
    for a, b in zip(*outs):
        assert torch.equal(a[1 - changed], b[1 - changed]) and not torch.equal(a[changed], b[changed])


def test_the_aggregators_second_frame_reads_the_first():
    """The first frame's attention is the whole-sequence aggregator's but for the cache's 8 bits (bound as above), and
    the second frame's depends on the first picture."""
    from qvggt_b200.aggregator import AggConfig
    from qvggt_b200.streaming import StreamingAggregator
    from qvggt_b200.synthetic import random_vggt_aggregator
    dev = torch.device("cuda", 0)
    agg = random_vggt_aggregator(AggConfig(depth=1, layer_scale=1.0), 4, dev, 1, pe_depth=1, pe_layer_scale=1.0)
    parts = (agg.cfg, agg.pe, agg.agg_specials, agg.runner.frame_blocks, agg.runner.global_blocks)
    images = torch.rand(3, 3, 518, 518, generator=torch.Generator().manual_seed(5)).half().to(dev)
    agg.forward(images[:1])
    want = agg.runner.ws.attn.double()
    second = []
    for first in (0, 1):
        stream = StreamingAggregator(*parts, 1, dev, max_frames=2)
        stream.forward(images[first:first + 1])
        if first == 0:
            assert (stream.runner.ws.attn.double() - want).norm() <= 3e-2 * want.norm()
        frame_out, _ = stream.forward(images[2:])[-1]
        second.append((frame_out, stream.runner.ws.attn.clone()))
    assert torch.equal(second[0][0], second[1][0])        # a frame block does not look at other frames
    a, b = (s[1].double() for s in second)
    assert (a - b).norm() > 0.05 * a.norm()               # half of the keys are others
