"""GPU: frames one after another through the 8-bit cache against all frames at once with dense frame-causal attention."""
import pytest
import torch

from oracle import kv_cache as ok

pytestmark = pytest.mark.gpu


def _config():
    from qvggt_b200.aggregator import AggConfig
    return AggConfig(depth=2, tokens_per_frame=25, grid_w=5)


def _blocks(cfg, dev):
    from qvggt_b200.synthetic import random_block
    gen = torch.Generator(device=dev).manual_seed(5)
    return [[random_block(cfg, gen, dev) for _ in range(cfg.depth)] for _ in range(2)]


def _dense(cfg, blocks, frames, dev, streaming):
    """The runner with all frames at once, its global attention in 64 bits over unquantised K / V."""
    from qvggt_b200.aggregator import AggregatorRunner

    class Dense(AggregatorRunner):
        def _global_attention(self):
            T, H = self.T, cfg.heads
            q = self.ws.q.view(T, H, 64).double()
            k, v = (self.ws.kv_local[:, i * cfg.dim:(i + 1) * cfg.dim].reshape(T, H, 64).double() for i in (0, 1))
            if streaming.time_axis:
                pos = streaming._pos[:, :cfg.tokens_per_frame].repeat(1, frames)
                pos[0] = torch.arange(frames, device=dev).repeat_interleave(cfg.tokens_per_frame)
                q, k = (ok.rope_axes(x, pos, streaming.inv_freq, streaming.sections, "split").half().double()
                        for x in (q, k))
            frame = torch.arange(T, device=dev) // cfg.tokens_per_frame
            s = torch.einsum("ihd,jhd->hij", q, k) / 8
            w = s.masked_fill(frame[:, None] < frame[None], -torch.inf).softmax(-1)
            self.ws.attn.copy_(torch.einsum("hij,jhd->ihd", w, v).reshape(T, -1))

    run = Dense(cfg, *blocks, frames, dev)
    if streaming.time_axis:
        run.cos, run.sin = torch.ones_like(run.cos), torch.zeros_like(run.sin)
    return run


@pytest.mark.parametrize("time_axis", [False, True])
@pytest.mark.parametrize("per_step", [1, 3])
def test_streamed_frames_match_all_at_once(time_axis, per_step):
    """A layer's update is LayerScale (0.01) times a projection of the attention.  A code is off by at most half of
    amax / 127: about 1 % of a K or V element's size, so an update is off by about that much, the tokens by far less
    than 1e-3 of theirs; the updates themselves are compared to 3e-2 (both layers, K and V)."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = _blocks(cfg, dev)
    S, P = 6, cfg.tokens_per_frame
    x = torch.randn(S, P, cfg.dim, generator=torch.Generator().manual_seed(1)).half().to(dev)
    run = StreamingRunner(cfg, *blocks, per_step, S, dev, time_axis=time_axis, block_size=32)
    want = _dense(cfg, blocks, S, dev, run).forward(x.clone())[-1][1].view(S, P, -1)
    for _ in range(2):                  # again after a reset: the pool's blocks come back
        got = [run.step(x[i:i + per_step].clone())[-1][1].view(per_step, P, -1) for i in range(0, S, per_step)]
        got = torch.cat(got)
        dx, dw = (t.double() - x.double() for t in (got, want))
        assert (got.double() - want.double()).norm() <= 1e-3 * want.double().norm()
        assert (dx - dw).norm() <= 3e-2 * dw.norm()
        with pytest.raises(ValueError, match="holds"):
            run.step(x[:per_step].clone())
        run.reset()
    assert sorted(run.cache.free_ring.tolist()) == list(range(run.cache.free_ring.numel()))


def test_streams_are_independent():
    """Two streams in one runner give the bits of two runners."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = _blocks(cfg, dev)
    P = cfg.tokens_per_frame
    x = torch.randn(2, 4, P, cfg.dim, generator=torch.Generator().manual_seed(2)).half().to(dev)
    both = StreamingRunner(cfg, *blocks, 2, 4, dev, streams=2, time_axis=True)
    one = [StreamingRunner(cfg, *blocks, 2, 4, dev, time_axis=True) for _ in range(2)]
    for i in (0, 2):
        got = both.step(x[:, i:i + 2].reshape(4, P, -1).clone())[-1][1].view(2, 2 * P, -1)
        for s in range(2):
            want = one[s].step(x[s, i:i + 2].clone())[-1][1].view(2 * P, -1)
            assert (got[s].double() - want.double()).norm() <= 1e-3 * want.double().norm()


def test_streaming_aggregator_first_frame_is_the_models():
    """One frame, nothing cached: the streaming model is the model, but for the cache's 8 bits."""
    from qvggt_b200.aggregator import AggConfig
    from qvggt_b200.streaming import StreamingAggregator
    from qvggt_b200.synthetic import random_vggt_aggregator
    dev = torch.device("cuda", 0)
    agg = random_vggt_aggregator(AggConfig(depth=1), 4, dev, 1, pe_depth=1)
    parts = (agg.cfg, agg.pe, agg.agg_specials, agg.runner.frame_blocks, agg.runner.global_blocks)
    images = torch.rand(1, 3, 518, 518, generator=torch.Generator().manual_seed(3)).half().to(dev)
    want = agg.forward(images)[-1][1].double()
    stream = StreamingAggregator(*parts, 1, dev, max_frames=2)
    got = stream.forward(images)[-1][1].double()
    assert (got - want).norm() <= 1e-3 * want.norm()
    second = stream.forward(images)[-1][1].double()      # the same picture as frame 2: other special tokens, more keys
    assert torch.isfinite(second).all() and (second - got).norm() > 1e-3 * want.norm()
