"""The aggregator over frames as they arrive, on the 8-bit K/V cache.

:class:`~qvggt_b200.aggregator.VGGTAggregator` sees all frames of a sequence at
once: its global blocks attend from every token to every frame.  Here a step
takes the next frames only.  Their frame blocks and linears run as there; a
global block appends its K/V rows to the layer's cache
(:mod:`qvggt_b200.kv_cache`) and lets the new tokens attend to their own and
all earlier frames (the block-causal mask with one frame as its chunk), so a
frame costs its own linears and one pass over the cache, not a recomputation
of the sequence.  (The model itself attends to later frames as well: this is
its causal form, as for frames from a live camera.)

    plan -> [per layer] qkv (+ q/k norm, RoPE) -> append -> attend -> proj ...

With ``time_axis`` q and k of the global blocks turn by (time, height, width)
positions (:func:`~qvggt_b200.kv_cache.rope_axes`) in place of the model's
(height, width); the frame blocks, whose tokens all have one time, keep the
model's.  A 518 x 518 frame's K/V of all 24 layers take 68 MB of the cache.

    python -m qvggt_b200.streaming [--frames N] [--depth D] [--time-axis]

runs random weights over N frames and prints the time of each step.
"""
from __future__ import annotations

import torch

from .aggregator import AggConfig, AggregatorRunner, VGGTAggregator
from .kv_cache import PagedKVCache, rope_axes


class StreamingRunner(AggregatorRunner):
    """:class:`AggregatorRunner` whose global blocks read a cache of the earlier frames.

    ``streams`` independent sequences advance together, ``frames`` frames of
    each per step; the cache holds ``max_frames`` frames of each.  One GPU."""

    def __init__(self, cfg: AggConfig, frame_blocks, global_blocks, frames: int, max_frames: int, device,
                 streams: int = 1, time_axis: bool = False, block_size: int = 64):
        super().__init__(cfg, frame_blocks, global_blocks, streams * frames, device)
        if cfg.dim != cfg.heads * 64:
            raise ValueError(f"StreamingRunner: heads of 64 dims, got {cfg.dim} / {cfg.heads}")
        P = cfg.tokens_per_frame
        per_stream = -(-max_frames * P // block_size)
        self.frames, self.streams, self.max_frames, self.seen = frames, streams, max_frames, 0
        self.cache = PagedKVCache(len(global_blocks), streams * per_stream, cfg.heads, 64, streams, max_frames * P,
                                  block_size, self.device)
        self.time_axis = time_axis
        if time_axis:
            # the global blocks' projection turns by nothing; rope_axes follows it
            self.cos, self.sin = torch.ones_like(self.cos), torch.zeros_like(self.sin)
            self.sections = (8, 12, 12)
            self.inv_freq = torch.cat([cfg.rope_base ** (-torch.arange(n, dtype=torch.float32) / n)
                                       for n in self.sections]).to(self.device)
            p = torch.arange(P) - cfg.patch_start
            patch = p >= 0
            grid = torch.stack([torch.where(patch, p // cfg.grid_w + 1, 0), torch.where(patch, p % cfg.grid_w + 1, 0)])
            time = torch.arange(frames).repeat_interleave(P)[None]
            self._pos = torch.cat([time, grid.repeat(1, frames)]).repeat(1, streams).to(torch.int32).to(self.device)
        self._plan = None
        self._layer = 0

    def _global_attention(self) -> None:
        cfg, ws, T = self.cfg, self.ws, self.T
        q = ws.q.view(T, cfg.heads, 64)
        k = ws.kv_local[:, :cfg.dim].unflatten(1, (cfg.heads, 64))
        v = ws.kv_local[:, cfg.dim:].unflatten(1, (cfg.heads, 64))
        if self.time_axis:
            rope_axes(q, k, self._now, self.inv_freq, self.sections, layout="split", q_out=q, k_out=k)
        P = cfg.tokens_per_frame
        self.cache.append(self._layer, k, v, self._plan)
        self.cache.attend(self._layer, q, self._plan, self.frames * P, (self.seen + self.frames) * P, causal_chunk=P,
                          out=ws.attn.view(T, cfg.heads, 64))
        self._layer += 1

    def step(self, tokens: torch.Tensor, keep: tuple[int, ...] = ()) -> dict:
        """The next ``frames`` frames of every stream, tokens ``[streams * frames, P, C]`` fp16 (modified in place);
        returns :meth:`AggregatorRunner.forward`'s outputs for them."""
        if self.seen + self.frames > self.max_frames:
            raise ValueError(f"StreamingRunner: the cache holds {self.max_frames} frames, {self.seen} are in it")
        new = self.frames * self.cfg.tokens_per_frame
        self._plan = self.cache.plan(self.cache.lens + new, self.streams * new)
        self._layer = 0
        if self.time_axis:
            self._now = self._pos.clone()
            self._now[0] += self.seen
        outs = self.forward(tokens, keep)
        self.cache.commit(self._plan)
        self.seen += self.frames
        return outs

    def reset(self) -> None:
        """Ends every stream: its blocks go back to the pool."""
        self.cache.commit(self.cache.plan(torch.zeros_like(self.cache.lens), 0))
        self.seen = 0


class StreamingAggregator(VGGTAggregator):
    """:class:`VGGTAggregator` over frames as they arrive: ``frames`` images per call, ``max_frames`` in all.

    Takes :class:`VGGTAggregator`'s arguments (the weights and configuration
    are the same) plus ``max_frames`` and ``time_axis``; one GPU, one stream."""

    def __init__(self, cfg, pe, agg_specials, frame_blocks, global_blocks, frames: int, device, max_frames: int,
                 time_axis: bool = False, img_hw=(518, 518)):
        self._stream_args = (max_frames, time_axis)
        super().__init__(cfg, pe, agg_specials, frame_blocks, global_blocks, frames, device, img_hw=img_hw)

    def _make_runner(self, cfg, frame_blocks, global_blocks, frames, device, group, world, rank):
        max_frames, time_axis = self._stream_args
        return StreamingRunner(cfg, frame_blocks, global_blocks, frames, max_frames, device, time_axis=time_axis)

    def forward(self, images: torch.Tensor, keep: tuple[int, ...] = ()) -> dict:
        """The next images [frames, 3, H, W] fp16; outputs of their tokens as in :meth:`VGGTAggregator.forward`."""
        return self.runner.step(self.embed(images, frame_offset=self.runner.seen), keep)


def main(argv=None) -> None:
    import argparse

    from .synthetic import random_block

    ap = argparse.ArgumentParser(description="time the streaming aggregator's block stack on random weights")
    ap.add_argument("--frames", type=int, default=32)
    ap.add_argument("--depth", type=int, default=4)
    ap.add_argument("--time-axis", action="store_true")
    a = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    cfg = AggConfig(depth=a.depth)
    gen = torch.Generator(device=dev).manual_seed(0)
    blocks = [[random_block(cfg, gen, dev) for _ in range(a.depth)] for _ in range(2)]
    run = StreamingRunner(cfg, *blocks, 1, a.frames, dev, time_axis=a.time_axis)
    tokens = torch.randn(1, cfg.tokens_per_frame, cfg.dim, generator=gen, device=dev).half()
    for _ in range(2):                   # the second pass over the frames is the timed one
        run.reset()
        times = []
        for _ in range(a.frames):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            x = tokens.clone()
            e[0].record()
            run.step(x)
            e[1].record()
            times.append(e)
        torch.cuda.synchronize()
    for i, (b, e) in enumerate(times):
        if i in (0, 1) or (i + 1) % max(1, a.frames // 8) == 0:
            print(f"frame {i + 1:4d}: {b.elapsed_time(e):.3f} ms")
    c = run.cache
    print(f"cache: {(c.k.numel() + c.v.numel() + 4 * (c.k_scale.numel() + c.v_scale.numel())) / 1e9:.3f} GB for "
          f"{a.frames} frames, {a.depth} layers")


if __name__ == "__main__":
    main()
