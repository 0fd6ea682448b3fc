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

A stream's first frames can also come all at once, each stream with its own
number of them (:meth:`StreamingRunner.prompt`): their global attention runs
over the projections' own K / V rows
(:func:`~qvggt_b200.kv_cache.prompt_attention`), and the cache takes the rows
for the steps that follow.

``sink_frames`` lets a stream go on when the cache is full: each global layer
then also gathers how much attention each cached key has got
(:func:`~qvggt_b200.kv_cache.key_weights`), and before a step that would not
fit, every layer and head drops the keys that got least, except those of the
first ``sink_frames`` frames and the last ``recent_frames`` of the newest step.

With ``time_axis`` q and k of the global blocks turn by (time, height, width)
positions (:func:`~qvggt_b200.kv_cache.rope_axes`) in place of the model's
(height, width); the frame blocks, whose tokens all have one time, keep the
model's.  A 518 x 518 frame's K/V of all 24 layers take 68 MB of the cache.

    python -m qvggt_b200.streaming [--frames N] [--depth D] [--time-axis] [--prompt N] [--hold N]

runs random weights over N frames (the first ``--prompt`` of them at once, at
most ``--hold`` of them in the cache) and prints the time of each step.
"""
from __future__ import annotations

import copy

import torch

from .aggregator import AggConfig, AggregatorRunner, VGGTAggregator, Workspace
from .kv_cache import PagedKVCache, prompt_attention, rope_axes


class StreamingRunner(AggregatorRunner):
    """:class:`AggregatorRunner` whose global blocks read a cache of the earlier frames.

    ``streams`` independent sequences advance together, ``frames`` frames of
    each per step; the cache holds ``max_frames`` frames of each.  With
    ``sink_frames`` (0 or more) a stream that has filled it drops the tokens
    that got least attention, never those of its first ``sink_frames`` frames
    nor of the last ``recent_frames`` (at most ``frames``: tokens of earlier
    steps have no fixed place in the cache); ``weight_decay`` (0 to 1) ages what
    they have got, once a step.  One GPU."""

    def __init__(self, cfg: AggConfig, frame_blocks, global_blocks, frames: int, max_frames: int, device,
                 streams: int = 1, time_axis: bool = False, block_size: int = 64, sink_frames: int | None = None,
                 recent_frames: int = 0, weight_decay: float = 1.0):
        super().__init__(cfg, frame_blocks, global_blocks, streams * frames, device)
        if cfg.dim != cfg.heads * 64:
            raise ValueError(f"StreamingRunner: heads of 64 dims, got {cfg.dim} / {cfg.heads}")
        P = cfg.tokens_per_frame
        per_stream = -(-max_frames * P // block_size)
        if sink_frames is not None:
            if frames > max_frames or min(sink_frames, recent_frames) < 0 or sink_frames + recent_frames > max_frames - frames:
                raise ValueError(f"StreamingRunner: {sink_frames} + {recent_frames} frames that stay and {frames} new ones "
                                 f"do not fit {max_frames}")
            if recent_frames > frames:
                raise ValueError(f"StreamingRunner: recent_frames {recent_frames} must not pass a step's {frames}: the "
                                 f"tokens of earlier steps have no fixed place in the cache")
            if not 0 <= weight_decay <= 1:
                raise ValueError(f"StreamingRunner: weight_decay must be 0 to 1, got {weight_decay}")
        self.frames, self.streams, self.max_frames = frames, streams, max_frames
        self.sink_frames, self.recent_frames, self.weight_decay = sink_frames, recent_frames, weight_decay
        self._seen, self._held = [0] * streams, [0] * streams        # frames of each stream: so far, in the cache
        self.cache = PagedKVCache(len(global_blocks), streams * per_stream, cfg.heads, 64, streams, max_frames * P,
                                  block_size, self.device, weights=sink_frames is not None)
        self._lse = self._new_lse(self.T)
        self._cu = None                  # a prompt's running sums of the streams' tokens
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
            self._grid = grid.to(torch.int32).to(self.device)
            self._pos = self._positions([frames] * streams)
        self._plan = None
        self._layer = 0

    @property
    def seen(self) -> int:
        """Frames so far, of the stream that has most.  Assigned, it holds for every stream, and for what the cache holds."""
        return max(self._seen)

    @seen.setter
    def seen(self, frames: int) -> None:
        self._seen = [frames] * self.streams
        self._held = [min(frames, self.max_frames)] * self.streams

    def _positions(self, counts):
        """(time, height, width) of the tokens of `counts` frames of each stream, times from 0 on."""
        time = torch.cat([torch.arange(n, dtype=torch.int32) for n in counts]).to(self.device)
        time = time.repeat_interleave(self.cfg.tokens_per_frame)[None]
        return torch.cat([time, self._grid.repeat(1, sum(counts))])

    def _new_lse(self, tokens):
        if self.sink_frames is None:
            return None
        return torch.empty(self.cfg.heads, tokens, dtype=torch.float32, device=self.device)

    def _global_attention(self) -> None:
        cfg, ws, T = self.cfg, self.ws, self.T
        q = ws.q.view(T, cfg.heads, 64)
        k = ws.kv_local[:, :cfg.dim].unflatten(1, (cfg.heads, 64))
        v = ws.kv_local[:, cfg.dim:].unflatten(1, (cfg.heads, 64))
        if self.time_axis:
            rope_axes(q, k, self._now, self.inv_freq, self.sections, layout="split", q_out=q, k_out=k)
        P, out = cfg.tokens_per_frame, ws.attn.view(T, cfg.heads, 64)
        self.cache.append(self._layer, k, v, self._plan)
        if self._cu is not None:
            prompt_attention(q, k, v, self._cu, self._max_q, causal_chunk=P, out=out, lse=self._lse)
        else:
            self.cache.attend(self._layer, q, self._plan, self._max_q, self._max_kv, causal_chunk=P, out=out, lse=self._lse)
        if self._lse is not None:
            self.cache.weigh(self._layer, q, self._plan, self._lse, self._max_q, self._max_kv, causal_chunk=P,
                             decay=self.weight_decay)
        self._layer += 1

    def _make_room(self) -> None:
        """Room for the next step's frames, by eviction where the streams may evict."""
        most = self.max_frames - self.frames
        full = [n > most for n in self._held]
        if not any(full):
            return
        if self.sink_frames is None:
            raise ValueError(f"StreamingRunner: the cache holds {self.max_frames} frames, {max(self._held)} are in it")
        P = self.cfg.tokens_per_frame
        keep = [min(n, most) * P for n in self._held]
        moves = max(min(k, n * P - k) for k, n in zip(keep, self._held))
        self.cache.evict(torch.tensor(keep, dtype=torch.int32).to(self.device), moves, self.sink_frames * P,
                         self.recent_frames * P)
        self._held = [min(n, most) for n in self._held]

    def step(self, tokens: torch.Tensor, keep: tuple[int, ...] = ()) -> dict:
        """The next ``frames`` frames of every stream, tokens ``[streams * frames, P, C]`` fp16 (modified in place);
        returns :meth:`AggregatorRunner.forward`'s outputs for them."""
        self._make_room()
        P = self.cfg.tokens_per_frame
        new = self.frames * P
        self._plan = self.cache.plan(self.cache.lens + new, self.streams * new)
        self._layer, self._max_q, self._max_kv = 0, new, (max(self._held) + self.frames) * P
        if self.time_axis:
            self._now = self._pos.clone()
            if min(self._seen) == max(self._seen):
                self._now[0] += self._seen[0]
            else:
                self._now[0] += torch.tensor(self._seen, dtype=torch.int32).repeat_interleave(new).to(self.device)
        outs = self.forward(tokens, keep)
        self.cache.commit(self._plan)
        self._seen = [n + self.frames for n in self._seen]
        self._held = [n + self.frames for n in self._held]
        return outs

    def prompt(self, tokens: torch.Tensor, counts, keep: tuple[int, ...] = ()) -> dict:
        """The first ``counts[s]`` frames of each stream s at once (0 to ``max_frames``), tokens ``[sum(counts), P, C]``
        fp16, stream after stream (modified in place); returns :meth:`AggregatorRunner.forward`'s outputs for them.
        Their global attention reads their K / V rows as they are, not the cache's 8 bits (and what the cache's keys gather
        is by its log-sum-exps: see :func:`~qvggt_b200.kv_cache.key_weights`)."""
        P, counts = self.cfg.tokens_per_frame, [int(n) for n in counts]
        if len(counts) != self.streams or min(counts) < 0 or max(counts) > self.max_frames or max(counts) == 0:
            raise ValueError(f"StreamingRunner: {counts} frames for {self.streams} streams of up to {self.max_frames}")
        if self.seen:
            raise ValueError(f"StreamingRunner: a prompt comes first, {self.seen} frames were before it")
        total = sum(counts)
        if tokens.shape[0] != total:
            raise ValueError(f"StreamingRunner: {tokens.shape[0]} frames of tokens, the streams take {total}")
        lens = torch.tensor([n * P for n in counts], dtype=torch.int32).to(self.device)
        # the same runner over other activations: these frames' own workspace
        run = copy.copy(self)
        run.S_local, run.T = total, total * P
        run.ws = Workspace(run.T, run.T, self.cfg, self.device, self.w8a8)
        run._lse = self._new_lse(run.T)
        run._plan = plan = self.cache.plan(lens, run.T)
        run._cu, run._layer = plan.cu_new, 0
        run._max_q = run._max_kv = max(counts) * P
        if self.time_axis:
            run._now = self._positions(counts)
        outs = run.forward(tokens, keep)
        self.cache.commit(plan)
        self._seen, self._held = list(counts), list(counts)
        return outs

    def reset(self) -> None:
        """Ends every stream: its blocks go back to the pool."""
        self.cache.commit(self.cache.plan(torch.zeros_like(self.cache.lens), 0))
        self._seen, self._held = [0] * self.streams, [0] * self.streams


class StreamingAggregator(VGGTAggregator):
    """:class:`VGGTAggregator` over frames as they arrive: ``frames`` images per call, ``max_frames`` in the cache.

    Takes :class:`VGGTAggregator`'s arguments (the weights and configuration
    are the same) plus ``max_frames``, ``time_axis`` and, to go on when the cache
    is full, ``sink_frames``, ``recent_frames`` and ``weight_decay`` (see
    :class:`StreamingRunner`); one GPU, one stream."""

    def __init__(self, cfg, pe, agg_specials, frame_blocks, global_blocks, frames: int, device, max_frames: int,
                 time_axis: bool = False, img_hw=(518, 518), sink_frames: int | None = None, recent_frames: int = 0,
                 weight_decay: float = 1.0):
        self._stream_args = dict(time_axis=time_axis, sink_frames=sink_frames, recent_frames=recent_frames,
                                 weight_decay=weight_decay)
        self._max_frames = max_frames
        super().__init__(cfg, pe, agg_specials, frame_blocks, global_blocks, frames, device, img_hw=img_hw)

    def _make_runner(self, cfg, frame_blocks, global_blocks, frames, device, group, world, rank):
        return StreamingRunner(cfg, frame_blocks, global_blocks, frames, self._max_frames, device, **self._stream_args)

    def forward(self, images: torch.Tensor, keep: tuple[int, ...] = ()) -> dict:
        """The next images [frames, 3, H, W] fp16; outputs of their tokens as in :meth:`VGGTAggregator.forward`."""
        return self.runner.step(self.embed(images, frame_offset=self.runner.seen), keep)

    def prompt(self, images: torch.Tensor, keep: tuple[int, ...] = ()) -> dict:
        """The first images [n, 3, H, W] fp16 at once (n a multiple of ``frames``, the number the DINOv2 front takes at a
        time); outputs as in :meth:`forward` (see :meth:`StreamingRunner.prompt`)."""
        n, step = images.shape[0], self.S_local
        if n % step or not n:
            raise ValueError(f"StreamingAggregator: {n} images, the front takes {step} at a time")
        tokens = torch.empty(n, *self.tokens.shape[1:], dtype=self.tokens.dtype, device=self.tokens.device)
        for i in range(0, n, step):
            tokens[i:i + step] = self.embed(images[i:i + step], frame_offset=i)      # (one buffer for every call)
        return self.runner.prompt(tokens, [n], keep)


def main(argv=None) -> None:
    import argparse

    from .synthetic import random_block

    ap = argparse.ArgumentParser(description="time the streaming aggregator's block stack on random weights")
    ap.add_argument("--frames", type=int, default=32)
    ap.add_argument("--depth", type=int, default=4)
    ap.add_argument("--time-axis", action="store_true")
    ap.add_argument("--prompt", type=int, default=0, help="frames that come at once, first")
    ap.add_argument("--hold", type=int, default=0, help="frames the cache holds; then the least attended tokens go")
    a = ap.parse_args(argv)
    if not 0 <= a.prompt <= min(a.frames, a.hold or a.frames) or a.hold < 0 or a.hold == 1:
        ap.error("--prompt: at most --frames and --hold; --hold: 2 or more")
    dev = torch.device("cuda", torch.cuda.current_device())
    cfg = AggConfig(depth=a.depth)
    gen = torch.Generator(device=dev).manual_seed(0)
    blocks = [[random_block(cfg, gen, dev) for _ in range(a.depth)] for _ in range(2)]
    hold = a.hold or a.frames
    run = StreamingRunner(cfg, *blocks, 1, hold, dev, time_axis=a.time_axis, sink_frames=1 if a.hold else None)
    tokens = torch.randn(1, cfg.tokens_per_frame, cfg.dim, generator=gen, device=dev).half()
    for _ in range(2):                   # the second pass over the frames is the timed one
        run.reset()
        times = []
        while run.seen < a.frames:
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            first = a.prompt if not run.seen else 0
            x = tokens.repeat(first or 1, 1, 1)
            e[0].record()
            run.prompt(x, [first]) if first else run.step(x)
            e[1].record()
            times.append((run.seen, *e))
        torch.cuda.synchronize()
    for i, (n, b, e) in enumerate(times):
        if i in (0, 1) or n % max(1, a.frames // 8) == 0:
            print(f"to frame {n:4d}: {b.elapsed_time(e):.3f} ms")
    c = run.cache
    print(f"cache: {(c.k.numel() + c.v.numel() + 4 * (c.k_scale.numel() + c.v_scale.numel())) / 1e9:.3f} GB for "
          f"{hold} frames, {a.depth} layers")


if __name__ == "__main__":
    main()
