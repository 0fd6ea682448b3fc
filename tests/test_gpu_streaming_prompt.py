"""GPU: streams whose first frames come at once, and streams that go on when their cache is full."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok
from oracle import kv_evict as oe
from tests.test_gpu_streaming import _blocks, _config, _dense

pytestmark = pytest.mark.gpu


def _tokens(cfg, frames, seed):
    return torch.randn(frames, cfg.tokens_per_frame, cfg.dim, generator=torch.Generator().manual_seed(seed)).half().cuda()


@pytest.mark.parametrize("time_axis", [False, True])
def test_prompt_of_ragged_streams_matches_all_at_once(time_axis):
    """Each stream's first frames against dense frame-causal attention in 64 bits.  The attention rounds its weights and
    its output once each (2^-11), the residual is rounded to fp16 four times: the updates, some 1e-2 of the tokens, are
    off by about 2^-12 / 1e-2 of theirs and twice that between two runs, 5e-2 is double that."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = _blocks(cfg, dev)
    counts = [3, 1, 0, 5]
    x = _tokens(cfg, sum(counts), 1)
    run = StreamingRunner(cfg, *blocks, 1, 5, dev, streams=4, time_axis=time_axis, block_size=32)
    for _ in range(2):                   # again after a reset
        got = run.prompt(x.clone(), counts)[-1][1].view(sum(counts), cfg.tokens_per_frame, -1)
        at = 0
        for n in counts:
            if n:
                rows = slice(at, at + n)
                want = _dense(cfg, blocks, n, dev, run).forward(x[rows].clone())[-1][1].view(n, cfg.tokens_per_frame, -1)
                dx, dw = (t.double() - x[rows].double() for t in (got[rows], want))
                assert (dx - dw).norm() <= 5e-2 * dw.norm()
            at += n
        assert run.cache.lens.tolist() == [n * cfg.tokens_per_frame for n in counts] and run.seen == 5
        with pytest.raises(ValueError, match="comes first"):
            run.prompt(x.clone(), counts)
        run.reset()
    assert sorted(run.cache.free_ring.tolist()) == list(range(run.cache.free_ring.numel()))


@pytest.mark.parametrize("time_axis", [False, True])
def test_steps_after_a_prompt_match_all_at_once(time_axis):
    """Prompts of two lengths, then a step of both streams: the step's frames see the prompt's through the cache (the
    bound is the cache's, as for frames one after another: 3e-2 of the updates)."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = _blocks(cfg, dev)
    P = cfg.tokens_per_frame
    x = [_tokens(cfg, 6, s) for s in (3, 4)]
    counts = [4, 2]
    run = StreamingRunner(cfg, *blocks, 2, 6, dev, streams=2, time_axis=time_axis, block_size=32)
    run.prompt(torch.cat([t[:n] for t, n in zip(x, counts)]).clone(), counts)
    got = run.step(torch.cat([t[n:n + 2] for t, n in zip(x, counts)]).clone())[-1][1].view(2, 2, P, -1)
    for s, n in enumerate(counts):
        want = _dense(cfg, blocks, n + 2, dev, run).forward(x[s][:n + 2].clone())[-1][1].view(n + 2, P, -1)[n:]
        dx, dw = (t.double() - x[s][n:n + 2].double() for t in (got[s], want))
        assert (dx - dw).norm() <= 3e-2 * dw.norm()


@pytest.mark.parametrize("kind", ["w4", "w8"])
def test_prompt_and_step_of_either_weight_format(kind):
    """int8 blocks take the same path: their first frames at once are their first frames one after another, but for the
    cache's 8 bits (3e-2 of the updates) and the activations' (a code more or less: 1e-2)."""
    from qvggt_b200.streaming import StreamingRunner
    from tests.test_gpu_streaming_frames import _blocks as blocks_of
    dev = torch.device("cuda", 0)
    cfg = _config()
    blocks = blocks_of(cfg, dev, kind)
    x = _tokens(cfg, 3, 9)
    outs = []
    for first in (0, 2):
        run = StreamingRunner(cfg, *blocks, 1, 3, dev, block_size=32, sink_frames=0)
        got = [run.prompt(x[:2].clone(), [2])[-1][1]] if first else []
        got += [run.step(x[i:i + 1].clone())[-1][1] for i in range(first, 3)]
        outs.append(torch.cat([t.view(-1, cfg.dim) for t in got]).double() - x.view(-1, cfg.dim).double())
    assert (outs[0] - outs[1]).norm() <= 4e-2 * outs[0].norm()


def _snapshot(cache):
    return [t.cpu().numpy().copy() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weights,
                                             cache.block_tables, cache.lens)]


@pytest.mark.parametrize("per_step,hold,sink,recent", [(1, 3, 1, 1), (2, 5, 0, 1), (1, 2, 0, 0)])
def test_streams_go_on_when_the_cache_is_full(per_step, hold, sink, recent):
    """Two streams of 8 frames through a cache of a few.  Each step: the weights grow by one for each query row and head
    (within the attention's error of 2e-4), and what makes room is the restatement's choice and move, bit for bit."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    P, H = cfg.tokens_per_frame, cfg.heads
    run = StreamingRunner(cfg, *_blocks(cfg, dev), per_step, hold, dev, streams=2, block_size=32, sink_frames=sink,
                          recent_frames=recent)
    evicted = 0
    for i in range(0, 8, per_step):
        before = _snapshot(run.cache)
        run._make_room()
        after = _snapshot(run.cache)
        lens, keep = before[6].tolist(), [min(n, (hold - per_step) * P) for n in before[6].tolist()]
        assert after[6].tolist() == keep
        moves = max(1, max(min(k, n - k) for n, k in zip(lens, keep)))
        plan = oe.evict_plan(before[4], before[5], lens, keep, sink * P, recent * P, moves)
        for codes, scales in ((before[0], before[2]), (before[1], before[3])):
            oe.kv_evict(codes, scales, before[5], *plan)
        oe.evict_weights(before[4], before[5], *plan)
        for a, b in zip(before[:5], after[:5]):
            assert (a == b).all()
        evicted += sum(lens) - sum(keep)
        # what is held in the pool: each block once
        used = [int(b) for row, n in zip(after[5], keep) for b in row[:-(-n // 32)]]
        first, last = run.cache.free_range.tolist()
        ring = run.cache.free_ring.tolist()
        free = [ring[j % len(ring)] for j in range(first, last)]
        assert sorted(used + free) == list(range(len(ring)))

        def gathered():
            total = torch.zeros(cfg.depth, dtype=torch.float64)
            for b, n in enumerate(run.cache.lens.tolist()):
                j = torch.arange(n, device=dev)
                total += run.cache.weights[:, run.cache.block_tables[b, j // 32].long(), :, j % 32].double().sum((0, 2)).cpu()
            return total

        held = gathered()
        out = run.step(_tokens(cfg, 2 * per_step, 100 + i))[-1][1]
        assert torch.isfinite(out).all()
        rows = 2 * per_step * P * H
        assert ((gathered() - held) - rows).abs().max() <= 3e-4 * rows
    assert evicted > 0 and run.seen == 8 and run.cache.lens.tolist() == [hold * P] * 2
    run.reset()
    assert run.cache.lens.tolist() == [0, 0]


def test_weights_after_a_prompt():
    """A prompt's log-sum-exps are over its own fp16 keys, its weights over the cache's 8-bit ones: the weights are the
    operator's for these inputs, and a row hands out 1 times at most e^d, at least e^-d, where d is what rounding the keys may
    change a score by: scale |q|_1 times half a step (and the log-sum-exp's error of 2e-4)."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    P, H, counts = cfg.tokens_per_frame, cfg.heads, [3, 0, 1]
    run = StreamingRunner(cfg, *_blocks(cfg, dev), 1, 4, dev, streams=3, block_size=32, sink_frames=0)
    cache, weigh, calls = run.cache, run.cache.weigh, []

    def kept(layer, q, plan, lse, *args, **kwargs):
        calls.append((layer, q.clone(), lse.clone()))
        weigh(layer, q, plan, lse, *args, **kwargs)

    cache.weigh = kept
    run.prompt(_tokens(cfg, 4, 11), counts)
    assert [c[0] for c in calls] == list(range(cfg.depth))
    cu = torch.tensor([0, 3 * P, 3 * P, 4 * P])
    for layer, q, lse in calls:
        want, err = oe.key_weights(q, cache.k[layer], cache.k_scale[layer], cache.block_tables, cu, cache.lens, lse,
                                   torch.zeros_like(cache.weights[layer]), P, None, [0, 0, 0])
        assert ((cache.weights[layer].double() - want).abs() <= err).all()
        for b, n in enumerate(counts):
            ids = cache.block_tables[b, :-(-n * P // 32)].long()
            got = cache.weights[layer, ids].double().sum((0, 2))             # a block is one stream's
            rows = q[int(cu[b]):int(cu[b + 1])].double().abs().sum(-1)       # [tokens, heads]
            half = 0.5 * cache.k_scale[layer, ids].double().amax(0) if n else torch.zeros(H, device=dev).double()
            d = rows * half / 8 + 2e-4
            assert (got <= d.exp().sum(0)).all() and (got >= (-d).exp().sum(0)).all()
            assert n == 0 or float(d.max()) < 0.5


def test_evicting_what_nobody_looks_at_changes_little():
    """A third of the keys point away from every query; a cache that drops just as many drops those, and the attention
    over what is left is the attention over all (the lost weights, 40 keys of e^-16 each, and one rounding of moved rows)."""
    from qvggt_b200 import kv_cache
    H, D, bs, n = 2, 64, 32, 120
    g = torch.Generator(device="cuda").manual_seed(0)
    cache = kv_cache.PagedKVCache(1, 6, H, D, 1, n + 1, bs, weights=True)
    q = 0.3 * torch.randn(n, H, D, generator=g, device="cuda")
    q[..., 0] = 4
    k, v = (torch.randn(n, H, D, generator=g, device="cuda") for _ in range(2))
    dead = torch.randperm(n, generator=g, device="cuda")[:40]
    k[..., 0] = 4
    k[dead, :, 0] = -30
    q, k, v = q.half(), k.half(), v.half()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    plan = cache.plan(lens, n)
    cache.append(0, k, v, plan)
    lse = torch.empty(H, n, device="cuda")
    want = cache.attend(0, q, plan, n, n, out=None, lse=lse)
    cache.weigh(0, q, plan, lse, n, n)
    cache.commit(plan)
    moved = cache.evict(lens - 40, 40)
    gone = {int(j) for j in dead}
    for h in range(H):
        m = int(moved.counts[0, 0, h])
        kept_late = {int(j) for j in moved.src[0, 0, h, :m]}
        assert {int(j) for j in moved.dst[0, 0, h, :m]} == {j for j in gone if j < n - 40}
        assert kept_late == {j for j in range(n - 40, n) if j not in gone}
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = kv_cache.cached_attention(q, cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0], cache.block_tables, cu,
                                    cache.lens, n, n - 40)
    assert cache.lens.item() == n - 40
    # moved rows: half a step of the receiving block's scale, K's times |q| as a score's error, V's as the output's
    step = 0.5 * max(float(cache.k_scale.max()), float(cache.v_scale.max()))
    score = step * float(q.float().abs().sum(-1).max()) / 8
    assert (got.float() - want.float()).abs().max() <= 2 * score * float(v.abs().max()) + step + 40 * math.exp(-16) + 2e-3


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,bs,ql", [(64, 32, 3), (64, 64, 90), (128, 128, 3), (128, 32, 90)])
def test_attention_over_what_an_eviction_leaves(dtype, D, bs, ql):
    """Append, attend, weigh and evict.  Each place then holds its survivor, to half a step of the block's scale (1e-5 for the
    step itself), and new queries get the attention in 64 bits over the codes, scales and tables that are there, within the
    attention's own bound, which is far under its results."""
    from qvggt_b200 import kv_cache
    from tests.test_gpu_kv_cache import _check_attention
    H, hq, lens, keep = 2, 4, [300, 0, 135], [170, 5, 130]
    g = torch.Generator(device="cuda").manual_seed(D + ql)
    cache = kv_cache.PagedKVCache(1, 20, H, D, 3, 400, bs, weights=True)
    T, most = sum(lens), max(lens)
    q = torch.randn(T, hq, D, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(T, H, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    plan = cache.plan(ints(lens), T)
    cache.append(0, k, v, plan)
    lse = torch.empty(hq, T, device="cuda")
    cache.attend(0, q, plan, most, most, lse=lse)          # (no mask: with one the first tokens gather most, and stay)
    cache.weigh(0, q, plan, lse, most, most)
    cache.commit(plan)
    state = lambda: [t[0].clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    before, table = state(), cache.block_tables.clone()
    moved = cache.evict(ints(keep), 130, sink=3)
    assert cache.lens.tolist() == [170, 0, 130] and int(moved.counts.min(-1).values[0, 0]) > 20
    after = state()
    for r, n in ((0, 170), (2, 130)):
        for h in range(H):
            here = torch.arange(n, device="cuda")
            at, m = here.clone(), int(moved.counts[0, r, h])
            at[moved.dst[0, r, h, :m].long()] = moved.src[0, r, h, :m].long()
            old, new = table[r, at // bs].long(), cache.block_tables[r, here // bs].long()
            for side in range(2):
                x = before[side][old, h, at % bs].double() * before[2 + side][old, h, None].double()
                y = after[side][new, h, here % bs].double() * after[2 + side][new, h, None].double()
                assert ((x - y).abs() <= (0.5 + 1e-5) * after[2 + side][new, h, None].double()).all()
    x = torch.randn(2 * ql, hq, D, generator=g, device="cuda").to(dtype)
    cu, lse = ints([0, ql, ql, 2 * ql]), torch.empty(hq, 2 * ql, device="cuda")
    got = kv_cache.cached_attention(x, *after, cache.block_tables, cu, cache.lens, ql, 170, 0, lse=lse)
    ref = ok.cached_attention(x, *after, cache.block_tables, cu, cache.lens, 0)
    _check_attention(got, lse, ref, dtype, float(after[3].max() * 128), 170)
    assert ref[0].abs().max() > 0.2      # (the bound is some 2e-3, bf16's output rounding beside it)


def test_streaming_aggregator_prompt_is_the_models():
    """One frame at once, nothing cached: the model itself; then the next frame arrives."""
    from qvggt_b200.aggregator import AggConfig
    from qvggt_b200.streaming import StreamingAggregator
    from qvggt_b200.synthetic import random_vggt_aggregator
    dev = torch.device("cuda", 0)
    agg = random_vggt_aggregator(AggConfig(depth=1), 4, dev, 1, pe_depth=1)
    parts = (agg.cfg, agg.pe, agg.agg_specials, agg.runner.frame_blocks, agg.runner.global_blocks)
    images = torch.rand(2, 3, 518, 518, generator=torch.Generator().manual_seed(3)).half().to(dev)
    want = agg.forward(images[:1])[-1][1].double()
    stream = StreamingAggregator(*parts, 1, dev, max_frames=2, sink_frames=0, recent_frames=1)
    got = stream.prompt(images[:1])[-1][1].double()
    assert (got - want).norm() <= 1e-3 * want.norm()
    for _ in range(2):                   # the second of these makes room first
        assert torch.isfinite(stream.forward(images[1:])[-1][1]).all()
    assert stream.runner.seen == 3 and stream.runner.cache.lens.item() == 2 * 1374
    stream.runner.reset()
    both = stream.prompt(images)[-1][1]
    assert both.shape[0] == 2 * 1374 and torch.isfinite(both).all()
    assert (both[:1374].double() - got).norm() <= 1e-3 * got.norm()      # the first frame does not see the second


@pytest.mark.parametrize("per_step,hold,sink,recent,decay,match", [
    (1, 4, 0, 2, 1.0, "recent_frames"), (1, 4, -1, 1, 1.0, "fit"), (1, 4, 2, -1, 1.0, "fit"), (2, 5, 2, 2, 1.0, "fit"),
    (3, 2, 0, 0, 1.0, "fit"), (1, 4, 1, 1, 1.5, "decay"), (1, 4, 1, 1, float("nan"), "decay")])
def test_windows_that_cannot_be_kept_are_refused(per_step, hold, sink, recent, decay, match):
    """A recent window that reaches back past a step would pin what stands there, not the newest."""
    from qvggt_b200.streaming import StreamingRunner
    dev = torch.device("cuda", 0)
    cfg = _config()
    with pytest.raises(ValueError, match=match):
        StreamingRunner(cfg, *_blocks(cfg, dev), per_step, hold, dev, block_size=32, sink_frames=sink, recent_frames=recent,
                        weight_decay=decay)


def test_command_line(capsys):
    from qvggt_b200 import streaming
    streaming.main(["--frames", "5", "--depth", "1", "--prompt", "2", "--hold", "3", "--time-axis"])
    out = capsys.readouterr().out
    assert "to frame    2" in out and "to frame    5" in out and "3 frames, 1 layers" in out
