"""CPU: the restatements of the prompt and eviction operators against independent forms, and refusals that need no GPU."""
import math
import os
import re

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok
from oracle import kv_evict as oe
from qvggt_b200 import kv_cache as kc


def test_prompt_attention_is_masked_softmax():
    g = torch.Generator().manual_seed(0)
    lens, hq, hk, D, chunk = [7, 1, 0, 12], 4, 2, 8, 3
    T = sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g) for h in (hq, hk, hk))
    cu = [0, 7, 8, 8, 20]
    out, lse, mag = oe.prompt_attention(q, k, v, cu, chunk)
    seq = torch.tensor([b for b, n in enumerate(lens) for _ in range(n)])
    pos = torch.cat([torch.arange(n) for n in lens])
    seen = (seq[:, None] == seq[None]) & (pos[None] // chunk <= pos[:, None] // chunk)
    for h in range(hq):
        s = (q[:, h].double() @ k[:, h // 2].double().t()) / math.sqrt(D)
        w = s.masked_fill(~seen, -math.inf).softmax(-1)
        assert torch.allclose(out[:, h], w @ v[:, h // 2].double(), atol=1e-12)
        assert torch.allclose(mag[:, h], w @ v[:, h // 2].double().abs(), atol=1e-12)
        assert torch.allclose(lse[h], s.masked_fill(~seen, -math.inf).logsumexp(-1), atol=1e-12)
    v2 = v.clone()
    v2[5] = math.nan                     # seen by tokens 3 to 6 of the first sequence alone
    assert torch.isfinite(oe.prompt_attention(q, k, v2, cu, chunk)[0][[0, 1, 2] + list(range(7, 20))]).all()


@pytest.mark.parametrize("chunk", [0, 1, 4])
def test_key_weights_are_the_attentions_columns(chunk):
    """The sum over rows of the softmax that cached_attention's restatement computes, key by key; the rows hand out 1 each."""
    g = torch.Generator().manual_seed(1)
    ql, kl, hq, hk, D, bs = [3, 5, 0], [9, 70, 4], 4, 2, 8, 32
    nb = 5
    codes = torch.randint(-127, 128, (nb, hk, bs, D), generator=g, dtype=torch.int8)
    ks = torch.rand(nb, hk, generator=g) / 60
    table = torch.tensor([[4, -1, -1], [0, 2, 1], [3, -1, -1]], dtype=torch.int32)
    q = torch.randn(8, hq, D, generator=g).half()
    cu, lens = torch.tensor([0, 3, 8, 8]), torch.tensor(kl)
    lse = ok.cached_attention(q, codes, codes, ks, ks, table, cu, lens, chunk)[1]
    w = torch.rand(nb, hk, bs, generator=g)
    fresh = [6, 65, 4]
    got, err = oe.key_weights(q, codes, ks, table, cu, lens, lse, w, chunk, None, fresh, 0.5)
    want = w.double().clone()
    rows = 0
    for b, n in enumerate(kl):
        at = [(int(table[b, j // bs]), j % bs) for j in range(n)]
        for h in range(hk):
            total = torch.zeros(n, dtype=torch.float64)
            k = torch.stack([codes[x, h, y].double() * ks[x, h].double() for x, y in at])
            for i in range(ql[b]):
                for gq in (2 * h, 2 * h + 1):
                    lim = ok.key_limit(i, ql[b], n, chunk)
                    if lim:
                        total[:lim] += torch.softmax(k[:lim] @ q[int(cu[b]) + i, gq].double() / math.sqrt(D), 0)
                        rows += 1
            for j, (x, y) in enumerate(at):
                want[x, h, y] = total[j] + (0.5 * w[x, h, y].double() if j < fresh[b] else 0)
    assert torch.allclose(got, want, atol=1e-12) and (err >= 0).all()
    again = oe.key_weights(q, codes, ks, table, cu, lens, lse, torch.zeros_like(w), chunk)[0]
    assert abs(float(again.sum()) - rows) < 1e-9


def test_evict_plan_against_a_sort():
    rng = np.random.default_rng(0)
    layers, H, bs = 2, 3, 32
    lens, keep, sink, recent = [100, 33, 5, 64], [60, 33, 1, 20], 7, 4
    table = np.array([[5, 1, 7, 2], [0, 3, -1, -1], [4, -1, -1, -1], [8, 6, -1, -1]])
    w = rng.integers(0, 6, (layers, 9, H, bs)).astype(np.float32)
    w[rng.random(w.shape) < 0.1] = math.nan
    w[rng.random(w.shape) < 0.1] = math.inf
    src, dst, counts = oe.evict_plan(w, table, lens, keep, sink, recent, 40)
    for layer in range(layers):
        for b, (n, k) in enumerate(zip(lens, keep)):
            for h in range(H):
                m = counts[layer, b, h]
                assert (src[layer, b, h, m:] == -1).all() and (dst[layer, b, h, m:] == -1).all()
                s, d = src[layer, b, h, :m], dst[layer, b, h, :m]
                assert (np.diff(s) > 0).all() and (np.diff(d) > 0).all() and (d < k).all() and (s >= k).all() and (s < n).all()
                stays = np.sort(np.concatenate([np.setdiff1d(np.arange(k), d), s]))
                assert len(stays) == min(k, n)
                first, last = min(sink, k), min(recent, k - min(sink, k))
                if k >= n:
                    assert m == 0
                    continue
                assert np.isin(np.arange(first), stays).all() and np.isin(np.arange(n - last, n), stays).all()
                x = np.array([w[layer, table[b][j // bs], h, j % bs] for j in range(n)], np.float64)
                x = np.where(np.isnan(x), -1e39, np.minimum(x, 3.4028235e38))
                free = np.arange(first, n - last)
                best = free[np.lexsort((free, -x[free]))][:k - first - last]
                assert (np.sort(best) == stays[np.isin(stays, free)]).all()


def test_kv_evict_keeps_values_to_half_a_step():
    """Moved rows are off by half a step of the receiving block's scale, rows whose block's scale grew too, others not at
    all; the evicted rows' places hold the survivors."""
    rng = np.random.default_rng(1)
    lens, keep, bs, H, D = [90, 40], [50, 21], 32, 2, 8
    table = np.array([[3, 0, 5], [1, 4, -1]])
    codes = rng.integers(-127, 128, (1, 6, H, bs, D)).astype(np.int8)
    scales = np.exp(rng.normal(-4, 1, (1, 6, H))).astype(np.float32)
    w = rng.random((1, 6, H, bs)).astype(np.float32)
    plan = oe.evict_plan(w, table, lens, keep, 0, 0, 40)
    new_c, new_s, new_w = codes.copy(), scales.copy(), w.copy()
    oe.kv_evict(new_c, new_s, table, *plan)
    oe.evict_weights(new_w, table, *plan)
    assert (new_s >= scales).all()
    value = lambda c, s, b, h, j: c[0, table[b][j // bs], h, j % bs].astype(np.float64) * s[0, table[b][j // bs], h]
    for b in range(2):
        for h in range(H):
            m = plan[2][0, b, h]
            src, dst = plan[0][0, b, h, :m].tolist(), plan[1][0, b, h, :m].tolist()
            for j in range(keep[b]):
                old = src[dst.index(j)] if j in dst else j
                step = new_s[0, table[b][j // bs], h]
                off = np.abs(value(new_c, new_s, b, h, j) - value(codes, scales, b, h, old)).max()
                grown = step != scales[0, table[b][j // bs], h]
                assert off <= (0.5 * step * (1 + 1e-5) if j in dst or grown else 0)
                assert new_w[0, table[b][j // bs], h, j % bs] == w[0, table[b][old // bs], h, old % bs]


def test_packed_structures_match_the_header():
    hdr = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "qvggt_b200.h")).read()
    hdr = re.sub(r"/\*.*?\*/", "", hdr, flags=re.S)
    fields = {}
    for body, name in re.findall(r"typedef struct \{(.*?)\} (qvggt_\w+);", hdr, flags=re.S):
        n = 0
        for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
            if decl.startswith("qvggt_kv_cache"):
                n += fields["qvggt_kv_cache"]
                continue
            assert "*" in decl or decl.startswith(("int64_t", "double")), decl
            n += sum(int(m.group(1)) if (m := re.search(r"\[(\d+)\]", item)) else 1 for item in decl.split(","))
        fields[name] = n
    for name, pack in [("key_weights", kc._WEIGHTS), ("evict_plan", kc._EVICT_PLAN), ("kv_evict", kc._EVICT),
                       ("prompt_attention", kc._PROMPT)]:
        assert fields[f"qvggt_{name}_args"] * 8 == pack.__self__.size, name


def test_library_refuses_bad_arguments_without_a_gpu():
    """Argument checks come before any device call: code and message."""
    from qvggt_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()

    def refused(name, args, word, codes=(1, 2, 5)):
        assert getattr(lib, name)(args, None) in codes, name
        assert word in lib.qvggt_last_error(), lib.qvggt_last_error()

    n = _lib.i64(0)
    for args, word in [((8, 6, 4, 1, 8, 64), b"share"), ((8, 4, 4, 1, 8, 96), b"head_dim"), ((-1, 4, 4, 1, 8, 64), b"shape"),
                       ((8, 129, 1, 1, 8, 64), b"128 query heads")]:
        assert lib.qvggt_prompt_attention_scratch(*args, n) in (1, 2)
        assert word in lib.qvggt_last_error()

    def prompt(q=16, tok=64, scale=0.1, chunk=0, dtype=0, seqs=1, heads=1, cu=16):
        return kc._PROMPT(q, tok, 64, 16, 64, 64, 16, 64, 64, 16, 64, 64, 0, 4, heads, 1, 64, dtype, cu, seqs, 4, chunk, scale,
                          0, 0)
    for change, word in [(dict(scale=0.0), b"scale"), (dict(scale=math.nan), b"scale"), (dict(chunk=-1), b"chunk"),
                         (dict(dtype=2), b"dtype"), (dict(q=0), b"null"), (dict(cu=0), b"null"), (dict(q=8), b"aligned"),
                         (dict(tok=60), b"aligned"), (dict(tok=0), b"strides"), (dict(tok=-64), b"strides"),
                         (dict(seqs=-1), b"shape"), (dict(seqs=1 << 25), b"too many")]:
        refused("qvggt_prompt_attention", prompt(**change), word)
    assert lib.qvggt_prompt_attention(prompt(seqs=0, q=0), None) == 0

    def weigh(kc_=16, stride=2048, bs=32, d=64, q=16, dtype=0, lse=16, w=16, chunk=0, scale=0.1, decay=1.0, B=1):
        return kc._WEIGHTS(kc_, stride, 16, 4, 1, bs, d, q, 64, 64, 1, 1, dtype, lse, 16, 1, 16, 16, 0, B, 1, 32, chunk, w, w,
                           scale, decay)
    for change, word in [(dict(bs=48), b"block_size"), (dict(d=96), b"head_dim"), (dict(dtype=3), b"dtype"),
                         (dict(scale=-1.0), b"scale"), (dict(decay=-0.1), b"decay"), (dict(decay=math.nan), b"decay"),
                         (dict(chunk=-1), b"shape"), (dict(lse=0), b"null"), (dict(w=0), b"null"), (dict(kc_=8), b"aligned"),
                         (dict(stride=2040), b"aligned"), (dict(stride=1024), b"stride"), (dict(q=8), b"aligned")]:
        refused("qvggt_key_weights", weigh(**change), word)
    assert lib.qvggt_key_weights(weigh(B=0, w=0), None) == 0

    def plan(w=16, layers=1, bs=32, blocks=2, B=1, sink=0, moves=4, lens=16, length=0):
        return kc._EVICT_PLAN(w, layers, 4, 2, bs, 16, blocks, lens, 16, B, sink, 0, moves, length, 16, 16, 16)
    for change, word in [(dict(bs=33), b"block_size"), (dict(sink=-1), b"shape"), (dict(moves=-1), b"shape"),
                         (dict(length=-1), b"shape"), (dict(w=0), b"null"), (dict(lens=0), b"null"), (dict(w=8), b"aligned"),
                         (dict(blocks=1 << 30), b"2^30"), (dict(layers=1 << 20, B=1 << 24), b"too many")]:
        refused("qvggt_evict_plan", plan(**change), word)
    assert lib.qvggt_evict_plan(plan(B=0, w=0), None) == 0

    def move(stride=2 * 2048, layers=2, layer_stride=4 * 2 * 2048, keep=16, moves=4, blocks=2, bs=32):
        return kc._EVICT(16, 16, stride, 16, 16, 4, 2, bs, 64, layers, layer_stride, 0, 16, blocks, keep, 1, 16, 16, 16, moves)
    for change, word in [(dict(bs=48), b"block_size"), (dict(layer_stride=8), b"aligned"), (dict(layer_stride=2048), b"stride"),
                         (dict(keep=0), b"null"), (dict(layers=-1), b"shape"), (dict(blocks=1 << 28), b"2^30")]:
        refused("qvggt_kv_evict", move(**change), word)
    assert lib.qvggt_kv_evict(move(moves=0, keep=0), None) == 0


def test_python_refuses_cpu_tensors_and_bad_streams():
    q = torch.zeros(4, 2, 64).half()
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kc.prompt_attention(q, q, q, cu, 4)
    with pytest.raises(ValueError, match="CUDA"):
        kc.evict_plan(torch.zeros(1, 2, 2, 32), cu[None], cu[:1], cu[:1], 0, 0, 1)
    cache = kc.PagedKVCache(1, 4, 2, 64, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="without weights"):
        cache.evict(cu[:1], 1)
    with pytest.raises(ValueError, match="without weights"):
        cache.weigh(0, q, None, None, 1, 1)
    assert kc.PagedKVCache(2, 4, 2, 64, 1, 64, device="cpu", weights=True).weights.shape == (2, 4, 2, 64)

    from qvggt_b200.aggregator import AggConfig
    from qvggt_b200.streaming import StreamingRunner
    cfg = AggConfig(depth=0, tokens_per_frame=25, grid_w=5)
    for frames, hold, sink, recent in [(1, 3, 2, 1), (2, 1, 0, 0), (1, 2, -1, 0)]:
        with pytest.raises(ValueError, match="fit"):
            StreamingRunner(cfg, [], [], frames, hold, "cpu", sink_frames=sink, recent_frames=recent)
    run = StreamingRunner(cfg, [], [], 1, 3, "cpu", streams=2)
    x = torch.zeros(2, 25, cfg.dim).half()
    for counts, match in [([2], "streams"), ([2, -1], "streams"), ([4, 0], "streams"), ([0, 0], "streams"), ([2, 1], "tokens")]:
        with pytest.raises(ValueError, match=match):
            run.prompt(x, counts)


def test_the_frames_so_far_can_be_set():
    """`seen` is read and assigned, as by a program that restores or clears the cache itself; it counts for the room left."""
    from qvggt_b200.aggregator import AggConfig
    from qvggt_b200.streaming import StreamingRunner
    cfg = AggConfig(depth=0, tokens_per_frame=25, grid_w=5)
    run = StreamingRunner(cfg, [], [], 1, 3, "cpu", streams=2)
    assert run.seen == 0
    run.seen = 3
    assert run.seen == 3
    x = torch.zeros(2, 25, cfg.dim).half()
    with pytest.raises(ValueError, match="3 are in it"):
        run.step(x)
    with pytest.raises(ValueError, match="3 frames were before it"):
        run.prompt(x, [1, 1])
    run.seen = 0
    assert run.seen == 0
    run = StreamingRunner(cfg, [], [], 1, 3, "cpu", sink_frames=1)
    run.seen = 7                         # frames that have gone since are not in the cache
    assert run.seen == 7 and run._held == [3]


def test_streaming_aggregator_passes_the_runners_arguments(monkeypatch):
    """Windows and decay reach the runner."""
    from qvggt_b200.aggregator import AggConfig, VGGTAggregator
    from qvggt_b200.streaming import StreamingAggregator

    def init(self, cfg, pe, specials, frame_blocks, global_blocks, frames, device, img_hw):
        self.runner = self._make_runner(cfg, frame_blocks, global_blocks, frames, device, None, 1, 0)

    monkeypatch.setattr(VGGTAggregator, "__init__", init)
    cfg = AggConfig(depth=0, tokens_per_frame=25, grid_w=5)
    run = StreamingAggregator(cfg, None, None, [], [], 1, "cpu", max_frames=4, sink_frames=2, recent_frames=1,
                              weight_decay=0.9).runner
    assert (run.max_frames, run.sink_frames, run.recent_frames, run.weight_decay) == (4, 2, 1, 0.9)
    assert StreamingAggregator(cfg, None, None, [], [], 1, "cpu", max_frames=4).runner.weight_decay == 1
    with pytest.raises(ValueError, match="weight_decay"):
        StreamingAggregator(cfg, None, None, [], [], 1, "cpu", max_frames=4, sink_frames=2, weight_decay=2.0)
