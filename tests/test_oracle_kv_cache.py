"""CPU: the restatement of the streaming K/V cache operators against independent forms, and the refusals of the public calls."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok
from oracle import rope as orope
from qvggt_b200 import kv_cache as kc


# ------------------------------------------------------------------ restatement
@pytest.mark.parametrize("layout", ["axial", "split", "interleaved"])
@pytest.mark.parametrize("sections", [(5,), (8, 8), (2, 3, 3), (1, 2, 3, 4)])
def test_rope_is_a_rotation_and_its_inverse_is_its_gradient(layout, sections):
    g = torch.Generator().manual_seed(1)
    D = 2 * sum(sections) + 4
    T = 7
    x = torch.randn(T, 3, D, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 900, (len(sections), T), generator=g, dtype=torch.int32)
    f = torch.rand(sum(sections), generator=g)
    y = ok.rope_axes(x, pos, f, sections, layout)
    assert torch.allclose(ok.rope_axes(y, pos, f, sections, layout, inverse=True), x, atol=1e-12)
    assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
    assert torch.equal(y[..., D - 4:], x[..., D - 4:])
    # gradient of sum(w * y) in x, by central differences and by turning back
    w = torch.randn(T, 3, D, generator=g, dtype=torch.float64)
    grad = ok.rope_axes(w, pos, f, sections, layout, inverse=True)
    for t, h, d in [(0, 0, 0), (3, 1, D - 1), (6, 2, sum(sections)), (2, 0, 1)]:
        e = torch.zeros_like(x)
        e[t, h, d] = 1e-3
        num = ((w * ok.rope_axes(x + e, pos, f, sections, layout)).sum()
               - (w * ok.rope_axes(x - e, pos, f, sections, layout)).sum()) / 2e-3
        assert abs(num - grad[t, h, d]) < 1e-8


def test_rope_two_axes_is_the_models_2d_rope():
    """Axial sections (16, 16) with positions (row, column) are the aggregator's 2-D RoPE (its tables round to fp16)."""
    T = 60
    x = torch.randn(T, 2, 64, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    rows, cols = torch.arange(T) // 8 + 1, torch.arange(T) % 8 + 1
    f = 1.0 / (100.0 ** (torch.arange(0, 32, 2, dtype=torch.float32) / 32))
    y = ok.rope_axes(x, torch.stack([rows, cols]).int(), torch.cat([f, f]), (16, 16), "axial")

    def one(v, p):                       # rotate-half over 32 dims
        ang = (p[:, None].double() * f.double()).repeat(1, 2)[:, None]
        rot = torch.cat([-v[..., 16:], v[..., :16]], -1)
        return v * ang.cos() + rot * ang.sin()

    want = torch.cat([one(x[..., :32], rows), one(x[..., 32:], cols)], -1)
    assert torch.allclose(y, want, atol=1e-12)


def test_plan_against_a_dictionary_allocator():
    """Many steps: every held block is held once, tables map tokens to the blocks they were given."""
    rng = np.random.default_rng(0)
    B, bs, n, wide = 5, 4, 24, 12
    table = np.full((B, wide), -1, np.int32)
    ring, free = np.arange(n, dtype=np.int32), [0, n]
    lens = [0] * B
    for _ in range(60):
        target = [max(0, c + int(rng.integers(-9, 12))) for c in lens]
        r = ok.block_plan(lens, target, table, ring, free, bs, 64)
        held = [int(r["table"][b, j]) for b in range(B) for j in range(-(-r["lens"][b] // bs))]
        spare = [int(r["ring"][i % n]) for i in range(*r["free_range"])]
        assert sorted(held + spare) == list(range(n))
        if r["status"] == 0:
            assert r["lens"] == target
            for b in range(B):       # what was held before stays where it was
                keep = min(-(-lens[b] // bs), -(-target[b] // bs))
                assert (r["table"][b, :keep] == table[b, :keep]).all()
        else:
            assert r["lens"] == lens and r["free_range"] == free
        table, ring, free, lens = r["table"], r["ring"], r["free_range"], r["lens"]


@pytest.mark.parametrize("chunk", [0, 1, 3])
def test_attention_against_softmax_of_the_dequantised_rows(chunk):
    g = torch.Generator().manual_seed(3)
    bs, D, hk, hq = 4, 8, 2, 4
    kc_, vc = (torch.randint(-127, 128, (6, hk, bs, D), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.rand(6, hk, generator=g) * 0.02 + 0.001 for _ in range(2))
    table = torch.tensor([[3, 0, 5], [1, 4, -1]], dtype=torch.int32)
    cu, lens = torch.tensor([0, 5, 9], dtype=torch.int32), torch.tensor([11, 2], dtype=torch.int32)
    q = torch.randn(9, hq, D, generator=g)
    out, lse, mag = ok.cached_attention(q, kc_, vc, ks, vs, table, cu, lens, chunk)
    for b in range(2):
        ql, n = int(cu[b + 1] - cu[b]), int(lens[b])
        for i in range(ql):
            pos = n - ql + i
            vis = [j for j in range(n) if chunk == 0 or (pos >= 0 and j < (pos // chunk + 1) * chunk)]
            for h in range(hq):
                kv = h // 2
                row = cu[b] + i
                if not vis:
                    assert (out[row, h] == 0).all() and lse[h, row] == -math.inf
                    continue
                blk = [int(table[b, j // bs]) for j in vis]
                k = torch.stack([kc_[x, kv, j % bs].double() * ks[x, kv].double() for x, j in zip(blk, vis)])
                v = torch.stack([vc[x, kv, j % bs].double() * vs[x, kv].double() for x, j in zip(blk, vis)])
                s = k @ q[row, h].double() / math.sqrt(D)
                assert torch.allclose(out[row, h], torch.softmax(s, 0) @ v)
                assert torch.allclose(lse[h, row], torch.logsumexp(s, 0))


def test_append_error_is_half_a_step():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(11, 2, 8, generator=g).half()
    codes, scales = np.zeros((3, 2, 4, 8), np.int8), np.ones((3, 2), np.float32)
    table = [[2, 0, 1]]
    ok.append_f32(x[:6], codes, scales, table, [0], [0, 6])
    ok.append_f32(x[6:] * 3, codes, scales, table, [6], [0, 5])
    want = torch.cat([x[:6], x[6:] * 3]).double().numpy()
    for j in range(11):
        blk = table[0][j // 4]
        got = codes[blk, :, j % 4].astype(np.float64) * scales[blk][:, None]
        steps = 1.0 if j in (4, 5) else 0.5       # rows 4, 5 were rounded a second time
        assert (np.abs(got - want[j]) <= steps * scales[blk][:, None] * (1 + 1e-5)).all()


# ---------------------------------------------------------------------- refusals
def _cache(nb=4, h=2, bs=32, d=64):
    return (torch.zeros(nb, h, bs, d, dtype=torch.int8), torch.zeros(nb, h, bs, d, dtype=torch.int8),
            torch.ones(nb, h), torch.ones(nb, h))


def test_no_cpu_path():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    x = torch.zeros(3, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        kc.rope_axes(x, x, i(1, 3), torch.ones(32), (32,))
    with pytest.raises(ValueError, match="CUDA"):
        kc.block_plan(i(1), i(1), i(1, 2), i(4), torch.zeros(2, dtype=torch.int64), 32, 8)
    with pytest.raises(ValueError, match="CUDA"):
        kc.kv_append(x, x, *_cache(), i(1, 2), i(1), i(2), i(2))
    with pytest.raises(ValueError, match="CUDA"):
        kc.kv_gather(*_cache(), i(3))
    with pytest.raises(ValueError, match="CUDA"):
        kc.cached_attention(x, *_cache(), i(1, 2), i(2), i(1), 3, 64)


def test_cache_checks():
    k, v, ks, vs = _cache()
    assert kc._check_cache("t", k, v, ks, vs) == (4, 2, 32, 64)
    # blocks of a larger buffer: the block stride may differ
    both = torch.zeros(4, 2, 2, 32, 64, dtype=torch.int8)
    assert kc._check_cache("t", both[:, 0], both[:, 1], ks, vs) == (4, 2, 32, 64)
    with pytest.raises(TypeError):
        kc._check_cache("t", k.half(), v, ks, vs)
    with pytest.raises(ValueError):
        kc._check_cache("t", k, v[:3], ks, vs)
    with pytest.raises(ValueError):
        kc._check_cache("t", k.transpose(2, 3).contiguous().transpose(2, 3), v, ks, vs)
    with pytest.raises(ValueError):
        kc._check_cache("t", k, v, ks.double(), vs)
    with pytest.raises(ValueError):
        kc._check_cache("t", k, v, ks, vs[:, :1])
    with pytest.raises(ValueError):
        kc.PagedKVCache(1, 4, 2, 96, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        kc.PagedKVCache(1, 4, 2, 64, 1, 64, block_size=48, device="cpu")


def test_library_refuses_bad_arguments_without_a_gpu():
    """Argument checks come before any device call: code and message."""
    import os

    from qvggt_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    n = _lib.i64(0)
    for args, word in [((8, 6, 4, 1, 8, 64, 64), b"share"), ((8, 4, 4, 1, 8, 64, 96), b"head_dim"),
                       ((-1, 4, 4, 1, 8, 64, 64), b"shape")]:
        assert lib.qvggt_cached_attention_scratch(*args, n) in (1, 2)
        assert word in lib.qvggt_last_error()
    plan = lambda requests, bs: kc._PLAN(0, 0, requests, 0, 1, 0, 8, 0, bs, 0, 0, 0, 0, 0, 0, 0)
    assert lib.qvggt_block_plan(plan(9000, 32), None) == 2
    assert lib.qvggt_block_plan(plan(1, 33), None) == 1
    assert lib.qvggt_block_plan(plan(1, 32), None) == 1 and b"null" in lib.qvggt_last_error()
    rope = lambda pairs, dtype: kc._ROPE(16, 64, 64, 16, 64, 64, 1, *(0,) * 7, 4, 64, 16, 4, 16, pairs, 0, 0, 0, 1, 0,
                                         0, dtype)
    assert lib.qvggt_rope_axes(rope(40, 0), None) == 1 and b"fit" in lib.qvggt_last_error()
    assert lib.qvggt_rope_axes(rope(32, 2), None) == 2
    cache = lambda bs, stride: (16, 16, stride, 16, 16, 4, 1, bs, 64)
    assert lib.qvggt_kv_append(kc._APPEND(*cache(48, 4096), 16, 64, 64, 16, 64, 64, 1, 0, 16, 1, 16, 16, 16, 1, 1),
                               None) == 2
    assert lib.qvggt_kv_gather(kc._GATHER(*cache(32, 2056), 16, 1, 16, 128, 0), None) == 5
    attend = lambda scale, chunk: kc._ATTEND(*cache(32, 2048), 16, 64, 64, 16, 64, 64, 0, 1, 1, 0, 16, 1, 16, 16, 1, 1,
                                             32, chunk, scale, 0, 0)
    for args, word in [((0.0, 0), b"scale"), ((float("nan"), 0), b"scale"), ((0.1, -1), b"chunk")]:
        assert lib.qvggt_cached_attention(attend(*args), None) == 1 and word in lib.qvggt_last_error()


def test_packed_structures_match_the_header():
    """Every field of the header's argument structures is 64 bits wide, so their number is the packed size."""
    import os
    import re
    hdr = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                            "qvggt_b200.h")).read()
    hdr = re.sub(r"/\*.*?\*/", "", hdr, flags=re.S)
    fields = {}
    for body, name in re.findall(r"typedef struct \{(.*?)\} (qvggt_\w+);", hdr, flags=re.S):
        n = 0
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            if decl.startswith("qvggt_kv_cache"):
                n += fields["qvggt_kv_cache"]
                continue
            assert "*" in decl or decl.startswith(("int64_t", "double")), decl
            for item in decl.split(","):
                m = re.search(r"\[(\d+)\]", item)
                n += int(m.group(1)) if m else 1
        fields[name] = n
    for name, pack in [("rope_axes", kc._ROPE), ("block_plan", kc._PLAN), ("kv_append", kc._APPEND),
                       ("kv_gather", kc._GATHER), ("cached_attention", kc._ATTEND)]:
        assert fields[f"qvggt_{name}_args"] * 8 == pack.__self__.size, name
