"""GPU: the streaming K/V cache operators against their 64-bit (codes: 32-bit) restatement.

Tolerances are bounds derived from the arithmetic, element by element; each
test states its terms.  U[dtype] is half a unit in the last place of the
output type, relative.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}     # half the smallest step
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def kc():
    from qvggt_b200 import _lib, kv_cache
    _lib.device_status(clear=True)
    yield kv_cache
    assert _lib.device_status(clear=True) == 0


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------ rope
def _rope_bound(x, ref, dtype):
    # output rounding; sine and cosine off by at most 2^-20 (angle reduced in
    # double, rounded to float: 2^-23.5; sincosf 2 ulp), times |x lo| + |x hi| <= 2 max|x|
    return U[dtype] * ref.abs() * (1 + 2 ** -9) + 2.0 ** -19 * x.double().abs().amax(-1, keepdim=True) + TINY[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["axial", "split", "interleaved"])
@pytest.mark.parametrize("T,hq,hk,D,sections", [
    (1, 1, 1, 64, (16, 16)), (5, 3, 1, 64, (8, 12, 12)), (130, 16, 16, 128, (22, 21, 21)), (77, 4, 2, 80, (7, 9)),
    (33, 2, 2, 256, (32, 32, 32, 32)), (2500, 2, 1, 64, (32,)), (19, 1, 3, 10, (1, 2))])
def test_rope_axes(kc, dtype, layout, T, hq, hk, D, sections):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    q = torch.randn(T, hq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(T, hk, D, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 100000, (len(sections), T), generator=g, device="cuda", dtype=torch.int32)
    pos[:, 0] = 0
    f = torch.rand(sum(sections), generator=g, device="cuda")
    f[0] = 1.0
    for inverse in (False, True):
        a, b = kc.rope_axes(q, k, pos, f, sections, layout, inverse)
        for x, y in ((q, a), (k, b)):
            ref = ok.rope_axes(x, pos, f, sections, layout, inverse)
            assert ((y.double() - ref).abs() <= _rope_bound(x, ref, dtype)).all()


def test_rope_axes_strided_in_place_and_without_keys(kc):
    g = torch.Generator(device="cuda").manual_seed(5)
    T, H, D, sections = 41, 3, 64, (8, 8, 8)
    qkv = torch.randn(T, 3 * H * D + 8, generator=g, device="cuda").half()
    q, k = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:2 * H * D].view(T, H, D)
    pos = torch.randint(0, 50, (3, T + 7), generator=g, device="cuda", dtype=torch.int32)[:, 3:3 + T]
    f = torch.rand(24, generator=g, device="cuda")
    want = kc.rope_axes(q.contiguous(), k.contiguous(), pos.contiguous(), f, sections, "split")
    only, none = kc.rope_axes(q, None, pos, f, sections, "split")
    assert none is None and torch.equal(only, want[0])
    # heads outermost, an odd element offset
    odd = torch.randn(H * T * D + 1, generator=g, device="cuda").half()[1:].view(H, T, D).transpose(0, 1)
    got, _ = kc.rope_axes(odd, None, pos, f, sections, "interleaved")
    assert torch.equal(got, kc.rope_axes(odd.contiguous(), None, pos, f, sections, "interleaved")[0])
    rest = qkv[:, 2 * H * D:].clone()
    kc.rope_axes(q, k, pos, f, sections, "split", q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 2 * H * D:], rest)
    kc.rope_axes(q, k, pos, f, sections, "split", inverse=True, q_out=q, k_out=k)
    empty, _ = kc.rope_axes(q[:0], None, pos[:, :0], f, sections)
    assert empty.shape == (0, H, D)


# ------------------------------------------------------------------------ plan
def _plan_case(rng, B, bs, n, wide, most):
    """A table whose requests hold random distinct blocks, and the ring of the others."""
    order = rng.permutation(n).astype(np.int32)
    cached, at = [], 0
    table = np.full((B, wide), -1, np.int32)
    for b in range(B):
        want = int(rng.integers(0, min(wide, max(1, n // max(1, B))) + 1))
        table[b, :want] = order[at:at + want]
        at += want
        cached.append(max(0, want * bs - int(rng.integers(0, bs))) if want else 0)
    head = int(rng.integers(0, 5 * n))
    ring = np.full(n, -1, np.int32)
    ring[(head + np.arange(n - at)) % n] = order[at:]
    target = [int(min(wide * bs, max(0, c + rng.integers(-most, most + 1)))) for c in cached]
    return cached, target, table, ring, [head, head + n - at]


def _run_plan(kc, cached, target, table, ring, free, bs, max_new):
    t, r = torch.tensor(table, device="cuda"), torch.tensor(ring, device="cuda")
    c, g, f = ints(cached), ints(target), torch.tensor(free, dtype=torch.int64, device="cuda")
    outs = []
    for _ in range(2):               # the same inputs once more: the same result
        p = kc.block_plan(c, g, t, r, f, bs, max_new)
        outs.append(dict(table=t.cpu().numpy(), ring=r.cpu().numpy(), slots=p.slots.tolist(),
                         cu_new=p.cu_new.tolist(), cu_blocks=p.cu_blocks.tolist(), lens=p.lens.tolist(),
                         free_range=p.free_range.tolist(), status=p.status.item()))
    return outs


def _same_plan(got, want):
    assert (got["table"] == want["table"]).all() and (got["ring"] == want["ring"]).all()
    for key in ("slots", "cu_new", "cu_blocks", "lens", "free_range", "status"):
        assert got[key] == want[key], key


@pytest.mark.parametrize("B,bs,n,wide,most,seed", [
    (1, 32, 4, 3, 40, 0), (1, 1, 9, 9, 5, 1), (3, 64, 40, 20, 500, 2), (33, 16, 300, 12, 90, 3),
    (1000, 32, 4000, 9, 60, 4), (513, 128, 700, 4, 1, 5), (8192, 32, 20000, 5, 33, 6)])
def test_block_plan(kc, B, bs, n, wide, most, seed):
    rng = np.random.default_rng(seed)
    for k in range(3):
        case = _plan_case(rng, B, bs, n, wide, most)
        total = sum(max(0, t - c) for c, t in zip(case[0], case[1]))
        want = ok.block_plan(*case, bs, total + 7 * k)
        for got in _run_plan(kc, *case, bs, total + 7 * k):
            _same_plan(got, want)


def test_block_plan_all_or_nothing(kc):
    table, ring = np.full((3, 2), -1, np.int32), np.arange(4, dtype=np.int32)
    table[0, 0] = 3
    base = ([20, 0, 0], table, ring, [0, 3])
    for target, most, status in [([20, 65, 1], 200, 2), ([64, 33, 20], 200, 1), ([20, -1, 3], 200, 3),
                                 ([32, 33, 0], 44, 4), ([32, 33, 0], 45, 0), ([0, 64, 32], 100, 0), ([20, 0, 0], 0, 0)]:
        want = ok.block_plan(base[0], target, table, ring, base[3], 32, most)
        assert want["status"] == status
        for got in _run_plan(kc, base[0], target, table, ring, base[3], 32, most):
            _same_plan(got, want)


# ---------------------------------------------------------------- append, gather
def _random_table(rng, need, num, wide):
    order = rng.permutation(num)
    table, at = np.full((len(need), wide), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def _cu(v):
    return np.concatenate([[0], np.cumsum(v)]).astype(np.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cached,new,H,D,bs", [
    ([0], [1], 1, 64, 32), ([0, 5, 64], [1, 1, 1], 2, 128, 64), ([63, 64, 65, 0], [1, 1, 130, 0], 3, 64, 64),
    ([100], [700], 16, 64, 128), ([31, 0, 7], [2, 64, 33], 4, 128, 32), ([0] * 40, list(range(40)), 1, 64, 32)])
def test_append_is_bit_exact_and_gather_reads_it_back(kc, dtype, cached, new, H, D, bs):
    rng = np.random.default_rng(len(cached) + D)
    g = torch.Generator().manual_seed(len(cached) + bs)
    target = [c + n for c, n in zip(cached, new)]
    need = [-(-t // bs) for t in target]
    num, wide = sum(need) + 3, max(need) + 2
    table = _random_table(rng, need, num, wide)
    codes = [rng.integers(-127, 128, (num, H, bs, D)).astype(np.int8) for _ in range(2)]
    scales = [np.exp(rng.normal(-4, 1, (num, H))).astype(np.float32) for _ in range(2)]
    dev = [torch.tensor(a, device="cuda") for a in codes + scales]
    T = sum(new)
    kv = (torch.randn(T, 2, H, D, generator=g) * torch.exp(torch.randn(T, 1, H, 1, generator=g))).to(dtype)
    cu = _cu(new)
    units = _cu([(t - 1) // bs - c // bs + 1 if t > c else 0 for c, t in zip(cached, target)])
    on = kv.cuda()
    kc.kv_append(on[:, 0], on[:, 1], *dev, torch.tensor(table, device="cuda"), ints(cached), ints(cu.tolist()),
                 ints(units.tolist()))
    for s in range(2):
        ok.append_f32(kv[:, s], codes[s], scales[s], table, cached, cu)
        assert (dev[s].cpu().numpy() == codes[s]).all()
        assert (dev[2 + s].cpu().numpy() == scales[s]).all()
    slots = [int(table[b, j // bs]) * bs + j % bs for b, t in enumerate(target) for j in range(t)] + [-1]
    rows = kc.kv_gather(*dev, ints(slots), dtype)
    at = np.array(slots[:-1])
    want = [codes[s][at // bs, :, at % bs].astype(np.float32) * scales[s][at // bs][..., None] for s in range(2)]
    want = torch.tensor(np.stack(want, 1)).to(dtype).reshape(len(at), -1)
    assert torch.equal(rows[:-1].cpu(), want) and (rows[-1] == 0).all()


def test_append_special_values(kc):
    """Zeros, infinities and NaN: finite values keep their precision, infinities saturate, NaN becomes 0."""
    H, D, bs = 2, 64, 32
    kv = torch.zeros(6, 2, H, D, dtype=torch.float16)
    kv[0, 0, 0, :4] = torch.tensor([1.0, -2.0, math.inf, -math.inf])
    kv[1, 0, 0, 0] = math.nan
    kv[:, 1, 0] = 2.0 ** -24          # the smallest fp16
    kv[2, 1, 1, 5] = math.inf         # nothing finite in this head but zeros
    codes = [np.zeros((2, H, bs, D), np.int8) for _ in range(2)]
    scales = [np.full((2, H), 7.0, np.float32) for _ in range(2)]
    dev = [torch.tensor(a, device="cuda") for a in codes + scales]
    table, on = np.array([[1]], np.int32), kv.cuda()
    kc.kv_append(on[:, 0], on[:, 1], *dev, torch.tensor(table, device="cuda"), ints([0]), ints([0, 6]), ints([0, 1]))
    for s in range(2):
        ok.append_f32(kv[:, s], codes[s], scales[s], table, [0], [0, 6])
        assert (dev[s].cpu().numpy() == codes[s]).all() and (dev[2 + s].cpu().numpy() == scales[s]).all()
    assert codes[0][1, 0, 0, :4].tolist() == [64, -127, 127, -127] and codes[0][1, 0, 1, 0] == 0
    assert scales[0][1, 0] == np.float32(2) / np.float32(127) and scales[1][1, 1] == np.float32(2.0 ** -60)


# --------------------------------------------------------------------- attention
def _attn_inputs(seed, ql, kl, hq, hk, D, bs, dtype, spare=3):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // bs) for n in kl]
    num = sum(need) + spare
    table = torch.tensor(_random_table(rng, need, num, max(need + [1])), device="cuda")
    kcodes, vcodes = (torch.randint(-128, 128, (num, hk, bs, D), generator=g, device="cuda", dtype=torch.int8)
                      for _ in range(2))
    ks, vs = (torch.exp(0.7 * torch.randn(num, hk, generator=g, device="cuda")) / 80 for _ in range(2))
    q = torch.randn(sum(ql), hq, D, generator=g, device="cuda").to(dtype)
    return q, kcodes, vcodes, ks, vs, table, ints(_cu(ql).tolist()), ints(kl)


def _check_attention(got, lse, ref, dtype, vmax, n):
    """|error| <= output rounding
                + (P's fp16 rounding 2^-11, scores and exponentials 2^-13) * sum w |v|
                + P's steps below fp16's normal range: n keys, 2^-25 each of the largest |v|."""
    out, want_lse, mag = ref
    bound = U[dtype] * out.abs() * 1.01 + (2.0 ** -11 + 2.0 ** -13) * mag + n * 2.0 ** -25 * vmax + TINY[dtype]
    assert torch.isfinite(got).all()
    assert ((got.double() - out).abs() <= bound).all(), float(((got.double() - out).abs() / bound).max())
    none = torch.isinf(want_lse)
    assert (lse[none] == -math.inf).all()
    assert ((lse.double() - want_lse)[~none].abs() <= 2e-4).all()


CASES = [
    # ql, kl, hq, hk, D, bs, chunk
    ([1], [1], 1, 1, 64, 32, 0), ([1], [300], 16, 16, 128, 64, 0), ([1, 1, 1], [64, 65, 63], 4, 4, 64, 64, 1),
    ([3, 1, 0, 5], [9, 0, 40, 5], 2, 1, 64, 32, 1), ([5], [2], 3, 1, 128, 32, 1),          # rows without keys
    ([4, 7], [900, 33], 14, 2, 128, 128, 1), ([16], [1000], 6, 2, 64, 64, 5), ([17], [2049], 1, 1, 64, 64, 0),
    ([40, 1, 130], [70, 700, 131], 4, 2, 64, 64, 1), ([129], [129], 8, 8, 128, 32, 1),
    ([260], [1300], 2, 2, 64, 128, 60), ([300, 20], [300, 1555], 3, 1, 128, 64, 7),
    ([274], [822], 2, 2, 64, 64, 274), ([1374], [1374], 2, 2, 64, 64, 0), ([2], [20000], 1, 1, 64, 64, 1),
    ([1] * 70, [17 * i % 640 for i in range(70)], 4, 1, 64, 32, 1), ([513], [600], 7, 1, 64, 32, 1),
    ([256], [256], 5, 1, 128, 128, 0), ([700], [3], 1, 1, 64, 64, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ql,kl,hq,hk,D,bs,chunk", CASES)
def test_cached_attention(kc, dtype, ql, kl, hq, hk, D, bs, chunk):
    args = _attn_inputs(len(ql) + D + sum(kl), ql, kl, hq, hk, D, bs, dtype)
    lse = torch.full((hq, sum(ql)), 7.0, device="cuda")
    got = kc.cached_attention(*args, max(ql), max(kl), chunk, lse=lse)
    ref = ok.cached_attention(*args, chunk)
    vmax = float((args[4].max() * 128))
    _check_attention(got, lse, ref, dtype, vmax, max(kl))
    # again, and without lse: the same bits
    assert torch.equal(kc.cached_attention(*args, max(ql), max(kl), chunk), got)


@pytest.mark.parametrize("ql,kl,hint", [([2], [5000], 1), ([2], [50], 200000), ([200], [3000], 10),
                                        ([200], [200], 100000)])
def test_cached_attention_length_hint_is_only_a_hint(kc, ql, kl, hint):
    """max_kv lays out the work; longer and shorter lengths are served all the same."""
    args = _attn_inputs(1, ql, kl, 2, 2, 64, 64, torch.float16)
    lse = torch.empty(2, sum(ql), device="cuda")
    got = kc.cached_attention(*args, max(ql), hint, 1, lse=lse)
    _check_attention(got, lse, ok.cached_attention(*args, 1), torch.float16, float(args[4].max() * 128), max(kl))


@pytest.mark.parametrize("ql,chunk", [([3], 1), ([150], 1), ([150], 64)])
def test_cached_attention_strides_scale_and_scratch(kc, ql, chunk):
    T, hq, D, kl = sum(ql), 4, 64, [333]
    q, kcodes, vcodes, ks, vs, table, cu, lens = _attn_inputs(9, ql, kl, hq, 2, D, 64, torch.bfloat16)
    qkv = torch.randn(T, 3 * hq * D, device="cuda").bfloat16()
    qs = qkv[:, hq * D:2 * hq * D].view(T, hq, D)
    qs.copy_(q)
    both = torch.empty(kcodes.shape[0], 2, *kcodes.shape[1:], dtype=torch.int8, device="cuda")
    both[:, 0], both[:, 1] = kcodes, vcodes
    wide = torch.zeros(hq, T, 2 * D, device="cuda").bfloat16()
    out = wide.transpose(0, 1)[..., D:]
    need = kc.attention_scratch_bytes(T, hq, 2, 1, max(ql), 333, D)
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    got = kc.cached_attention(qs, both[:, 0], both[:, 1], ks, vs, table, cu, lens, max(ql), 333, chunk, scale=0.3,
                              out=out, scratch=scratch)
    assert got is out and (wide[..., :D] == 0).all()
    ref = ok.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, chunk, scale=0.3)
    lse = torch.empty(hq, T, device="cuda")
    kc.cached_attention(qs, both[:, 0], both[:, 1], ks, vs, table, cu, lens, max(ql), 333, chunk, scale=0.3, lse=lse)
    _check_attention(got, lse, ref, torch.bfloat16, float(vs.max() * 128), 333)


@pytest.mark.parametrize("ql", [4, 200])
def test_cached_attention_masked_blocks_may_hold_anything(kc, ql):
    """Scales of blocks that a row does not see are NaN or infinite, table entries past the length are out of range."""
    kl, bs = 320, 32
    q, kcodes, vcodes, ks, vs, table, cu, lens = _attn_inputs(4, [ql], [kl], 2, 2, 64, bs, torch.float16)
    chunk = 64
    args = (q, kcodes, vcodes, ks, vs, table, cu, lens)
    want = ok.cached_attention(*args, chunk)
    table = torch.cat([table, torch.full((1, 2), 2 ** 30, dtype=torch.int32, device="cuda")], 1)
    got = kc.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, ql, kl, chunk)
    vmax = float(vs.max() * 128)
    lse = torch.empty(2, ql, device="cuda")
    kc.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, ql, kl, chunk, lse=lse)
    _check_attention(got, lse, want, torch.float16, vmax, kl)
    # the last chunk's keys poisoned: rows of earlier chunks keep their bits
    last = table[0, (kl - chunk) // bs:kl // bs].long()
    ks2, vs2 = ks.clone(), vs.clone()
    ks2[last], vs2[last] = math.nan, math.inf
    bad = kc.cached_attention(q, kcodes, vcodes, ks2, vs2, table, cu, lens, ql, kl, chunk)
    early = [i for i in range(ql) if ok.key_limit(i, ql, kl, chunk) <= kl - chunk]
    late = [i for i in range(ql) if i not in early]
    assert torch.equal(bad[early], got[early]) and torch.isnan(bad[late]).any(-1).all()


@pytest.mark.parametrize("ql", [2, 140])
def test_cached_attention_extreme_scales(kc, ql):
    """V scales from 2^-60 to large, K scales that make one key dominate."""
    q, kcodes, vcodes, ks, vs, table, cu, lens = _attn_inputs(6, [ql], [500], 2, 1, 64, 64, torch.float16)
    vs[table[0, :3].long()] = 2.0 ** -60
    vs[table[0, 4].long()] = 300.0
    ks[table[0, 2].long()] *= 40
    lse = torch.empty(2, ql, device="cuda")
    got = kc.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, ql, 500, 1, lse=lse)
    out, want_lse, mag = ok.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, 1)
    # scores up to ~2000 here: their fp32 rounding (64 terms) is a relative error of the weights of up to
    # 2000 * 2^-22, on top of the usual terms
    err = 2.0 ** -11 + 2000 * 2.0 ** -22
    vmax = 300.0 * 128
    bound = 2.0 ** -11 * out.abs() * 1.01 + err * 2 * mag + 500 * 2.0 ** -25 * vmax + 2.0 ** -25
    assert ((got.double() - out).abs() <= bound).all()
    assert ((lse.double() - want_lse).abs() <= 2000 * 2.0 ** -22 + 2e-4).all()


def test_cached_attention_skips_and_reports_bad_blocks_and_lengths(kc):
    from qvggt_b200 import _lib
    q, kcodes, vcodes, ks, vs, table, cu, lens = _attn_inputs(8, [2, 3], [100, 90], 2, 2, 64, 32, torch.float16)
    good = kc.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, lens, 3, 100, 0)
    assert _lib.device_status() == 0
    bad = table.clone()
    bad[0, 1] = kcodes.shape[0]
    got = kc.cached_attention(q, kcodes, vcodes, ks, vs, bad, cu, lens, 3, 100, 0)
    assert _lib.device_status(clear=True) == 0x201
    assert torch.equal(got[2:], good[2:]) and torch.isfinite(got).all()
    for wrong in (ints([100000, 90]), ints([-3, 90])):
        got = kc.cached_attention(q, kcodes, vcodes, ks, vs, table, cu, wrong, 3, 100, 0)
        assert _lib.device_status(clear=True) == 0x202
        assert torch.equal(got[2:], good[2:])
    kc.cached_attention(q, kcodes, vcodes, ks, vs, table, ints([0, 2, 99]), lens, 3, 100, 0)
    assert _lib.device_status(clear=True) == 0x202
    kc.kv_append(q[:, :, :], q, kcodes, vcodes, ks, vs, bad, ints([33, 0]), ints([0, 2, 5]), ints([0, 1, 2]))
    assert _lib.device_status(clear=True) == 0x201
    kc.kv_gather(kcodes, vcodes, ks, vs, ints([0, kcodes.shape[0] * 32]))
    assert _lib.device_status(clear=True) == 0x201


def test_cached_attention_past_two_gib(kc):
    """Blocks whose codes start beyond 2^31 elements."""
    num, H, bs, D = 2 ** 31 // (16 * 64 * 64) + 40, 16, 64, 64
    k, v = (torch.zeros(num, H, bs, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = torch.ones(num, H, device="cuda"), torch.ones(num, H, device="cuda")
    small = _attn_inputs(3, [3], [150], H, H, D, bs, torch.float16, spare=0)
    far = torch.arange(num - 3, num, device="cuda")
    at = small[5][0].long()
    k[far], v[far], ks[far], vs[far] = small[1][at], small[2][at], small[3][at], small[4][at]
    table = far.to(torch.int32)[None].contiguous()
    for ql in (3, 150):
        q = torch.randn(ql, H, D, device="cuda").half()
        cu = ints([0, ql])
        want = kc.cached_attention(q, *small[1:6], cu, small[7], ql, 150, 1)
        assert torch.equal(kc.cached_attention(q, k, v, ks, vs, table, cu, small[7], ql, 150, 1), want)
    x = torch.randn(5, 2, H, D, device="cuda").half()
    new = table[:, 2:].contiguous()
    kc.kv_append(x[:, 0], x[:, 1], k, v, ks, vs, new, ints([0]), ints([0, 5]), ints([0, 1]))
    rows = kc.kv_gather(k, v, ks, vs, (new[0, 0] * bs + torch.arange(5, device="cuda")).to(torch.int32))
    assert (rows.float() - x.reshape(5, -1).float()).abs().max() <= 0.5 * float(ks[far].max()) * 1.01


def test_other_stream(kc):
    args = _attn_inputs(11, [4, 90], [700, 400], 4, 2, 64, 64, torch.float16)
    want = kc.cached_attention(*args, 90, 700, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        # behind a slow kernel that writes the queries: the call must be on this stream
        q = torch.zeros_like(args[0])
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            a = a @ a * 1e-3
        q.copy_(args[0] + (a[0, 0] * 0).half().nan_to_num())
        got = kc.cached_attention(q, *args[1:], 90, 700, 1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


# -------------------------------------------------------------------- the cache
def test_paged_cache_streams_like_one_pass(kc):
    """Three requests growing over several steps, one ended and reused: each step equals the restatement on what the
    cache then holds, and the new rows are in it to half a step of its scales (and fp16's rounding)."""
    H, D, bs, layers = 2, 64, 32, 2
    cache = kc.PagedKVCache(layers, 24, H, D, 3, 256, bs)
    g = torch.Generator(device="cuda").manual_seed(0)
    lens = [0, 0, 0]
    for new in ([40, 1, 0], [3, 31, 64], [-1, 1, 1], [50, 5, 2]):
        target = [0 if n < 0 else c + n for c, n in zip(lens, new)]
        counts = [max(0, t - c) for c, t in zip(lens, target)]
        T = sum(counts)
        plan = cache.plan(ints(target), T)
        cache.check(plan)
        x = torch.randn(3, T, H, D, generator=g, device="cuda").half()
        for layer in range(layers):
            cache.append(layer, x[1] + layer, x[2], plan)
            q = x[0]
            got = cache.attend(layer, q, plan, max(counts), max(target), 1)
            lse = torch.empty(H, T, device="cuda")
            kc.cached_attention(q, cache.k[layer], cache.v[layer], cache.k_scale[layer], cache.v_scale[layer],
                                cache.block_tables, plan.cu_new, plan.lens, max(counts), max(target), 1, lse=lse)
            ref = ok.cached_attention(q, cache.k[layer], cache.v[layer], cache.k_scale[layer], cache.v_scale[layer],
                                      cache.block_tables, plan.cu_new, plan.lens, 1)
            _check_attention(got, lse, ref, torch.float16, float(cache.v_scale[layer].max() * 128), max(target))
        rows = cache.gather(0, plan.slots)
        want = torch.cat([x[1].reshape(T, -1), x[2].reshape(T, -1)], 1).float()
        step = max(float(cache.k_scale[0].max()), float(cache.v_scale[0].max()))
        assert (rows.float() - want).abs().max() <= 0.5 * step * 1.01 + 2.0 ** -9
        cache.commit(plan)
        lens = target
    cache.check(cache.plan(ints([256, 256, 256]), 1000))       # the pool's 24 blocks to the last one
    with pytest.raises(RuntimeError, match="table row"):
        cache.check(cache.plan(ints([256, 257, 256]), 1000))
    assert cache.lens.tolist() == lens


def test_refusals(kc):
    q, kcodes, vcodes, ks, vs, table, cu, lens = _attn_inputs(2, [4], [50], 4, 2, 64, 32, torch.float16)
    ok_args = dict(max_q=4, max_kv=50)
    call = kc.cached_attention
    from qvggt_b200._lib import QvggtError
    with pytest.raises(TypeError):
        call(q.float(), kcodes, vcodes, ks, vs, table, cu, lens, **ok_args)
    with pytest.raises(ValueError, match="head_dim"):
        call(q[..., :32], kcodes, vcodes, ks, vs, table, cu, lens, **ok_args)
    with pytest.raises(QvggtError, match="share"):
        call(q[:, :3].contiguous(), kcodes, vcodes, ks, vs, table, cu, lens, **ok_args)
    with pytest.raises(TypeError):
        call(q, kcodes, vcodes, ks, vs, table.long(), cu, lens, **ok_args)
    with pytest.raises(ValueError):
        call(q, kcodes, vcodes, ks, vs, table, cu[:1], lens, **ok_args)
    with pytest.raises(QvggtError, match="aligned"):
        odd = torch.zeros(4 * 4 * 64 + 1, device="cuda").half()[1:].view(4, 4, 64)
        call(odd, kcodes, vcodes, ks, vs, table, cu, lens, **ok_args)
    with pytest.raises(QvggtError, match="scale"):
        call(q, kcodes, vcodes, ks, vs, table, cu, lens, 4, 50, 0, scale=-1.0)
    with pytest.raises(QvggtError, match="causal_chunk"):
        call(q, kcodes, vcodes, ks, vs, table, cu, lens, 4, 50, -1)
    with pytest.raises(ValueError, match="lse"):
        call(q, kcodes, vcodes, ks, vs, table, cu, lens, 4, 50, lse=torch.empty(4, 5, device="cuda"))
    with pytest.raises(ValueError, match="scratch"):
        call(q, kcodes, vcodes, ks, vs, table, cu, lens, 4, 50000,
             scratch=torch.empty(1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="devices|CUDA"):
        call(q, kcodes, vcodes, ks, vs, table.cpu(), cu, lens, **ok_args)
    with pytest.raises(ValueError, match="layout"):
        kc.rope_axes(q, None, ints([[0, 1, 2, 3]]), torch.ones(8, device="cuda"), (8,), layout="half")
    with pytest.raises(QvggtError, match="fit"):
        kc.rope_axes(q, None, ints([[0, 1, 2, 3]]), torch.ones(33, device="cuda"), (33,))
    with pytest.raises(ValueError, match="positions"):
        kc.rope_axes(q, None, ints([[0, 1, 2]]), torch.ones(8, device="cuda"), (8,))
    with pytest.raises(QvggtError, match="aligned"):
        kc.kv_append(q[:, :2, :], torch.zeros(4 * 2 * 64 + 4, device="cuda").half()[4:].view(4, 2, 64), kcodes, vcodes,
                     ks, vs, table, lens, cu, cu)
    with pytest.raises(ValueError):
        kc.kv_append(q, q, kcodes, vcodes, ks, vs, table, lens, cu, cu)
    with pytest.raises(QvggtError, match="power of two"):
        kc.block_plan(lens, lens, table, table.view(-1), torch.zeros(2, dtype=torch.int64, device="cuda"), 48, 4)
