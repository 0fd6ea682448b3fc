"""GPU: gathered key weights, the choice of the keys that stay and their move, against their restatement.

Weights are compared within a bound derived element by element (``oracle.kv_evict.key_weights`` states its terms); the
choice is whole numbers, the move's codes and scales 32-bit arithmetic: both bit for bit.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as ok
from oracle import kv_evict as oe

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def kc():
    from qvggt_b200 import _lib, kv_cache
    _lib.device_status(clear=True)
    yield kv_cache
    assert _lib.device_status(clear=True) == 0


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(v):
    return np.concatenate([[0], np.cumsum(v)]).astype(np.int32).tolist()


def random_table(rng, lens, bs, spare=3, wider=0):
    need = [-(-n // bs) for n in lens]
    num = sum(need) + spare
    order = rng.permutation(num)
    table, at = np.full((len(need), max(need + [1]) + wider), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, num


# ---------------------------------------------------------------- gathered weights
def weigh_inputs(seed, ql, kl, hq, hk, D, bs, dtype, chunk):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    table, num = random_table(rng, kl, bs)
    codes = torch.randint(-128, 128, (num, hk, bs, D), generator=g, device="cuda", dtype=torch.int8)
    ks = torch.exp(0.7 * torch.randn(num, hk, generator=g, device="cuda")) / 80
    q = torch.randn(sum(ql), hq, D, generator=g, device="cuda").to(dtype)
    table, cu, lens = torch.tensor(table, device="cuda"), ints(cu_of(ql)), ints(kl)
    lse = ok.cached_attention(q, codes, codes, ks, ks, table, cu, lens, chunk)[1].float()
    w = torch.rand(num, hk, bs, generator=g, device="cuda") * 3
    return q, codes, ks, table, cu, lens, lse, w


def check_weights(got, want):
    value, err = want
    assert torch.isfinite(got).all()
    off = (got.double() - value).abs()
    assert (off <= err).all(), float((off / err.clamp(min=1e-300)).max())


WEIGH = [
    # ql, kl, hq, hk, D, bs, chunk
    ([1], [1], 1, 1, 64, 32, 0), ([1], [300], 16, 16, 128, 64, 0), ([1, 1, 1], [64, 65, 63], 4, 4, 64, 64, 1),
    ([3, 1, 0, 5], [9, 0, 40, 5], 2, 1, 64, 32, 1), ([5], [2], 3, 1, 128, 32, 1),          # rows without keys
    ([4, 7], [900, 33], 14, 2, 128, 128, 1), ([16], [1000], 6, 2, 64, 64, 5), ([17], [2049], 1, 1, 64, 64, 0),
    ([40, 1, 130], [70, 700, 131], 4, 2, 64, 64, 1), ([129], [129], 8, 8, 128, 32, 1),
    ([260], [1300], 2, 2, 64, 128, 60), ([300, 20], [300, 1555], 3, 1, 128, 64, 7),
    ([274], [822], 2, 2, 64, 64, 274), ([1374], [1374], 2, 2, 64, 64, 0), ([2], [20000], 1, 1, 64, 64, 1),
    ([1] * 70, [17 * i % 640 for i in range(70)], 4, 1, 64, 32, 1), ([513], [600], 7, 1, 64, 32, 1),
    ([256], [256], 5, 1, 128, 128, 0), ([700], [3], 1, 1, 64, 64, 2), ([2, 3], [77, 500], 130, 1, 64, 32, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ql,kl,hq,hk,D,bs,chunk", WEIGH)
def test_key_weights(kc, dtype, ql, kl, hq, hk, D, bs, chunk):
    *args, w = weigh_inputs(len(ql) + D + sum(kl), ql, kl, hq, hk, D, bs, dtype, chunk)
    fresh = ints([max(0, n - m) for m, n in zip(ql, kl)])
    out = w.clone()
    got = kc.key_weights(*args, w, max(ql), max(kl), chunk, fresh_from=fresh, decay=0.75, out=out)
    assert got is out
    check_weights(got, oe.key_weights(*args, w, chunk, None, fresh, 0.75))
    # in place, everything adding to what it has; the same bits twice
    want = oe.key_weights(*args, w, chunk)
    first, second = w.clone(), w.clone()
    for x in (first, second):
        assert kc.key_weights(*args, x, max(ql), max(kl), chunk) is x
    check_weights(first, want)
    assert torch.equal(first, second)


@pytest.mark.parametrize("ql,kl", [([40, 0, 130], [70, 700, 131]), ([0, 0, 300], [10, 0, 2000]), ([0, 0], [300, 40])])
def test_key_weights_of_requests_without_queries(kc, ql, kl):
    """Their keys only age; so do all, where there is no query at all, whatever max_q says."""
    *args, w = weigh_inputs(6, ql, kl, 4, 2, 64, 64, torch.float16, 1)
    for most in (max(ql), 500):
        got = kc.key_weights(*args, w, most, max(kl), 1, decay=0.5, out=w.clone())
        check_weights(got, oe.key_weights(*args, w, 1, None, None, 0.5))


@pytest.mark.parametrize("ql,hint", [(2, 1), (2, 300000), (200, 1), (200, 300000)])
def test_key_weights_length_hint_is_only_a_hint(kc, ql, hint):
    *args, w = weigh_inputs(3, [ql], [3000], 2, 2, 64, 64, torch.float16, 1)
    want = oe.key_weights(*args, w, 1)
    check_weights(kc.key_weights(*args, w, ql, hint, 1), want)


@pytest.mark.parametrize("ql", [3, 150])
def test_key_weights_add_up(kc, ql):
    """Each row hands out a weight of 1: the keys' new weights sum to the number of rows."""
    q, codes, ks, table, cu, lens, lse, w = weigh_inputs(5, [ql, ql], [500, 900], 4, 2, 64, 64, torch.float16, 0)
    attn = torch.empty_like(lse)
    kc.cached_attention(q, codes, codes, ks, ks, table, cu, lens, ql, 900, 0, lse=attn)
    out = torch.zeros_like(w)
    kc.key_weights(q, codes, ks, table, cu, lens, attn, w, ql, 900, 0, decay=0.0, out=out)
    # the attention's log-sum-exp is off by up to 2e-4
    assert (out.sum((0, 2)).double() - 2 * 2 * ql).abs().max() <= 2 * 2 * ql * 3e-4


@pytest.mark.parametrize("ql", [4, 200])
def test_key_weights_masked_places_and_odd_rows(kc, ql):
    """NaN in hidden blocks' scales, in weights that start fresh, in queries without a finite lse; broadcast queries."""
    kl, bs, chunk = 320, 32, 64
    q, codes, ks, table, cu, lens, lse, w = weigh_inputs(7, [ql], [kl], 2, 2, 64, bs, torch.float16, chunk)
    fresh = ints([kl - 100])
    want = oe.key_weights(q, codes, ks, table, cu, lens, lse, w, chunk, None, fresh, 1.0)
    table = torch.cat([table, torch.full((1, 2), 2 ** 30, dtype=torch.int32, device="cuda")], 1)
    w2 = w.clone()
    places = torch.arange(kl - 100, kl, device="cuda")
    w2[table[0, places // bs].long(), :, places % bs] = math.nan
    out = w.clone()
    kc.key_weights(q, codes, ks, table, cu, lens, lse, w2, ql, kl, chunk, fresh_from=fresh, out=out)
    check_weights(out, want)
    # rows that count for nothing: -inf, +inf and NaN, with queries to match
    q2, lse2 = q.clone(), lse.clone()
    lse2[:, 0], lse2[0, 1], lse2[1, 2] = -math.inf, math.inf, math.nan
    q2[0], q2[1, 0], q2[2, 1] = math.inf, math.nan, -math.inf
    out = w.clone()
    kc.key_weights(q2, codes, ks, table, cu, lens, lse2, w, ql, kl, chunk, out=out)
    check_weights(out, oe.key_weights(q2, codes, ks, table[:, :-2], cu, lens, lse2, w, chunk))
    # the last chunk's scales poisoned: only its own keys notice
    last = table[0, (kl - chunk) // bs:kl // bs].long()
    ks2 = ks.clone()
    ks2[last] = math.nan
    lse3 = lse.clone()
    late = [i for i in range(ql) if ok.key_limit(i, ql, kl, chunk) > kl - chunk]
    lse3[:, late] = math.nan
    base, out = w.clone(), w.clone()
    kc.key_weights(q, codes, ks, table, cu, lens, lse3, w, ql, kl, chunk, out=base)
    kc.key_weights(q, codes, ks2, table, cu, lens, lse3, w, ql, kl, chunk, out=out)
    assert torch.equal(out, base) and torch.isfinite(out).all()
    # one query for all tokens, and tokens in reverse
    one = q[:1].expand(ql, -1, -1)
    lse1 = ok.cached_attention(one, codes, codes, ks, ks, table[:, :-2], cu, lens, chunk)[1].float()
    got = kc.key_weights(one, codes, ks, table, cu, lens, lse1, w, ql, kl, chunk, out=w.clone())
    check_weights(got, oe.key_weights(one, codes, ks, table[:, :-2], cu, lens, lse1, w, chunk))


def test_key_weights_strides_and_untouched_places(kc):
    ql, kl, hq, D = [3, 90], [100, 333], 4, 64
    q, codes, ks, table, cu, lens, lse, w = weigh_inputs(9, ql, kl, hq, 2, D, 64, torch.bfloat16, 1)
    T = sum(ql)
    qkv = torch.randn(T, 3 * hq * D, device="cuda").bfloat16()
    qs = qkv[:, hq * D:2 * hq * D].view(T, hq, D)
    qs.copy_(q)
    both = torch.empty(codes.shape[0], 2, *codes.shape[1:], dtype=torch.int8, device="cuda")
    both[:, 0] = codes
    out = torch.full_like(w, -5.0)
    kc.key_weights(qs, both[:, 0], ks, table, cu, lens, lse, w, 90, 333, 1, scale=0.2, out=out)
    used = torch.zeros_like(w, dtype=torch.bool)
    for b, n in enumerate(kl):
        j = torch.arange(n, device="cuda")
        used[table[b, j // 64].long(), :, j % 64] = True
    assert (out[~used] == -5).all()
    value, err = oe.key_weights(q, codes, ks, table, cu, lens, lse, w, 1, 0.2)
    assert ((out.double() - value).abs() <= err)[used].all()


def test_key_weights_reports_bad_blocks_and_lengths(kc):
    from qvggt_b200 import _lib
    for ql in ([2, 3], [140, 3]):
        q, codes, ks, table, cu, lens, lse, w = weigh_inputs(8, ql, [100, 90], 2, 2, 64, 32, torch.float16, 0)
        good = kc.key_weights(q, codes, ks, table, cu, lens, lse, w, max(ql), 100, 0, out=w.clone())
        assert _lib.device_status() == 0
        bad = table.clone()
        bad[0, 1] = codes.shape[0]
        got = kc.key_weights(q, codes, ks, bad, cu, lens, lse, w, max(ql), 100, 0, out=w.clone())
        assert _lib.device_status(clear=True) == 0x201
        skipped = int(table[0, 1])
        assert torch.equal(got[skipped], w[skipped])
        rest = [i for i in range(codes.shape[0]) if i != skipped]
        assert torch.equal(got[rest], good[rest])
        second = table[1, :3].long()
        for wrong in (ints([100000, 90]), ints([-3, 90])):
            got = kc.key_weights(q, codes, ks, table, cu, wrong, lse, w, max(ql), 100, 0, out=w.clone())
            assert _lib.device_status(clear=True) == 0x202
            assert torch.equal(got[second], good[second]) and torch.equal(got[table[0, :4].long()], w[table[0, :4].long()])
        kc.key_weights(q, codes, ks, table, ints([0, ql[0], 999]), lens, lse, w, max(ql), 100, 0, out=w.clone())
        assert _lib.device_status(clear=True) == 0x202


# ----------------------------------------------------------------------- choice
def run_choice(kc, w, table, lens, keep, sink, recent, m, hint=0):
    dev = torch.tensor(w, device="cuda"), torch.tensor(table, device="cuda"), ints(lens), ints(keep)
    p = kc.evict_plan(*dev, sink, recent, m, hint)
    return tuple(t.cpu().numpy() for t in p)


def check_choice(kc, w, table, lens, keep, sink, recent, m=None, hint=0):
    m = max([min(k, n - k) for n, k in zip(lens, keep) if 0 <= k < n] + [0]) if m is None else m
    want = oe.evict_plan(w, table, lens, keep, sink, recent, m)
    for _ in range(2):
        for got, ref in zip(run_choice(kc, w, table, lens, keep, sink, recent, m, hint), want):
            assert (got == ref).all()


@pytest.mark.parametrize("layers,H,bs,lens,part,sink,recent,hint", [
    (1, 1, 32, [1], 0.0, 0, 0, 0), (1, 1, 32, [2], 0.5, 0, 0, 0), (2, 3, 64, [100, 0, 65, 1], 0.5, 0, 0, 0),
    (1, 2, 128, [700, 33], 0.75, 5, 9, 0), (3, 16, 32, [333], 0.97, 40, 30, 0), (1, 1, 64, [5000], 0.5, 0, 0, 0),
    (1, 2, 64, [3000, 17, 2500], 0.9, 1374, 700, 0), (1, 1, 32, [20001], 0.3, 3, 1, 0), (1, 1, 32, [20001], 0.3, 3, 1, 64),
    (1, 1, 128, [9000], 0.5, 10 ** 9, 0, 0), (1, 1, 128, [900], 0.5, 7, 10 ** 9, 0), (1, 1, 64, [400], 0.0, 3, 3, 0),
    (40, 16, 32, [64], 0.5, 1, 1, 0)])
def test_evict_plan(kc, layers, H, bs, lens, part, sink, recent, hint):
    rng = np.random.default_rng(sum(lens) + bs)
    table, num = random_table(rng, lens, bs, wider=2)
    w = np.exp(rng.normal(0, 2, (layers, num, H, bs))).astype(np.float32)
    keep = [int(n * part) for n in lens]
    check_choice(kc, w, table, lens, keep, sink, recent, hint=hint)
    # equal weights, signs, and values that have no order
    few = rng.integers(0, 3, w.shape).astype(np.float32)
    check_choice(kc, few, table, lens, keep, sink, recent, hint=hint)
    check_choice(kc, np.zeros_like(w), table, lens, keep, sink, recent, hint=hint)
    odd = rng.choice(np.array([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3.4028235e38, -1.0, 2.0], np.float32),
                     w.shape)
    check_choice(kc, odd, table, lens, keep, sink, recent, hint=hint)


@pytest.mark.parametrize("n,bs", [(1, 32), (3, 32), (4095, 32), (4097, 64), (16383, 128), (16384, 32), (16387, 64), (45056, 128),
                                  (45059, 32), (49152, 64), (49153, 64), (65541, 128)])
def test_evict_plan_borders_between_lanes(kc, n, bs):
    """Lengths about a multiple of what a thread, a CTA or its shared memory takes, with `sink`, `recent` and `keep` that end
    inside a quad of positions, on its edge, and past one another; weights all different, and of five values."""
    rng = np.random.default_rng(n)
    table, num = random_table(rng, [n], bs)
    w = rng.permutation(num * bs).astype(np.float32).reshape(1, num, 1, bs) - num
    few = rng.integers(0, 5, w.shape).astype(np.float32)
    for sink, recent, keep in ((0, 0, n // 2), (5, 7, n - 1), (n // 3 + 1, n // 4, n * 3 // 4), (n // 2, n, n - n // 5),
                               (1, 1, min(n, 2)), (2, 1, min(n - 1, 6)), (0, n // 2, n // 3), (n, 0, n // 7 + 1)):
        if keep >= n:
            continue
        check_choice(kc, w, table, [n], [keep], sink, recent)
        check_choice(kc, few, table, [n], [keep], sink, recent)


def test_evict_plan_longer_than_shared_memory(kc):
    """More keys than four CTAs hold: they are read again for each digit."""
    rng = np.random.default_rng(1)
    n, bs = 500000, 128
    table, num = random_table(rng, [n], bs)
    w = np.exp(rng.normal(0, 1, (1, num, 1, bs))).astype(np.float32)
    w[rng.random(w.shape) < 0.3] = 0
    for keep in (n // 2, n - 1, 1, n - n // 5):
        check_choice(kc, w, table, [n], [keep], 100, 50)


def test_evict_plan_nothing_to_do_and_short_lists(kc):
    from qvggt_b200 import _lib
    rng = np.random.default_rng(2)
    table, num = random_table(rng, [100, 50, 80], 32)
    w = rng.random((2, num, 2, 32)).astype(np.float32)
    check_choice(kc, w, table, [100, 50, 80], [100, 70, 80], 0, 0, m=3)
    check_choice(kc, w, table, [100, 50, 80], [100, 50, 80], 0, 0, m=0)
    assert _lib.device_status() == 0
    # lists too short: what fits is there, and it is reported
    w[:] = np.arange(32)[None, None, None] + np.arange(num)[None, :, None, None]
    for got, ref in zip(run_choice(kc, w, table, [100, 50, 80], [50, 25, 40], 0, 0, 4),
                        oe.evict_plan(w, table, [100, 50, 80], [50, 25, 40], 0, 0, 4)):
        assert (got == ref).all()
    assert _lib.device_status(clear=True) == 0x202
    # lengths outside their range: no moves for them
    for bad in ([10 ** 6, 50, 80], [-1, 50, 80]):
        for got, ref in zip(run_choice(kc, w, table, bad, [50, 25, 40], 0, 0, 40),
                            oe.evict_plan(w, table, [0, 50, 80], [50, 25, 40], 0, 0, 40)):
            assert (got == ref).all()
        assert _lib.device_status(clear=True) == 0x202
    got = run_choice(kc, w, table, [100, 50, 80], [-5, 25, 40], 0, 0, 40)
    assert (got[2][:, 0] == 0).all() and _lib.device_status(clear=True) == 0x202
    # a block outside the cache: its tokens go first
    off = table.copy()
    off[0, 1] = num
    src, dst, counts = run_choice(kc, w, off, [100, 50, 80], [68, 50, 80], 0, 0, 32)
    assert (dst[:, 0, :, :32] == np.arange(32, 64)).all() and (src[:, 0, :, :32] == np.arange(68, 100)).all()
    assert _lib.device_status(clear=True) == 0x201


# ------------------------------------------------------------------------- move
def move_case(rng, layers, H, D, bs, lens, keep, m):
    table, num = random_table(rng, lens, bs, wider=1)
    codes = [rng.integers(-127, 128, (layers, num, H, bs, D)).astype(np.int8) for _ in range(2)]
    scales = [np.exp(rng.normal(-4, 1, (layers, num, H))).astype(np.float32) for _ in range(2)]
    w = np.exp(rng.normal(0, 2, (layers, num, H, bs))).astype(np.float32)
    return table, codes, scales, w, oe.evict_plan(w, table, lens, keep, 0, 2, m)


def run_move(kc, table, codes, scales, w, plan, keep, strided=False):
    k, v = (torch.tensor(a, device="cuda") for a in codes)
    if strided:                          # K and V of a block beside each other
        both = torch.stack([k, v], 2)
        k, v = both[:, :, 0], both[:, :, 1]
    dev = [k, v] + [torch.tensor(a, device="cuda") for a in scales] + [None if w is None else torch.tensor(w, device="cuda")]
    kc.kv_evict(*dev, torch.tensor(table, device="cuda"), ints(keep),
                kc.EvictPlan(*(torch.tensor(x, device="cuda") for x in plan)))
    return [None if t is None else t.cpu().numpy() for t in dev]


@pytest.mark.parametrize("layers,H,D,bs,lens,part", [
    (1, 1, 64, 32, [2], 0.5), (2, 3, 64, 64, [100, 0, 65, 1], 0.5), (1, 2, 128, 128, [700, 33], 0.75),
    (3, 4, 64, 32, [333], 0.9), (1, 1, 128, 64, [5000], 0.5), (1, 2, 64, 64, [3000, 17, 2500], 0.6),
    (2, 1, 64, 128, [4096, 128], 0.5), (1, 16, 128, 32, [200] * 5, 0.8)])
def test_kv_evict_is_bit_exact(kc, layers, H, D, bs, lens, part):
    rng = np.random.default_rng(sum(lens) + D)
    keep = [int(n * part) for n in lens]
    m = max(min(k, n - k) for n, k in zip(lens, keep)) + 2
    table, codes, scales, w, plan = move_case(rng, layers, H, D, bs, lens, keep, m)
    for strided in (False, True):
        got = run_move(kc, table, codes, scales, w, plan, keep, strided)
        want = [c.copy() for c in codes], [s.copy() for s in scales], w.copy()
        for c, s in zip(*want[:2]):
            oe.kv_evict(c, s, table, *plan)
        oe.evict_weights(want[2], table, *plan)
        for a, b in zip(got, [*want[0], *want[1], want[2]]):
            assert (a == b).all()
    # without weights: the same codes and scales
    for a, b in zip(run_move(kc, table, codes, scales, None, plan, keep)[:4], [*want[0], *want[1]]):
        assert (a == b).all()


def test_kv_evict_repeated_is_the_same(kc):
    """The moves carried out twice change nothing more: sources stay, and incoming rows fit the scales by then.  (But for
    blocks that take rows from the one that the new length falls into: its scale may have grown and rounded them.)"""
    rng = np.random.default_rng(3)
    lens, keep, bs = [900, 130], [500, 77], 64
    table, codes, scales, w, plan = move_case(rng, 2, 2, 64, bs, lens, keep, 400)
    once = run_move(kc, table, codes, scales, w, plan, keep)
    twice = run_move(kc, table, once[:2], once[2:4], once[4], plan, keep)
    same = np.ones(scales[0].shape, bool)
    for i in np.ndindex(*plan[2].shape):
        layer, b, h = i
        for s, d in zip(plan[0][i][:plan[2][i]], plan[1][i][:plan[2][i]]):
            if s // bs == keep[b] // bs:
                same[layer, table[b][d // bs], h] = False
    assert 0.5 < same.mean() < 1
    for a, b in zip(once, twice):
        assert (a[same] == b[same]).all()
    assert (once[4] == twice[4]).all()


def test_kv_evict_skips_and_reports_bad_moves(kc):
    from qvggt_b200 import _lib
    rng = np.random.default_rng(4)
    lens, keep = [300, 200], [150, 100]
    table, codes, scales, w, plan = move_case(rng, 1, 2, 64, 32, lens, keep, 150)
    src, dst, counts = (x.copy() for x in plan)
    spoiled = [x.copy() for x in plan]
    spoiled[0][0, 0, 0, 0] = 10 ** 6                 # a source past the table
    spoiled[0][0, 0, 1, 3] = 5                       # a source that does not go
    for pair, i in (((0, 0), 0), ((0, 1), 3)):       # what is left of the plan without them
        h = pair[1]
        n = counts[0, 0, h]
        src[0, 0, h, i:n - 1], dst[0, 0, h, i:n - 1] = src[0, 0, h, i + 1:n].copy(), dst[0, 0, h, i + 1:n].copy()
        counts[0, 0, h] -= 1
    got = run_move(kc, table, codes, scales, w, spoiled, keep)
    assert _lib.device_status(clear=True) == 0x202
    want = [c.copy() for c in codes], [s.copy() for s in scales], w.copy()
    for c, s in zip(*want[:2]):
        oe.kv_evict(c, s, table, src, dst, counts)
    oe.evict_weights(want[2], table, src, dst, counts)
    for a, b in zip(got, [*want[0], *want[1], want[2]]):
        assert (a == b).all()
    # a count past the lists, a negative length, a block outside the cache
    for change in ("count", "keep", "block"):
        p, k, t = [x.copy() for x in plan], list(keep), table.copy()
        if change == "count":
            p[2][0, 0] = 151
        elif change == "keep":
            k[0] = -1
        else:
            t[0, :] = -7
        got = run_move(kc, t, codes, scales, w, p, k)
        assert _lib.device_status(clear=True) == (0x201 if change == "block" else 0x202)
        mine = table[0][table[0] >= 0]
        assert all((a[:, mine] == b[:, mine]).all() for a, b in zip(got, [*codes, *scales, w]))


def test_kv_evict_reports_places_outside_and_takes_any_keep_without_moves(kc):
    """Destinations at or past the new length and before 0 are skipped and reported, also where they lie in no block below
    it or nothing stays; a request that holds no more than `keep` has no moves, however large `keep` is."""
    from qvggt_b200 import _lib
    rng = np.random.default_rng(6)
    lens, bs = [300, 200], 32
    for keep, ends in (([150, 100], [(0, -1)]), ([160, 100], [(-1, 290)]), ([150, 100], [(-1, 155)]),
                       ([160, 100], [(0, -1), (-1, 160)])):
        table, codes, scales, w, plan = move_case(rng, 1, 2, 64, bs, lens, keep, 150)
        spoiled, left = [x.copy() for x in plan], [x.copy() for x in plan]
        n = plan[2][0, 0, 1]
        lo, hi = 0, n
        for end, place in ends:
            spoiled[1][0, 0, 1, end % n] = place
            lo, hi = (1, hi) if end == 0 else (lo, n - 1)
        for x in left[:2]:
            x[0, 0, 1, :hi - lo] = x[0, 0, 1, lo:hi].copy()
        left[2][0, 0, 1] = hi - lo
        got = run_move(kc, table, codes, scales, w, spoiled, keep)
        assert _lib.device_status(clear=True) == 0x202
        for c, s in zip(codes, scales):
            oe.kv_evict(c, s, table, *left)
        oe.evict_weights(w, table, *left)
        for a, b in zip(got, [*codes, *scales, w]):
            assert (a == b).all()
    # nothing stays, but moves are asked for
    table, codes, scales, w, plan = move_case(rng, 1, 2, 64, bs, lens, [150, 100], 150)
    got = run_move(kc, table, codes, scales, w, plan, [0, 0])
    assert _lib.device_status(clear=True) == 0x202
    assert all((a == b).all() for a, b in zip(got, [*codes, *scales, w]))
    # far more than the tables hold: nothing moves, nothing is wrong
    keep = [2 ** 31 - 1, 100]
    table, codes, scales, w, plan = move_case(rng, 1, 2, 64, bs, lens, keep, 100)
    got = run_move(kc, table, codes, scales, w, plan, keep)
    assert _lib.device_status(clear=True) == 0
    for c, s in zip(codes, scales):
        oe.kv_evict(c, s, table, *plan)
    oe.evict_weights(w, table, *plan)
    assert all((a == b).all() for a, b in zip(got, [*codes, *scales, w]))


# --------------------------------------------------------------- streams, graphs
def test_another_stream_and_a_graph(kc):
    """Weights, choice and move on a side stream behind a slow kernel, and captured into two graphs replayed in turn."""
    ql, kl, keep, bs, H, D = [70], [900], [600], 64, 2, 64
    q, codes, ks, table, cu, lens, lse, w = weigh_inputs(12, ql, kl, H, H, D, bs, torch.float16, 1)
    m = 300

    def step(q, k, v, ks, vs, w):
        kc.key_weights(q, k[0], ks[0], table, cu, lens, lse, w[0], 70, 900, 1, decay=0.5)
        plan = kc.evict_plan(w, table, lens, ints_keep, 10, 20, m)
        kc.kv_evict(k, v, ks, vs, w, table, ints_keep, plan)
        return plan

    ints_keep = ints(keep)
    base = [q, codes[None].clone(), codes[None].flip(-1).contiguous(), ks[None].clone(), ks[None].clone() * 2, w[None].clone()]
    fresh = lambda: [t.clone() for t in base]
    ref = fresh()
    plan = step(*ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    late = fresh()
    torch.cuda.current_stream().synchronize()
    with torch.cuda.stream(s):
        qq = torch.zeros_like(q)
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            a = a @ a * 1e-3
        qq.copy_(late[0] + (a[0, 0] * 0).half().nan_to_num())
        other = step(qq, *late[1:])
    s.synchronize()
    for x, y in zip([*plan, *ref[1:]], [*other, *late[1:]]):
        assert torch.equal(x, y)
    states, graphs, plans = [fresh(), fresh()], [], []
    for st in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plans.append(step(*st))
        graphs.append(g)
    for st in states:
        for t, b in zip(st, base):
            t.copy_(b)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for st, p in zip(states, plans):
        for x, y in zip([*plan, *ref[1:]], [*p, *st[1:]]):
            assert torch.equal(x, y)


# -------------------------------------------------------------------- refusals
def test_refusals(kc):
    from qvggt_b200._lib import QvggtError
    q, codes, ks, table, cu, lens, lse, w = weigh_inputs(2, [4], [50], 4, 2, 64, 32, torch.float16, 0)
    args = [q, codes, ks, table, cu, lens, lse, w]

    def weigh(match, error, max_q=4, max_kv=50, chunk=0, **change):
        names = ["q", "codes", "ks", "table", "cu", "lens", "lse", "w"]
        rest = {k: v for k, v in change.items() if k not in names}
        with pytest.raises(error, match=match):
            kc.key_weights(*[change.get(n, a) for n, a in zip(names, args)], max_q, max_kv, chunk, **rest)

    weigh("float16", TypeError, q=q.float())
    weigh("head_dim", ValueError, q=q[..., :32])
    weigh("share", QvggtError, q=q[:, :3].contiguous(), lse=lse[:3].contiguous())
    weigh("lse", ValueError, lse=lse[:, :3])
    weigh("int8", TypeError, codes=codes.float())
    weigh("k_scale", ValueError, ks=ks[:, :1])
    weigh("weights", ValueError, w=w[:, :1])
    weigh("out", ValueError, out=w.double())
    weigh("fresh_from", ValueError, fresh_from=ints([1, 2]))
    weigh("decay", QvggtError, decay=1.5)
    weigh("decay", QvggtError, decay=math.nan)
    weigh("scale", QvggtError, scale=0.0)
    weigh("shape", QvggtError, chunk=-1)
    weigh("CUDA|devices", ValueError, lse=lse.cpu())
    weigh("aligned", QvggtError, q=torch.zeros(4 * 4 * 64 + 1, device="cuda").half()[1:].view(4, 4, 64))

    w4 = w[None]
    keep = ints([20])
    with pytest.raises(ValueError, match="weights"):
        kc.evict_plan(w, table, lens, keep, 0, 0, 10)
    with pytest.raises(ValueError, match="keep"):
        kc.evict_plan(w4, table, lens, ints([1, 2]), 0, 0, 10)
    with pytest.raises(ValueError, match="max_moves"):
        kc.evict_plan(w4, table, lens, keep, 0, 0, -1)
    with pytest.raises(QvggtError, match="shape"):
        kc.evict_plan(w4, table, lens, keep, -1, 0, 10)
    with pytest.raises(QvggtError, match="block_size"):
        kc.evict_plan(torch.zeros(1, 4, 2, 48, device="cuda"), table, lens, keep, 0, 0, 10)
    with pytest.raises(QvggtError, match="aligned"):
        kc.evict_plan(torch.zeros(w.numel() + 1, device="cuda")[1:].view(w4.shape), table, lens, keep, 0, 0, 10)
    plan = kc.evict_plan(w4, table, lens, keep, 0, 0, 30)
    k5, s3 = codes[None], ks[None]
    with pytest.raises(TypeError, match="int8"):
        kc.kv_evict(codes, codes, ks, ks, None, table, keep, plan)
    with pytest.raises(ValueError, match="strides"):
        kc.kv_evict(k5, k5.transpose(2, 3).contiguous().transpose(2, 3), s3, s3, None, table, keep, plan)
    with pytest.raises(ValueError, match="k_scale"):
        kc.kv_evict(k5, k5, s3, s3[..., :1], None, table, keep, plan)
    with pytest.raises(ValueError, match="weights"):
        kc.kv_evict(k5, k5, s3, s3, w4[:, :2].contiguous(), table, keep, plan)
    with pytest.raises(ValueError, match="src"):
        kc.kv_evict(k5, k5, s3, s3, w4, table, keep, kc.EvictPlan(plan.src[0], plan.dst[0], plan.counts))
    with pytest.raises(ValueError, match="counts"):
        kc.kv_evict(k5, k5, s3, s3, w4, table, keep, kc.EvictPlan(plan.src, plan.dst, plan.counts[..., :1].contiguous()))
    with pytest.raises(ValueError, match="CUDA|devices"):
        kc.kv_evict(k5, k5, s3, s3, w4, table, keep.cpu(), plan)
