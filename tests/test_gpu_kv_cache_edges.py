"""GPU: the streaming K/V cache operators where their numbers or their inputs leave the ordinary range."""
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


def _one_request(seed, ql, n, hq, hk, D, bs, dtype):
    """q and a cache of one request whose blocks are shuffled."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    nb = -(-n // bs)
    kcodes, vcodes = (torch.randint(-127, 128, (nb + 3, hk, bs, D), generator=g, device="cuda", dtype=torch.int8)
                      for _ in range(2))
    ks, vs = (torch.exp(0.7 * torch.randn(nb + 3, hk, generator=g, device="cuda")) / 80 for _ in range(2))
    q = torch.randn(ql, hq, D, generator=g, device="cuda").to(dtype)
    table = torch.randperm(nb + 3, generator=g, device="cuda")[None, :nb].to(torch.int32).contiguous()
    return q, kcodes, vcodes, ks, vs, table, ints([0, ql]), ints([n])


def _check(got, lse, ref, dtype, vmax, n):
    """As in test_gpu_kv_cache: output rounding; the weights' fp16 rounding 2^-11 and the scores' and exponentials'
    2^-13, of sum w |v|; weights under fp16's normal range, 2^-25 of the largest |v| for each key."""
    out, want_lse, mag = ref
    bound = U[dtype] * out.abs() * 1.01 + (2.0 ** -11 + 2.0 ** -13) * mag + n * 2.0 ** -25 * vmax + TINY[dtype]
    assert torch.isfinite(got).all() and torch.isfinite(lse).all()
    assert ((got.double() - out).abs() <= bound).all(), float(((got.double() - out).abs() / bound).max())
    assert ((lse.double() - want_lse).abs() <= 2e-4).all()


# --------------------------------------------------------------- tiny scores
@pytest.mark.parametrize("chunk", [0, 1])
@pytest.mark.parametrize("ql,n", [(1, 1), (1, 31), (1, 33), (3, 100), (16, 47), (140, 200)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -100])
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_and_keys_of_nothing(kc, dtype, size, D, ql, n, chunk):
    """Zero (or, in bf16, tiny) queries over keys stored with the smallest scale, a unit of 32 keys seen in part: every
    visible key weighs the same.  (fp16 holds no 2^-100: zeros again.)"""
    q, kcodes, vcodes, ks, vs, table, cu, lens = _one_request(D + n, ql, n, 2, 1, D, 32, dtype)
    q = (q.float() * size).to(dtype)
    if size == 0:
        kcodes.zero_()
    ks.fill_(2.0 ** -60)
    args = (q, kcodes, vcodes, ks, vs, table, cu, lens)
    lse = torch.empty(2, ql, device="cuda")
    got = kc.cached_attention(*args, ql, n, chunk, lse=lse)
    ref = ok.cached_attention(*args, chunk)
    none = torch.isinf(ref[1]).t()                # (a causal query before the first key)
    assert not none.any()
    _check(got, lse, ref, dtype, float(vs.max() * 127), n)


@pytest.mark.parametrize("ql,n", [(1, 17), (3, 100), (140, 200)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scale_as_small_as_it_may_be(kc, dtype, D, ql, n):
    """A scale near the smallest that is accepted: times a block's smallest scale it is no float any more, and every
    visible key weighs the same."""
    args = _one_request(D + ql, ql, n, 2, 1, D, 32, dtype)
    args[3].fill_(2.0 ** -60)
    lse = torch.empty(2, ql, device="cuda")
    got = kc.cached_attention(*args, ql, n, 1, scale=2e-30, lse=lse)
    _check(got, lse, ok.cached_attention(*args, 1, scale=2e-30), dtype, float(args[4].max() * 127), n)


@pytest.mark.parametrize("ql", [3, 150])
@pytest.mark.parametrize("D", [64, 128])
def test_value_scales_far_apart(kc, D, ql):
    """V scales 2^-60 and 2^20: the keys of the small ones weigh what their scores say."""
    args = _one_request(D, ql, 640, 2, 1, D, 32, torch.bfloat16)
    q, kcodes, vcodes, ks, vs, table, cu, lens = args
    vs.fill_(2.0 ** -60)
    vs[table[0, 3].long()] = 2.0 ** 20
    lse = torch.empty(2, ql, device="cuda")
    got = kc.cached_attention(*args, ql, 640, lse=lse)
    _check(got, lse, ok.cached_attention(*args), torch.bfloat16, 2.0 ** 27, 640)


# ------------------------------------------------------------------- plan
def _plan(kc, cached, target, table, ring, free, bs, max_new, guard=16):
    """block_plan with guard words on both sides of the ring and the table; checks them and that the call repeats."""
    def guarded(a):
        buf = torch.full((a.size + 2 * guard,), -77, dtype=torch.int32, device="cuda")
        buf[guard:guard + a.size] = torch.tensor(a.reshape(-1), device="cuda")
        return buf, buf[guard:guard + a.size].view(a.shape)
    (tb, t), (rb, r) = guarded(table), guarded(ring)
    c, g, f = ints(cached), ints(target), torch.tensor(free, dtype=torch.int64, device="cuda")
    outs = []
    for _ in range(2):
        p = kc.block_plan(c, g, t, r, f, bs, max_new)
        outs.append(dict(table=t.tolist(), ring=r.tolist(), slots=p.slots.tolist(), cu_new=p.cu_new.tolist(),
                         cu_blocks=p.cu_blocks.tolist(), lens=p.lens.tolist(), free_range=p.free_range.tolist(),
                         status=p.status.item()))
        for buf in (tb, rb):
            assert (buf[:guard] == -77).all() and (buf[-guard:] == -77).all()
    assert outs[0] == outs[1]
    return outs[0]


def _same(got, want):
    want = dict(want, table=want["table"].tolist(), ring=want["ring"].tolist())
    for key in want:
        assert got[key] == want[key], key


@pytest.mark.parametrize("cached,target,free,status", [
    ([64, 96, 96], [0, 0, 0], [2, 4], 5),        # eight blocks come back into a ring of four that has two free
    ([96, 96, 96], [0, 0, 0], [3, 5], 5),        # nine: the last would land behind the ring
    ([64, 64, 0], [32, 0, 0], [1, 3], 5),        # three into room for two: would overwrite a free one
    ([64, 0, 0], [0, 64, 0], [1, 3], 0),         # two back into room for two, two taken
    ([32, 0, 0], [64, 0, 0], [-3, 1], 5), ([32, 0, 0], [64, 0, 0], [3, 2], 5), ([32, 0, 0], [32, 0, 0], [3, 2], 5),
    ([32, 0, 0], [64, 64, 64], [0, 5], 5), ([32, 0, 0], [64, 64, 64], [2 ** 62, 2 ** 62 + 4], 1),
    ([32, 0, 0], [64, 64, 32], [2 ** 62 + 1, 2 ** 62 + 5], 0), ([64, 64, -1], [0, 0, 0], [0, 4], 3)])
def test_plan_refuses_lengths_and_ranges_that_do_not_fit_the_pool(kc, cached, target, free, status):
    """Stale lengths or a range out of order: all or nothing, and nothing outside the ring is touched."""
    table = np.array([[3, 2, 0], [1, 0, 3], [2, 1, 1]], np.int32)
    ring = np.arange(4, dtype=np.int32)
    want = ok.block_plan(cached, target, table, ring, free, 32, 200)
    assert want["status"] == status
    _same(_plan(kc, cached, target, table, ring, free, 32, 200), want)


@pytest.mark.parametrize("bs,wide,num,first", [(2 ** 20, 8, 2047, 0), (2 ** 24, 1, 127, 1)])
def test_plan_counts_more_tokens_than_32_bits_hold(kc, bs, wide, num, first):
    """512 requests of 2^23 new tokens each: 2^32 in all, far over max_new, which holds one of them."""
    B, most = 512, 2 ** 23
    table = torch.zeros(B, wide, dtype=torch.int32, device="cuda")
    ring = torch.arange(num, dtype=torch.int32, device="cuda")
    cached = torch.full((B,), first, dtype=torch.int32, device="cuda")
    free = torch.tensor([0, num], dtype=torch.int64, device="cuda")
    p = kc.block_plan(cached, cached + most, table, ring, free, bs, most)
    assert p.status.item() == 4
    assert (p.cu_new == 0).all() and (p.slots == -1).all() and torch.equal(p.lens, cached)
    p = kc.block_plan(cached[:1], cached[:1] + most, table[:1], ring, free, bs, most)      # one of them is served
    assert p.status.item() == 0 and p.cu_new.tolist() == [0, most] and torch.equal(p.lens, cached[:1] + most)
    want = first + torch.arange(most, device="cuda")       # blocks 0, 1, ... of the ring, or block 0 of the table
    assert torch.equal(p.slots.long(), want)


@pytest.mark.parametrize("cached,target,where,bad,lost", [
    ([10, 64], [40, 64], "ring", 4, range(22, 30)),          # taken: the second block's tokens have no slot
    ([10, 64], [40, 64], "table", -1, range(0, 22)),         # held: those that go into the first block
    ([10, 64], [20, 0], "table", 2 ** 27 + 1, range(0, 10)), # times 32 it wraps to the slot 32
    ([32, 64], [32, 0], "returned", 4, [])])                 # given back
def test_plan_reports_block_ids_outside_the_pool(kc, cached, target, where, bad, lost):
    from qvggt_b200 import _lib
    table, ring, free = np.array([[3, -1], [1, 0]], np.int32), np.array([2, 9, 9, 9], np.int32), [0, 1]
    if where == "ring":
        ring[0] = bad
    else:
        table[(0, 0) if where == "table" else (1, 1)] = bad
    want = ok.block_plan(cached, target, table, ring, free, 32, 40)
    want["slots"] = [-1 if i in lost else x for i, x in enumerate(want["slots"])]
    assert want["status"] == 0
    _same(_plan(kc, cached, target, table, ring, free, 32, 40), want)
    assert _lib.device_status(clear=True) == 0x201


# ------------------------------------------------------- lengths out of order
@pytest.mark.parametrize("ql", [3, 80])
def test_attention_reports_decreasing_query_starts(kc, ql):
    """A request with a negative number of queries is skipped and reported; its neighbours are served."""
    from qvggt_b200 import _lib
    q, kcodes, vcodes, ks, vs, table, _, _ = _one_request(3, 3 * ql, 90, 2, 2, 64, 32, torch.float16)
    three, lens = table.expand(3, -1).contiguous(), ints([90, 70, 50])
    args = (q, kcodes, vcodes, ks, vs, three)
    got = kc.cached_attention(*args, ints([0, ql, ql - 2, 2 * ql]), lens, ql + 2, 90)
    assert _lib.device_status(clear=True) == 0x202
    want = kc.cached_attention(*args, ints([0, ql, ql, 2 * ql]), lens, ql + 2, 90)
    assert _lib.device_status(clear=True) == 0
    assert torch.equal(got[:ql - 2], want[:ql - 2])       # rows [ql - 2, ql) belong to two requests here
    part = kc.cached_attention(*args, ints([0, 0, ql - 2, 2 * ql]), lens, ql + 2, 90)
    assert torch.equal(got[ql:2 * ql], part[ql:2 * ql])


@pytest.mark.parametrize("cached,cu_new,cu_blocks,served", [
    ([-1000, 0], [0, 2, 5], [0, 1, 2], 1), ([-2 ** 31, 0], [0, 2, 5], [0, 1, 2], 1),         # negative lengths
    ([2 ** 31 - 1, 0], [0, 2, 5], [0, 1, 2], 1), ([64, 0], [0, 2, 5], [0, 1, 2], 1),         # past the row's end
    ([0, 0], [0, 2, 5], [900, 901, 902], None), ([0, 0], [0, 2, 5], [40, 1, 2], 1),          # no such blocks
    ([0, 0], [0, 2, 5], [-2 ** 31, 1, 2], 1), ([0, 0], [5, 2, 0], [0, 1, 2], None),
    ([0, 0], [-9, -7, 5], [0, 1, 2], None), ([0, 0], [0, 2, 6], [0, 1, 2], 0)])              # no such rows
def test_append_reports_lengths_out_of_order(kc, cached, cu_new, cu_blocks, served):
    """Lengths and running sums that no plan gives: what they name is skipped and reported, the other request is served,
    and no other block is touched."""
    from qvggt_b200 import _lib
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = [np.full((6, 2, 32, 64), 7, np.int8) for _ in range(2)]
    scales = [np.ones((6, 2), np.float32) for _ in range(2)]
    dev = [torch.tensor(a, device="cuda") for a in codes + scales]
    kv = torch.randn(5, 2, 2, 64, generator=g, device="cuda").half()
    # the table stands between rows that name block 2
    table = ints([[2, 2], [1, 4], [3, 5], [2, 2]])[1:3]
    kc.kv_append(kv[:, 0], kv[:, 1], *dev, table, ints(cached), ints(cu_new), ints(cu_blocks), 4)
    assert _lib.device_status(clear=True) == 0x202
    for s in range(2):
        if served is not None:
            rows = kv[cu_new[served]:cu_new[served + 1], s].cpu()
            ok.append_f32(rows, codes[s], scales[s], [[1 + 2 * served]], [0], [0, len(rows)])
        assert (dev[s].cpu().numpy() == codes[s]).all() and (dev[2 + s].cpu().numpy() == scales[s]).all()


def test_append_reports_a_bound_that_is_too_small(kc):
    """max_units 1 where the new rows touch two blocks: the first is written, the loss of the second reported."""
    from qvggt_b200 import _lib
    codes = [torch.zeros(2, 1, 32, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.ones(2, 1, device="cuda") for _ in range(2)]
    x = torch.ones(40, 1, 64, device="cuda").half()
    args = (x, x, *codes, *scales, ints([[1, 0]]), ints([0]), ints([0, 40]), ints([0, 2]))
    kc.kv_append(*args, 1)
    assert _lib.device_status(clear=True) == 0x202
    assert all((c[1] == 127).all() and (c[0] == 0).all() for c in codes)
    kc.kv_append(*args, 2)
    assert _lib.device_status(clear=True) == 0
    assert all((c[1] == 127).all() and (c[0, :, :8] == 127).all() and (c[0, :, 8:] == 0).all() for c in codes)


# -------------------------------------------------------------------- strides
@pytest.mark.parametrize("ql", [3, 150])
@pytest.mark.parametrize("hq,hk,D", [(4, 4, 64), (6, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_takes_queries_in_any_order(kc, dtype, hq, hk, D, ql):
    """Heads outermost, a token stride that is no multiple of the head stride, one head or one token broadcast: what the
    same queries give densely (the broadcast ones within the bounds, as another kernel may serve them)."""
    n, T = 400, ql + 7
    q, *cache = _one_request(D + hq, T, n, hq, hk, D, 64, dtype)
    cu, lens = ints([7, T]), ints([n])            # the first rows are no request's
    args = (*cache[:5], cu, lens, ql, n, 1)
    want = kc.cached_attention(q, *args)[7:]
    outermost = q.transpose(0, 1).contiguous().transpose(0, 1)
    padded = torch.zeros(T, 3 * hq * D + 8, device="cuda", dtype=dtype)[:, 8 + hq * D:8 + 2 * hq * D].view(T, hq, D)
    spread = torch.zeros(T, hq, 3, D + 8, device="cuda", dtype=dtype)[:, :, 1, :D]
    out = torch.zeros(hq, T, D + 8, device="cuda", dtype=dtype).transpose(0, 1)[..., :D]
    for x in (outermost, padded.copy_(q), spread.copy_(q)):
        assert torch.equal(kc.cached_attention(x, *args)[7:], want)
        kc.cached_attention(x, *args, out=out)
        assert torch.equal(out[7:], want) and (out[:7] == 0).all()
    lse = torch.zeros(hq, T, device="cuda")
    for x in (q[:, 1:2].expand(-1, hq, -1), q[9:10].expand(T, -1, -1)):
        got = kc.cached_attention(x, *args, lse=lse)
        ref = ok.cached_attention(x, *cache[:5], cu, lens, 1)
        assert (lse[:, :7] == 0).all()
        _check(got[7:], lse[:, 7:], (ref[0][7:], ref[1][:, 7:], ref[2][7:]), dtype, float(cache[3].max() * 127), n)
