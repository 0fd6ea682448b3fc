"""GPU: attention over packed sequences against its 64-bit restatement.

Bound, element by element: the output's rounding, the weights' rounding to the inputs' type (and 2^-13 for scores and
exponentials) times sum w |v|, and for fp16 the weights' steps below its normal range: n keys, 2^-25 each of the largest |v|.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv_evict as oe

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
U = {t: torch.finfo(t).eps / 2 for t in DTYPES}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


@pytest.fixture(scope="module")
def kc():
    from qvggt_b200 import _lib, kv_cache
    _lib.device_status(clear=True)
    yield kv_cache
    assert _lib.device_status(clear=True) == 0


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(lens, start=0):
    return [start] + [start + int(x) for x in np.cumsum(lens)]


def inputs(seed, T, hq, hk, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (hq, hk, hk)]


def check(got, lse, ref, dtype, vmax, n):
    out, want_lse, mag = ref
    floor = n * 2.0 ** -25 * vmax if dtype is torch.float16 else 0.0
    bound = U[dtype] * out.abs() * 1.01 + (U[dtype] + 2.0 ** -13) * mag + floor + TINY[dtype]
    assert torch.isfinite(got).all()
    off = (got.double() - out).abs()
    assert (off <= bound).all(), float((off / bound).max())
    assert ((lse.double() - want_lse).abs() <= 2e-4).all()


CASES = [
    # lens, hq, hk, D, chunk
    ([1], 1, 1, 64, 0), ([1, 1, 1], 3, 1, 128, 1), ([5], 2, 2, 64, 1), ([60, 23, 1, 0, 7], 16, 16, 128, 1),
    ([128], 2, 2, 64, 1), ([129], 2, 2, 64, 0), ([255, 256, 257], 4, 2, 64, 1), ([64, 65, 63], 2, 1, 128, 1),
    ([700, 33], 14, 2, 128, 1), ([700, 33], 14, 2, 64, 5), ([300, 20, 411], 3, 1, 128, 7), ([274 * 3, 274], 2, 2, 64, 274),
    ([1374], 2, 2, 64, 0), ([2049], 1, 1, 64, 1), ([2049], 1, 1, 128, 0), ([3000, 10, 1500], 2, 2, 64, 1),
    ([2000, 1, 2748], 2, 1, 128, 1374), ([1] * 70, 4, 1, 64, 1), ([17 * i % 200 for i in range(40)], 4, 4, 64, 1),
    ([40, 3], 128, 1, 64, 1), ([130], 100, 1, 128, 1), ([513, 1200], 5, 1, 64, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hq,hk,D,chunk", CASES)
def test_prompt_attention(kc, dtype, lens, hq, hk, D, chunk):
    T = sum(lens)
    q, k, v = inputs(T + D, T, hq, hk, D, dtype)
    lse = torch.full((hq, T), 7.0, device="cuda")
    cu = cu_of(lens)
    got = kc.prompt_attention(q, k, v, ints(cu), max(lens), chunk, lse=lse)
    check(got, lse, oe.prompt_attention(q, k, v, cu, chunk), dtype, float(v.abs().max()), max(lens))
    # again, and without lse: the same bits
    assert torch.equal(kc.prompt_attention(q, k, v, ints(cu), max(lens), chunk), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hint,chunk", [([50], 100000, 1), ([3000, 20], 5000, 1), ([3000, 20], 3020, 64)])
def test_length_hint_and_rows_outside(kc, dtype, lens, hint, chunk):
    """max_len may be larger than needed; rows before and behind the sequences keep what they hold, and what they hold
    (NaN) reaches nobody."""
    T = 9 + sum(lens) + 300
    q, k, v = inputs(1, T, 2, 2, 64, dtype)
    cu = cu_of(lens, 9)
    want = oe.prompt_attention(q, k, v, cu, chunk)
    for t in (q, k, v):
        t[:9], t[cu[-1]:] = math.nan, math.nan
    out = torch.full_like(q, 3.0)
    lse = torch.full((2, T), 7.0, device="cuda")
    got = kc.prompt_attention(q, k, v, ints(cu), hint, chunk, out=out, lse=lse)
    assert got is out and (out[:9] == 3).all() and (out[cu[-1]:] == 3).all()
    assert (lse[:, :9] == 7).all() and (lse[:, cu[-1]:] == 7).all()
    inside = slice(9, cu[-1])
    check(got[inside], lse[:, inside], [want[0][inside], want[1][:, inside], want[2][inside]], dtype,
          float(v[inside].abs().max()), max(lens))


@pytest.mark.parametrize("D,hq,hk", [(64, 4, 2), (128, 2, 2), (64, 2, 1)])
def test_strides_scale_and_scratch(kc, D, hq, hk):
    lens, chunk, dtype = [1300, 77], 1, torch.bfloat16
    T = sum(lens)
    q, k, v = inputs(9, T, hq, hk, D, dtype)
    cu = cu_of(lens)
    qkv = torch.randn(T, hq + 2 * hk, D, device="cuda").to(dtype)
    qs, ks, vs = qkv.split([hq, hk, hk], 1)
    for a, b in zip((qs, ks, vs), (q, k, v)):
        a.copy_(b)
    wide = torch.zeros(hq, T, 2 * D, device="cuda").to(dtype)
    out = wide.transpose(0, 1)[..., D:]
    need = kc.prompt_scratch_bytes(T, hq, hk, 2, 1300, D)
    scratch = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    lse = torch.empty(hq, T, device="cuda")
    got = kc.prompt_attention(qs, ks, vs, ints(cu), 1300, chunk, scale=0.3, out=out, lse=lse, scratch=scratch)
    assert got is out and (wide[..., :D] == 0).all()
    check(got, lse, oe.prompt_attention(q, k, v, cu, chunk, 0.3), dtype, float(v.abs().max()), 1300)
    # heads outermost
    heads = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(kc.prompt_attention(*heads, ints(cu), 1300, chunk, scale=0.3), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,hq,hk", [(64, 2, 2), (64, 8, 2), (128, 2, 2), (128, 12, 4)])
@pytest.mark.parametrize("longest", [63, 64, 65, 128, 129])
def test_lengths_about_one_tile(kc, dtype, D, hq, hk, longest):
    """Tiles of 64 and of 128 keys, full and not, with NaN where a token does not look; both paths of the same rows."""
    lens = [longest, 1, longest // 2, longest - 1]
    T = sum(lens)
    q, k, v = inputs(longest + hq, T, hq, hk, D, dtype)
    cu = cu_of(lens)
    for chunk in (0, 1, 16):
        lse = torch.empty(hq, T, device="cuda")
        got = kc.prompt_attention(q, k, v, ints(cu), longest, chunk, lse=lse)
        want = oe.prompt_attention(q, k, v, cu, chunk)
        check(got, lse, want, dtype, float(v.abs().max()), longest)
        # a hint that asks for 128-key tiles
        check(kc.prompt_attention(q, k, v, ints(cu), 200, chunk, lse=lse), lse, want, dtype, float(v.abs().max()), longest)
        if chunk == 0:
            continue
        at = longest // 2 // chunk * chunk
        k2, v2 = k.clone(), v.clone()
        k2[at:longest], v2[at:longest] = math.nan, math.nan
        bad = kc.prompt_attention(q, k2, v2, ints(cu), longest, chunk)
        assert torch.equal(bad[:at], got[:at]) and torch.equal(bad[longest:], got[longest:])
        assert torch.isnan(bad[at:longest]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,chunk,n,hq", [(64, 40, 200, 2), (128, 1, 150, 1), (64, 1374, 2748, 1), (64, 64, 1500, 4),
                                          (128, 500, 1800, 2)])
def test_what_a_token_does_not_see(kc, dtype, D, chunk, n, hq):
    """NaN and infinities in later chunks and in the next sequence leave a token's bits as they are; the tokens that see
    them get NaN and infinities where 64-bit arithmetic has them."""
    lens = [n, 90]
    q, k, v = inputs(4, sum(lens), hq, 1, D, dtype)
    cu = ints(cu_of(lens))
    base_lse, lse = (torch.empty(hq, sum(lens), device="cuda") for _ in range(2))
    base = kc.prompt_attention(q, k, v, cu, n, chunk, lse=base_lse)
    at = (n // 2 + 3) // chunk * chunk + chunk // 3          # a token of a middle chunk
    first = at // chunk * chunk                              # whose chunk begins here
    v2 = v.clone()
    v2[at, 0, 3], v2[at, 0, D - 1], v2[at + 1, 0, 5] = math.nan, math.inf, -math.inf
    v2[min(n - 1, at + 2 * chunk + 1), 0, D - 1] = -math.inf
    v2[n:] = math.nan                                        # the next sequence
    k2, q2 = k.clone(), q.clone()
    k2[n:], q2[n:] = math.nan, math.nan
    got = kc.prompt_attention(q2, k2, v2, cu, n, chunk, lse=lse)
    assert torch.equal(got[:first], base[:first]) and torch.equal(lse[:, :n], base_lse[:, :n])
    ref = oe.prompt_attention(q2[:n], k2[:n], v2[:n], [0, n], chunk)[0]
    assert torch.equal(torch.isnan(got[:n]), torch.isnan(ref)) and torch.equal(torch.isinf(got[:n]), torch.isinf(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[:n][inf].double(), ref[inf])
    plain = torch.isfinite(ref)
    assert ((got[:n].double() - base[:n].double())[plain].abs() <= 2 * U[dtype] * base[:n].double()[plain].abs() + 2e-6).all()
    assert torch.isnan(got[n:]).all()
    # a key of NaN, one of infinities: rows that see it are NaN, the others as they were
    for x in (math.nan, math.inf):
        k3 = k.clone()
        k3[at, 0, 7] = x
        got = kc.prompt_attention(q, k3, v, cu, n, chunk, lse=lse)
        assert torch.equal(got[:first], base[:first]) and torch.equal(got[n:], base[n:])
        ref = oe.prompt_attention(q[:n], k3[:n], v[:n], [0, n], chunk)[0]
        assert torch.equal(torch.isnan(got[:n]), torch.isnan(ref))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,hq,chunk", [([40, 17], 1, 1), ([60, 3], 2, 16), ([100, 100, 100], 1, 1), ([200, 90], 4, 40),
                                           ([700, 60], 1, 274), ([1500, 90], 1, 64), ([2100, 700], 2, 1)])
def test_the_largest_values_that_a_token_does_not_see(kc, dtype, D, lens, hq, chunk):
    """The largest finite values of V in later chunks, in the next sequence and behind the last one leave a token's bits as
    they are: 2^-125 of them would be 8."""
    T, n = sum(lens), lens[0]
    q, k, v = inputs(T + D, T + 50, hq, 1, D, dtype)
    cu, big = ints(cu_of(lens)), torch.finfo(dtype).max
    base_lse, lse = (torch.zeros(hq, T + 50, device="cuda") for _ in range(2))
    base = kc.prompt_attention(q, k, v, cu, max(lens), chunk, out=torch.zeros_like(q), lse=base_lse)
    for at, end in ((T, T + 50), (n, T + 50), (n // 2 // chunk * chunk, n), (0, n)):
        v2 = v.clone()
        v2[at:end, :, ::2], v2[at:end, :, 1::2] = big, -big
        got = kc.prompt_attention(q, k, v2, cu, max(lens), chunk, out=torch.zeros_like(q), lse=lse)
        assert torch.equal(got[:at], base[:at]) and torch.equal(got[end:], base[end:]) and torch.equal(lse, base_lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,chunk", [(60, 0), (60, 1), (200, 0), (200, 1), (1300, 16)])
def test_weights_too_small_to_count(kc, dtype, D, n, chunk):
    """Keys that a token sees with weights under 2^-500, and the largest finite values of V: 0 in 64 bits too.  (They take
    no part in the bound's steps below fp16's normal range: what is under half such a step is 0.)"""
    q, k, v = inputs(n + D, n, 1, 1, D, dtype)
    q[..., 0], k[..., 0] = 8, 0
    most = float(v.abs().max())
    far, big = slice(5, None, 7), torch.finfo(dtype).max
    k[far, :, 0] = -600                  # times 8 log2(e) / sqrt(head_dim): -612 at least, the other dims give some +-10
    v[far, :, ::2], v[far, :, 1::2] = big, -big
    lse = torch.empty(1, n, device="cuda")
    got = kc.prompt_attention(q, k, v, ints([0, n]), n, chunk, lse=lse)
    check(got, lse, oe.prompt_attention(q, k, v, [0, n], chunk), dtype, most, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,lens", [(64, [50, 40]), (128, [50, 40]), (64, [200, 90]), (128, [200, 90]), (64, [1500, 90])])
def test_scores_of_any_size(kc, dtype, D, lens):
    """A row with scaled scores up to 2^27 (fp16) and 2^31 (bf16) is a mean of what it sees; above, where the weights' type
    may hold none of them, it is NaN, not 0.  Either way the other rows keep theirs."""
    T, n = sum(lens), lens[0]
    q, k, v = inputs(T, T, 1, 1, D, dtype)
    at, cu = n // 2, [0, n, T]
    want = kc.prompt_attention(q, k, v, ints(cu), max(lens), 1)
    for x, ok in ((2048 if dtype is torch.float16 else 8192, True), (60000, False)):
        # 64 2048^2 log2(e) / 8 = 2^25.5, 64 8192^2 log2(e) / 8 = 2^29.5, half a power more with 128; 60000: over 2^35
        q[at:n], k[at:n] = x, x
        lse = torch.zeros(1, T, device="cuda")
        got = kc.prompt_attention(q, k, v, ints(cu), max(lens), 1, lse=lse)
        assert torch.equal(got[:at], want[:at]) and torch.equal(got[n:], want[n:]) and torch.isfinite(got[:at]).all()
        if not ok:
            assert torch.isnan(got[at:n]).all() and torch.isnan(lse[0, at:n]).all()
            continue
        ref = oe.prompt_attention(q, k, v, cu, 1)
        # log-sum-exps of some 10^7 to 10^9: five roundings (scale, maximum, sum, ln 2 and the product), 2^-24 each
        lse, far = lse.double(), ref[1][0, at:n]
        assert ((lse[0, at:n] - far).abs() <= 2.0 ** -21 * far.abs()).all()
        lse[0, at:n] = far
        near = got.clone()
        if n > 1024:
            # Items are cut, and the parts joined by log-sum-exps that fp32 holds to 2 and more at this size: any mean of
            # what a row sees among the large scores, whose rows weigh the same, may be the result.
            low, high = (f(v[at:n], 0).values for f in (torch.cummin, torch.cummax))
            step = 2 * U[dtype] * v.abs().max()
            assert (got[at:n] >= low - step).all() and (got[at:n] <= high + step).all()
            near[at:n] = ref[0][at:n].to(dtype)
        check(near, lse, ref, dtype, float(v.abs().max()), n)


def test_one_token_of_any_stride_and_out_in_place_of_q(kc):
    """The stride of an axis of length one means nothing; the result may take the queries' place."""
    for T, hq, hk in ((1, 4, 2), (1, 1, 1), (300, 1, 1)):
        q, k, v = inputs(6, T, hq, hk, 64, torch.float16)
        want = kc.prompt_attention(q, k, v, ints([0, T]), T, 1)
        odd = [t.as_strided(t.shape, (t.stride(0) if T > 1 else 3, t.stride(1) if t.shape[1] > 1 else 5, 1)) for t in (q, k, v)]
        assert torch.equal(kc.prompt_attention(*odd, ints([0, T]), T, 1), want)
    q, k, v = inputs(7, 3000, 4, 2, 64, torch.float16)
    want = kc.prompt_attention(q, k, v, ints([0, 2900, 3000]), 2900, 1)
    assert kc.prompt_attention(q, k, v, ints([0, 2900, 3000]), 2900, 1, out=q) is q and torch.equal(q, want)


def test_bad_sequences_are_skipped_and_reported(kc):
    from qvggt_b200 import _lib
    q, k, v = inputs(8, 300, 2, 2, 64, torch.float16)
    good = kc.prompt_attention(q, k, v, ints([0, 100, 300]), 200, 1)
    assert _lib.device_status() == 0
    for cu, served in [([0, 100, 301], slice(0, 100)), ([-1, 100, 300], slice(100, 300)), ([100, 0, 200], None)]:
        out = torch.full_like(q, 3.0)
        kc.prompt_attention(q, k, v, ints(cu), 200, 1, out=out)
        assert _lib.device_status(clear=True) == 0x202
        if served is not None:
            assert torch.equal(out[served], good[served])
    out = torch.full_like(q, 3.0)
    kc.prompt_attention(q, k, v, ints([0, 100, 300]), 150, 1, out=out)        # longer than max_len
    assert _lib.device_status(clear=True) == 0x202
    assert torch.equal(out[:100], good[:100]) and (out[100:] == 3).all()


def test_rows_past_two_gib(kc):
    """Rows that start beyond 2^31 elements, in every tensor."""
    n, H, D = 600, 1, 64
    stride = 2 ** 32 // n // 64 * 64
    big = torch.zeros(n * stride, dtype=torch.float16, device="cuda")
    q, k, v, out = (big[i * 64:].as_strided((n, H, D), (stride, D, 1)) for i in range(4))
    small = inputs(3, n, H, H, D, torch.float16)
    for a, b in zip((q, k, v), small):
        a.copy_(b)
    for chunk in (0, 1):
        got = kc.prompt_attention(q, k, v, ints([0, n]), n, chunk, out=out)
        assert torch.equal(got, kc.prompt_attention(*small, ints([0, n]), n, chunk))


def test_streams_and_graphs(kc):
    lens = [1100, 300]
    T = sum(lens)
    q, k, v = inputs(5, T, 4, 2, 64, torch.float16)
    cu = ints(cu_of(lens))
    want = kc.prompt_attention(q, k, v, cu, 1100, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(q)
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            a = a @ a * 1e-3
        late.copy_(q + (a[0, 0] * 0).half().nan_to_num())
        got = kc.prompt_attention(late, k, v, cu, 1100, 1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graphs, outs, qs = [], [], [torch.zeros_like(q) for _ in range(2)]
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kc.prompt_attention(x, k, v, cu, 1100, 1))
        graphs.append(g)
    qs[0].copy_(q)
    qs[1].copy_(q.flip(0))
    flipped = kc.prompt_attention(qs[1], k, v, cu, 1100, 1)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], flipped)


def test_refusals(kc):
    from qvggt_b200._lib import QvggtError
    q, k, v = inputs(2, 10, 4, 2, 64, torch.float16)
    cu = ints([0, 10])
    call = kc.prompt_attention
    with pytest.raises(TypeError, match="float16"):
        call(q.float(), k, v, cu, 10)
    with pytest.raises(TypeError):
        call(q, k.bfloat16(), v, cu, 10)
    with pytest.raises(ValueError, match="kv_heads"):
        call(q, k[:9], v, cu, 10)
    with pytest.raises(ValueError, match="kv_heads"):
        call(q, k, v[:, :1], cu, 10)
    with pytest.raises(QvggtError, match="share"):
        call(q[:, :3].contiguous(), k, v, cu, 10)
    with pytest.raises(QvggtError, match="head_dim"):
        call(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), cu, 10)
    with pytest.raises(QvggtError, match="128 query heads"):
        call(torch.zeros(10, 129, 64, device="cuda").half(), k[:, :1], v[:, :1], cu, 10)
    with pytest.raises(TypeError, match="int32"):
        call(q, k, v, cu.long(), 10)
    with pytest.raises(ValueError, match="cu"):
        call(q, k, v, cu[:0], 10)
    with pytest.raises(QvggtError, match="aligned"):
        call(torch.zeros(10 * 4 * 64 + 1, device="cuda").half()[1:].view(10, 4, 64), k, v, cu, 10)
    with pytest.raises(QvggtError, match="strides"):
        call(q, k[:1].expand(10, 2, 64), v, cu, 10)
    with pytest.raises(QvggtError, match="scale"):
        call(q, k, v, cu, 10, scale=0.0)
    with pytest.raises(QvggtError, match="causal_chunk"):
        call(q, k, v, cu, 10, -1)
    with pytest.raises(ValueError, match="lse"):
        call(q, k, v, cu, 10, lse=torch.empty(4, 9, device="cuda"))
    with pytest.raises(ValueError, match="scratch"):
        big = inputs(2, 4000, 4, 2, 64, torch.float16)
        call(*big, ints([0, 4000]), 4000, scratch=torch.empty(1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="CUDA|devices"):
        call(q, k, v, cu.cpu(), 10)
    assert call(q[:0], k[:0], v[:0], ints([0]), 0).shape == (0, 4, 64)
