"""The operators of the streaming key/value cache, as cases to measure: multi-axis rotary positions, block tables and slot
maps, the 8-bit cache write, and attention over that cache.

A case is a dict of plain values; :func:`prepare` builds its inputs on the GPU from a seed, :func:`run` makes one pass and
returns every output, and :func:`exact` evaluates the definition in 64 bits.  With ``own`` false, ``run`` computes the plain
form (elementary torch operations in 32 bits, rounded once); with ``own`` true it calls ``qvggt_b200.kv_cache``.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
SCALE_MIN = 2.0 ** -60      # smallest scale of a cache block
P = 1374                    # tokens of one 518 x 518 frame: camera, 4 registers, 37 x 37 patches
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one frame entering the aggregator: the model's own 2-D positions, 16 heads x 64
        dict(name="rope_frame", op="rope", T=P, hq=16, hk=16, D=64, sections="16,16", layout="axial", dtype="fp16",
             inverse=False),
        # 32 frames with (time, height, width) positions, in the direction of the gradient, keys shared by 4 heads
        dict(name="rope_video_bf16", op="rope", T=32 * P, hq=16, hk=4, D=64, sections="8,12,12", layout="split",
             dtype="bf16", inverse=True),
        # eight streams, each getting one more frame
        dict(name="plan_frames", op="plan", B=8, cached=20000, new=P, shrink=False, bs=64),
        # a thousand requests of all lengths, a third of them ending or cut back, the others growing
        dict(name="plan_many", op="plan", B=1000, cached=3000, new=97, shrink=True, bs=32),
        # the camera token of 32 streams: one token each, into blocks that are partly filled
        dict(name="append_tokens", op="append", B=32, cached=500, new=1, H=16, D=128, bs=64, dtype="fp16"),
        # seven ragged requests in bf16 with few heads
        dict(name="append_ragged_bf16", op="append", B=7, cached=301, new=913, H=4, D=128, bs=32, dtype="bf16"),
        # 32 frames at once into an empty cache
        dict(name="append_frames", op="append", B=1, cached=0, new=32 * P, H=16, D=64, bs=64, dtype="fp16"),
        # the smallest call: one camera token over a short cache
        dict(name="attn_token_short", op="attn", B=1, q=1, L=300, hq=16, hk=16, D=128, bs=64, chunk=0, ragged=0.0,
             dtype="fp16"),
        # one token for each of eight streams over 32 frames
        dict(name="attn_token_long", op="attn", B=8, q=1, L=32 * P, hq=16, hk=16, D=64, bs=64, chunk=1, ragged=0.3,
             dtype="fp16"),
        # 16 ragged requests, four query heads to each key head, bf16
        dict(name="attn_shared_bf16", op="attn", B=16, q=3, L=9001, hq=32, hk=8, D=128, bs=32, chunk=1, ragged=0.9,
             dtype="bf16"),
        # one new frame over the 31 before it and itself
        dict(name="attn_frame", op="attn", B=1, q=P, L=32 * P, hq=16, hk=16, D=64, bs=64, chunk=P, ragged=0.0,
             dtype="fp16"),
        # eight frames at once, each seeing the frames up to its own
        dict(name="attn_frames", op="attn", B=1, q=8 * P, L=8 * P, hq=16, hk=16, D=64, bs=64, chunk=P, ragged=0.0,
             dtype="fp16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "plan", "append", "append", "attn", "attn", "attn"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rope":
        D = rng.choice([64, 128])
        hk = rng.choice([1, 2, 4, 8, 16])
        n = D // 2
        sections = rng.choice([[n], [n // 2, n - n // 2], [n // 4, (n - n // 4) // 2, n - n // 4 - (n - n // 4) // 2],
                               [n // 4, n // 4]])
        return dict(op="rope", T=_logint(rng, 1, 40000 * 64 // D), hq=16, hk=hk, D=D,
                    sections=",".join(str(s) for s in sections),
                    layout=rng.choice(["axial", "split", "interleaved"]), dtype=dtype, inverse=rng.random() < 0.5)
    if op == "plan":
        return dict(op="plan", B=_logint(rng, 1, 1000), cached=_logint(rng, 1, 3000), new=_logint(rng, 1, 97),
                    shrink=rng.random() < 0.5, bs=rng.choice([32, 64, 128]))
    H, D, bs = rng.choice([1, 4, 8, 16]), rng.choice([64, 128]), rng.choice([32, 64, 128])
    if op == "append":
        B = _logint(rng, 1, 64)
        return dict(op="append", B=B, cached=rng.choice([0, _logint(rng, 1, 4000)]),
                    new=_logint(rng, 1, max(2, 40000 * 64 // (D * B))), H=H, D=D, bs=bs, dtype=dtype)
    group = rng.choice([1, 1, 2, 4, 7])
    B = _logint(rng, 1, 16)
    q = rng.choice([1, _logint(rng, 1, 16), _logint(rng, 17, 1400)])
    if q * group <= 16:
        most = 32 * P * 16 * 64 * 8 // (H * D)
    else:      # no more products than the largest listed case has
        most = 25 * 10 ** 10 // (4 * q * group * H * D)
    B = max(1, min(B, most // q))
    while most < q:
        q, most = q // 2, most * 2
    L = _logint(rng, q, max(q + 1, min(32 * P, most // B)))
    return dict(op="attn", B=B, q=q, L=L, hq=H * group, hk=H, D=D, bs=bs, chunk=rng.choice([0, 1, _logint(rng, 2, P)]),
                ragged=rng.choice([0.0, 0.5, 0.95]), dtype=dtype)


# ------------------------------------------------------- what a case's sizes mean
def _fraction(i):
    return (i * 0.6180339887498949) % 1.0


def _attn_lens(c):
    """(query lengths, key lengths) of the requests: ragged ones are shorter by up to that share."""
    ql = [max(1, int(round(c["q"] * (1 - c["ragged"] * _fraction(3 * i))))) for i in range(c["B"])]
    kl = [max(1, int(round(c["L"] * (1 - c["ragged"] * _fraction(i))))) for i in range(c["B"])]
    return ql, kl


def _plan_lens(c):
    """(cached, target) lengths of the requests."""
    cached = [int(round(c["cached"] * _fraction(i + 1))) for i in range(c["B"])]
    target = []
    for i, n in enumerate(cached):
        if c["shrink"] and i % 3 == 1:
            target.append(0 if i % 2 else n // 2)
        elif c["shrink"]:
            target.append(n + int(round(c["new"] * _fraction(5 * i + 2))))
        else:
            target.append(n + c["new"])
    return cached, target


def _append_lens(c):
    cached = [int(round(c["cached"] * (1 - 0.5 * _fraction(i)))) for i in range(c["B"])]
    new = [max(1, int(round(c["new"] * (1 - 0.5 * _fraction(2 * i))))) for i in range(c["B"])]
    return cached, [a + b for a, b in zip(cached, new)]


def _ceil(a, b):
    return -(-a // b)


def _touched(cached, target, bs):
    return [(t - 1) // bs - c // bs + 1 if t > c else 0 for c, t in zip(cached, target)]


def _sum0(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _visible(ql, kl, chunk):
    """(query, key) pairs that the mask leaves, per head."""
    if not chunk:
        return sum(a * b for a, b in zip(ql, kl))
    return sum(min(k, max(0, ((k - q + i) // chunk + 1) * chunk)) for q, k in zip(ql, kl) for i in range(q))


def work(c):
    op = c["op"]
    if op == "rope":
        axes = len(c["sections"].split(","))
        n = c["T"] * (c["hq"] + c["hk"]) * c["D"]
        return {"bytes": 4 * n + 4 * axes * c["T"], "flops": 3 * n}
    if op == "plan":
        cached, target = _plan_lens(c)
        tokens = sum(max(0, t - n) for n, t in zip(cached, target))
        moved = sum(abs(_ceil(t, c["bs"]) - _ceil(n, c["bs"])) for n, t in zip(cached, target))
        # lengths in and out, the two prefix sums, a slot for each token, each moved block read and written
        return {"bytes": 4 * (5 * c["B"] + tokens) + 8 * moved, "flops": 0}
    if op == "append":
        cached, target = _append_lens(c)
        new = sum(target) - sum(cached)
        old = sum(n % c["bs"] for n in cached)
        row = c["H"] * c["D"] * 2
        # new rows in (2 bytes) and their codes out (1); earlier codes of touched blocks in; the values of both out (2)
        return {"bytes": row * (3 * new + old + 2 * (new + old)), "flops": 4 * row * new}
    ql, kl = _attn_lens(c)
    pairs = _visible(ql, kl, c["chunk"])
    blocks = sum(_ceil(k, c["bs"]) for k in kl)
    n = 4 * sum(ql) * c["hq"] * c["D"] + 2 * sum(kl) * c["hk"] * c["D"] + blocks * (8 * c["hk"] + 4)
    return {"bytes": n, "flops": 4 * pairs * c["hq"] * c["D"]}


# -------------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(g, lens, spare, H, D, bs):
    """A cache that holds `lens` tokens per request in shuffled blocks, with room for `spare` tokens more each: codes of
    normal values, a scale for each block and head; the table; the blocks no request holds."""
    need = [_ceil(n + s, bs) for n, s in zip(lens, spare)]
    have = [_ceil(n, bs) for n in lens]
    num = sum(need) + 5
    codes = [(torch.randn(num, H, bs, D, generator=g, device=DEV, dtype=torch.float16) * 34).round_()
             .clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp(0.4 * torch.randn(num, H, generator=g, device=DEV)) / 34 for _ in range(2)]
    order = torch.randperm(num, generator=g, device=DEV).to(torch.int32)
    start = _sum0(have)
    wide = max(max(need), 1)
    cols = torch.arange(wide, device=DEV)
    at = (torch.tensor(start[:-1], device=DEV)[:, None] + cols).clamp(max=num - 1)
    table = torch.where(cols < torch.tensor(have, device=DEV)[:, None], order[at], -1).to(torch.int32).contiguous()
    return codes, scales, table, order[start[-1]:].contiguous(), num


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = c["op"]
    if op == "rope":
        sections = [int(s) for s in c["sections"].split(",")]
        T, dt, pairs = c["T"], DTYPES[c["dtype"]], sum(sections)
        # frame number, row and column of each token, as a video has them, from a random first frame
        first = int(torch.randint(0, 200, (1,), generator=g, device=DEV))
        tok = torch.arange(T, device=DEV)
        axes = [tok // P + first, tok % P // 37, tok % 37, tok % P]
        pos = torch.stack(axes[-len(sections) - 1:-1] if len(sections) < 4 else axes).to(torch.int32).contiguous()
        # each axis has its own falling frequencies
        inv = torch.cat([100.0 ** (-torch.arange(n, device=DEV, dtype=torch.float32) / n) for n in sections])
        lo, hi, axis, base = [], [], [], 0
        for a, n in enumerate(sections):
            for j in range(n):
                i = base + j
                axis.append(a)
                lo.append({"axial": 2 * base + j, "split": i, "interleaved": 2 * i}[c["layout"]])
                hi.append({"axial": 2 * base + n + j, "split": i + pairs, "interleaved": 2 * i + 1}[c["layout"]])
            base += n
        # q and k as column ranges of one projection's output
        qk = torch.randn(T, c["hq"] + c["hk"], c["D"], generator=g, device=DEV).to(dt)
        return dict(op=op, q=qk[:, :c["hq"]], k=qk[:, c["hq"]:], positions=pos, inv_freq=inv, sections=tuple(sections),
                    layout=c["layout"], inverse=c["inverse"], lo=torch.tensor(lo, device=DEV),
                    hi=torch.tensor(hi, device=DEV), axis=torch.tensor(axis, device=DEV))
    if op == "plan":
        cached, target = _plan_lens(c)
        bs = c["bs"]
        have, need = [_ceil(n, bs) for n in cached], [_ceil(n, bs) for n in target]
        num = sum(max(a, b) for a, b in zip(have, need)) + 7
        wide = max(max(have), max(need))
        order = torch.randperm(num, generator=g, device=DEV).to(torch.int32)
        start = torch.tensor(_sum0(have)[:-1], device=DEV)
        cols = torch.arange(wide, device=DEV)
        held = torch.tensor(have, device=DEV)
        table = torch.where(cols < held[:, None], order[(start[:, None] + cols).clamp(max=num - 1)], -1)
        # the free blocks stand in a ring, from a place that wraps around its end
        free = num - sum(have)
        head = num * 3 + num - 1 - int(torch.randint(0, free, (1,), generator=g, device=DEV))
        ring = torch.full((num,), -1, dtype=torch.int32, device=DEV)
        ring[(head + torch.arange(free, device=DEV)) % num] = order[sum(have):]
        return dict(op=op, cached=_ints(cached), target=_ints(target), table=table.to(torch.int32).contiguous(),
                    ring=ring, free=torch.tensor([head, head + free], dtype=torch.int64, device=DEV), bs=bs,
                    most=sum(max(0, t - n) for n, t in zip(cached, target)))
    dt, H, D, bs = DTYPES[c["dtype"]], c.get("H", c.get("hk")), c["D"], c["bs"]
    if op == "append":
        cached, target = _append_lens(c)
        codes, scales, table, rest, num = _cache(g, cached, [t - n for n, t in zip(cached, target)], H, D, bs)
        # every request's new blocks are in its table already
        have, need = [_ceil(n, bs) for n in cached], [_ceil(n, bs) for n in target]
        more = torch.tensor(_sum0([b - a for a, b in zip(have, need)])[:-1], device=DEV)
        cols = torch.arange(table.shape[1], device=DEV)
        held, full = torch.tensor(have, device=DEV)[:, None], torch.tensor(need, device=DEV)[:, None]
        at = (more[:, None] + cols - held).clamp(0, max(0, rest.numel() - 1))
        table = torch.where((cols >= held) & (cols < full), rest[at], table).to(torch.int32).contiguous()
        T = sum(target) - sum(cached)
        # K and V as column ranges of one projection's output; tokens differ in size
        kv = torch.randn(T, 2, H, D, generator=g, device=DEV)
        kv = (kv * torch.exp(0.5 * torch.randn(T, 1, H, 1, generator=g, device=DEV))).to(dt)
        # the slots of every token in the blocks that are written, earlier tokens among them
        ids = [(b, j) for b, (n, t) in enumerate(zip(cached, target)) for j in (n // bs * bs, t)]
        first = torch.tensor([j for _, j in ids[::2]], device=DEV)
        last = torch.tensor([j for _, j in ids[1::2]], device=DEV)
        b = torch.repeat_interleave(torch.arange(len(cached), device=DEV), last - first)
        j = torch.arange(b.numel(), device=DEV) - torch.tensor(_sum0((last - first).tolist())[:-1], device=DEV)[b] + first[b]
        slots = (table[b, j // bs].long() * bs + j % bs).to(torch.int32)
        return dict(op=op, k=kv[:, 0], v=kv[:, 1], kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1], table=table,
                    cached=_ints(cached), cu_new=_ints(_sum0([t - n for n, t in zip(cached, target)])),
                    cu_blocks=_ints(_sum0(_touched(cached, target, bs))), units=sum(_touched(cached, target, bs)),
                    slots=slots, bs=bs)
    ql, kl = _attn_lens(c)
    codes, scales, table, _, num = _cache(g, kl, [0] * len(kl), H, D, bs)
    q = torch.randn(sum(ql), c["hq"], D, generator=g, device=DEV).to(dt)
    # a few queries look for one key, so that their weights are sharp
    q[::5] *= 3
    return dict(op=op, q=q, kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1], table=table, cu_q=_ints(_sum0(ql)),
                kv_lens=_ints(kl), max_q=max(ql), max_kv=max(kl), chunk=c["chunk"], bs=bs)


# --------------------------------------------------------------- plain forms
def _plain_rope(s):
    ang = s["positions"][s["axis"]].t().float() * s["inv_freq"]
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    if s["inverse"]:
        sin = -sin

    def turn(x):
        y = x.float()
        a, b = y[..., s["lo"]], y[..., s["hi"]]
        y = y.clone()
        y[..., s["lo"]] = a * cos - b * sin
        y[..., s["hi"]] = b * cos + a * sin
        return y.to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _cumsum0(x):
    return torch.nn.functional.pad(x.cumsum(0), (1, 0)).to(torch.int32)


def _plain_plan(s):
    bs, ring, table, most = s["bs"], s["ring"], s["table"], s["most"]
    cached, target = s["cached"].long(), s["target"].long()
    N, (B, wide) = ring.numel(), table.shape
    head, tail = s["free"][0], s["free"][1]
    have, need = (cached + bs - 1) // bs, (target + bs - 1) // bs
    enough = (need - have).clamp(min=0).sum() <= tail - head
    fits = need.max() <= wide
    status = torch.where(fits, torch.where(enough, 0, 1), 2).to(torch.int32)
    target = torch.where(enough & fits, target, cached)
    need = (target + bs - 1) // bs
    grow, drop = (need - have).clamp(min=0), (have - need).clamp(min=0)
    first, freed = _cumsum0(grow).long(), _cumsum0(drop).long()
    cols = torch.arange(wide, device=table.device)
    new = (cols >= have[:, None]) & (cols < need[:, None])
    at = (head + first[:-1, None] + cols - have[:, None]) % N
    back = (cols >= need[:, None]) & (cols < have[:, None])
    to = torch.where(back, (tail + freed[:-1, None] + cols - need[:, None]) % N, N)
    ring = torch.nn.functional.pad(ring, (0, 1)).scatter(0, to.reshape(-1), table.reshape(-1))[:N]
    table = torch.where(new, s["ring"][at], table)
    count = (target - cached).clamp(min=0)
    cu_new = _cumsum0(count)
    n = torch.arange(most, device=table.device)
    b = torch.searchsorted(cu_new[1:].long(), n, right=True).clamp(max=B - 1)
    pos = cached[b] + n - cu_new[b]
    slots = table[b, (pos // bs).clamp(max=wide - 1)].long() * bs + pos % bs
    slots = torch.where(n < cu_new[-1], slots, -1).to(torch.int32)
    touched = torch.where(count > 0, (target - 1) // bs - cached // bs + 1, 0)
    free = torch.stack([head + first[-1], tail + freed[-1]])
    return table, ring, slots, cu_new, _cumsum0(touched), target.to(torch.int32), free, status.reshape(1)


def _plain_append(s):
    bs, T = s["bs"], s["k"].shape[0]
    cached, cu_new, cu_blocks = s["cached"].long(), s["cu_new"].long(), s["cu_blocks"].long()
    n = torch.arange(T, device=cached.device)
    b = torch.searchsorted(cu_new[1:], n, right=True)
    pos = cached[b] + n - cu_new[b]
    unit = cu_blocks[b] + pos // bs - cached[b] // bs
    block = s["table"][b, pos // bs].long()
    u = torch.arange(s["units"], device=cached.device)
    ub = torch.searchsorted(cu_blocks[1:], u, right=True)
    ublock = s["table"][ub, cached[ub] // bs + u - cu_blocks[ub]].long()
    older = torch.where(u == cu_blocks[ub], cached[ub] % bs, 0)      # earlier tokens in the block
    outs = []
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.float()
        a = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        most = torch.zeros(s["units"], x.shape[1], device=x.device)
        most.scatter_reduce_(0, unit[:, None].expand_as(a), a, "amax")
        before = torch.where(older[:, None] > 0, scales[ublock], 0.0)
        new = torch.maximum(torch.maximum(before, most / 127.0), torch.full_like(most, SCALE_MIN))
        inv = 1.0 / new
        # earlier codes of the block move to its new scale
        kept = (codes[ublock].float() * (before * inv)[..., None, None]).round().clamp(-127, 127).to(torch.int8)
        live = torch.arange(bs, device=x.device)[None, None, :, None] < older[:, None, None, None]
        codes[ublock] = torch.where(live, kept, codes[ublock])
        scales[ublock] = new
        c = (x * inv[unit][..., None]).round().clamp(-127, 127)
        codes[block, :, pos % bs] = torch.where(c.isnan(), 0.0, c).to(torch.int8)
        at = s["slots"].long()
        outs.append((codes[at // bs, :, at % bs].float() * scales[at // bs][..., None]).to(s["k"].dtype))
    return torch.stack(outs, 1).reshape(s["slots"].numel(), -1), s["ks"], s["vs"]


def _plain_attn(s):
    q, table, cu, kl, bs = s["q"], s["table"].long().clamp(min=0), s["cu_q"].long(), s["kv_lens"].long(), s["bs"]
    T, hq, D = q.shape
    B, nb = table.shape
    H = s["kc"].shape[1]
    dev = q.device

    def rows(codes, scales):
        x = codes[table].float() * scales[table][..., None, None]        # [B, nb, H, bs, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, H, 1, nb * bs, D)

    i = torch.arange(s["max_q"], device=dev)
    ql = cu[1:] - cu[:-1]
    qp = q[(cu[:-1, None] + i).clamp(max=T - 1)].float()                 # [B, max_q, hq, D]
    qp = qp.reshape(B, -1, H, hq // H, D).permute(0, 2, 3, 1, 4)
    S = (qp @ rows(s["kc"], s["ks"]).transpose(-1, -2)) * (1.0 / math.sqrt(D))
    pos = (kl - ql)[:, None] + i
    most = kl[:, None].expand(-1, s["max_q"])
    if s["chunk"]:
        most = torch.minimum(most, (torch.div(pos, s["chunk"], rounding_mode="floor") + 1) * s["chunk"])
    hidden = torch.arange(nb * bs, device=dev) >= most[..., None]        # [B, max_q, keys]
    S.masked_fill_(hidden[:, None, None], -math.inf)
    m = S.amax(-1, keepdim=True).clamp(min=-1e30)
    p = S.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p @ rows(s["vc"], s["vs"])) / l.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], hq, D)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu[1:], t, right=True)
    return o[b, t - cu[b]].to(q.dtype)


def run(state):
    s = state
    if not own:
        return {"rope": _plain_rope, "plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[s["op"]](s)
    from qvggt_b200 import kv_cache
    if s["op"] == "rope":
        return kv_cache.rope_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], layout=s["layout"],
                                  inverse=s["inverse"])
    if s["op"] == "plan":
        p = kv_cache.block_plan(s["cached"], s["target"], s["table"], s["ring"], s["free"], s["bs"], s["most"])
        return s["table"], s["ring"], p.slots, p.cu_new, p.cu_blocks, p.lens, p.free_range, p.status
    if s["op"] == "append":
        kv_cache.kv_append(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["cached"], s["cu_new"],
                           s["cu_blocks"], s["units"])
        return kv_cache.kv_gather(s["kc"], s["vc"], s["ks"], s["vs"], s["slots"], s["k"].dtype), s["ks"], s["vs"]
    return kv_cache.cached_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["cu_q"], s["kv_lens"],
                                     s["max_q"], s["max_kv"], causal_chunk=s["chunk"])


# ------------------------------------------------------ definitions in 64 bits
def _exact_rope(s):
    out = []
    for x in (s["q"], s["k"]):
        z = x.double().clone()
        for j, (lo, hi, a) in enumerate(zip(s["lo"].tolist(), s["hi"].tolist(), s["axis"].tolist())):
            t = s["positions"][a].double() * s["inv_freq"][j].double() * (-1 if s["inverse"] else 1)
            w = torch.complex(x[..., lo].double(), x[..., hi].double()) * torch.polar(torch.ones_like(t), t)[:, None]
            z[..., lo], z[..., hi] = w.real, w.imag
        out.append(z)
    return tuple(out)


def _exact_append(s):
    bs, dt = s["bs"], torch.float64
    cached, cu, table = s["cached"].tolist(), s["cu_new"].tolist(), s["table"].tolist()
    res, scales_out = [], []
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        codes, scales = codes.to(dt), scales.to(dt)
        for b, n in enumerate(cached):
            end = n + cu[b + 1] - cu[b]
            for j in range(n // bs, _ceil(end, bs)):
                lo, hi = max(n, j * bs), min(end, (j + 1) * bs)
                if lo >= hi:
                    continue
                blk, old = table[b][j], max(0, n - j * bs)
                rows = x[cu[b] + lo - n:cu[b] + hi - n].to(dt).transpose(0, 1)      # [H, rows, D]
                sc = (rows.abs().amax((1, 2)) / 127).clamp(min=SCALE_MIN)
                if old:
                    sc = torch.maximum(sc, scales[blk])
                    codes[blk, :, :old] = (codes[blk, :, :old] * (scales[blk] / sc)[:, None, None]).round()
                codes[blk, :, lo - j * bs:hi - j * bs] = (rows / sc[:, None, None]).round()
                scales[blk] = sc
        at = s["slots"].long()
        res.append(codes[at // bs, :, at % bs] * scales[at // bs][..., None])
        scales_out.append(scales)
    return torch.stack(res, 1).reshape(s["slots"].numel(), -1), scales_out[0], scales_out[1]


def _exact_attn(s):
    q, bs, D, H = s["q"], s["bs"], s["q"].shape[2], s["kc"].shape[1]
    cu, kl = s["cu_q"].tolist(), s["kv_lens"].tolist()
    group = q.shape[1] // H
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(kl):
        blocks = s["table"][b, :_ceil(n, bs)].long()
        nq = cu[b + 1] - cu[b]
        pos = torch.arange(n - nq, n, device=q.device, dtype=torch.float64)
        lim = torch.full_like(pos, n) if not s["chunk"] else ((pos / s["chunk"]).floor() + 1) * s["chunk"]
        seen = torch.arange(n, device=q.device)[None] < lim[:, None]
        for h in range(H):
            k = (s["kc"][blocks, h].double() * s["ks"][blocks, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["vc"][blocks, h].double() * s["vs"][blocks, h].double()[:, None, None]).reshape(-1, D)[:n]
            for g in range(h * group, (h + 1) * group):
                w = (q[cu[b]:cu[b + 1], g].double() @ k.t()) / math.sqrt(D)
                w = torch.where(seen, w, -math.inf)
                w = torch.where(seen.any(1, keepdim=True), torch.softmax(w, 1), 0.0)
                out[cu[b]:cu[b + 1], g] = w @ v
    return out


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None      # whole numbers only
    return {"rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[op](prepare(case, seed))
