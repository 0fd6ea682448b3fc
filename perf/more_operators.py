"""Prompts of several streams and a cache of bounded size, as cases to measure: attention over packed sequences, the attention
weight that each cached key has gathered, the choice of the keys that stay, and their move into the places of those that go.

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
        # the smallest call: a few camera tokens of five streams, 16 heads x 128
        dict(name="prompt_short", op="prompt", B=5, L=60, unit=1, ragged=0.98, hq=16, hk=16, D=128, chunk=1,
             dtype="fp16"),
        # four streams that begin with one to six frames each, every frame seeing its own and the earlier ones
        dict(name="prompt_frames", op="prompt", B=4, L=6 * P, unit=P, ragged=0.9, hq=16, hk=16, D=64, chunk=P,
             dtype="fp16"),
        # causal sequences of odd lengths, four query heads to each key head, bf16
        dict(name="prompt_shared_bf16", op="prompt", B=9, L=4099, unit=1, ragged=0.9, hq=32, hk=8, D=128, chunk=1,
             dtype="bf16"),
        # the aggregator's 32 frames at once, frame-causal
        dict(name="prompt_long", op="prompt", B=1, L=32 * P, unit=P, ragged=0.0, hq=16, hk=16, D=64, chunk=P,
             dtype="fp16"),
        # one camera token over a short cache
        dict(name="weigh_short", op="weigh", B=1, q=1, L=300, hq=16, hk=16, D=128, bs=64, chunk=0, ragged=0.0,
             decay=1.0, dtype="fp16"),
        # one token for each of eight streams over 32 frames
        dict(name="weigh_token", op="weigh", B=8, q=1, L=32 * P, hq=16, hk=16, D=64, bs=64, chunk=1, ragged=0.3,
             decay=0.95, dtype="fp16"),
        # 16 ragged requests, four query heads to each key head, bf16
        dict(name="weigh_shared_bf16", op="weigh", B=16, q=3, L=9001, hq=32, hk=8, D=128, bs=32, chunk=1, ragged=0.9,
             decay=1.0, dtype="bf16"),
        # one new frame over the 31 before it and itself
        dict(name="weigh_frame", op="weigh", B=1, q=P, L=32 * P, hq=16, hk=16, D=64, bs=64, chunk=P, ragged=0.0,
             decay=0.95, dtype="fp16"),
        # one layer of eight streams, a quarter of whose tokens go
        dict(name="choose_layer", op="choose", layers=1, B=8, L=8001, part=0.75, ragged=0.5, H=16, bs=64, sink=5,
             recent=0.02),
        # all 24 layers of one stream of 32 frames, which makes room for one frame
        dict(name="choose_stack", op="choose", layers=24, B=1, L=32 * P, part=31 / 32, ragged=0.0, H=16, bs=64, sink=P,
             recent=1 / 16),
        # one layer of eight streams, a quarter of whose tokens go, and the reading of what stays
        dict(name="evict_layer", op="evict", layers=1, B=8, L=2001, part=0.75, ragged=0.5, H=16, D=128, bs=32, sink=5,
             recent=0.02, dtype="bf16"),
        # four layers of one stream of 32 frames cut to 16, and the reading of what stays
        dict(name="evict_stack", op="evict", layers=4, B=1, L=32 * P, part=0.5, ragged=0.0, H=16, D=64, bs=64, sink=P,
             recent=1 / 16, dtype="fp16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "weigh", "weigh", "weigh", "choose", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    H, D, bs = rng.choice([1, 4, 8, 16]), rng.choice([64, 128]), rng.choice([32, 64, 128])
    group = rng.choice([1, 1, 2, 4, 7])
    ragged = rng.choice([0.0, 0.5, 0.95])
    if op == "prompt":
        # no more products than a fifth of the largest listed case's
        most = int(math.sqrt(16 * 10 ** 11 / (4 * H * group * D)))
        B = _logint(rng, 1, 16)
        L = _logint(rng, 1, int(most / math.sqrt(B)))
        unit = rng.choice([1, 1, max(1, L // 5)])
        return dict(op="prompt", B=B, L=L // unit * unit, unit=unit, ragged=ragged, hq=H * group, hk=H, D=D,
                    chunk=rng.choice([0, 1, unit if unit > 1 else _logint(rng, 2, P)]), dtype=dtype)
    if op == "weigh":
        B = _logint(rng, 1, 16)
        q = rng.choice([1, _logint(rng, 1, 16), _logint(rng, 17, 1400)])
        if q * group <= 32:
            most = 32 * P * 16 * 64 * 8 // (H * D)
        else:      # no more products than the largest listed case has
            most = 12 * 10 ** 10 // (2 * q * group * H * D)
        B = max(1, min(B, most // q))
        while most < q:
            q, most = q // 2, most * 2
        L = _logint(rng, q, max(q + 1, min(32 * P, most // B)))
        return dict(op="weigh", B=B, q=q, L=L, hq=H * group, hk=H, D=D, bs=bs,
                    chunk=rng.choice([0, 1, _logint(rng, 2, P)]), ragged=ragged, decay=rng.choice([1.0, 0.95]),
                    dtype=dtype)
    B, layers = _logint(rng, 1, 16), _logint(rng, 1, 24 if op == "choose" else 4)
    most = 24 * 32 * P * 16 if op == "choose" else 4 * 32 * P * 16 * 64 // D
    L = _logint(rng, 200, max(400, min(60000, most // (layers * B * H))))
    c = dict(op=op, layers=layers, B=B, L=L, part=rng.choice([0.5, 0.75, 0.9, 0.97]), ragged=ragged, H=H, bs=bs,
             sink=rng.choice([0, 5, 1 + L // 30]), recent=rng.choice([0.0, 0.02, 0.1]))
    if op == "evict":
        c.update(D=D, dtype=dtype)
    return c


# ------------------------------------------------------- what a case's sizes mean
def _fraction(i):
    return (i * 0.6180339887498949) % 1.0


def _prompt_lens(c):
    return [max(c["unit"], int(round(c["L"] * (1 - c["ragged"] * _fraction(i)) / c["unit"])) * c["unit"])
            for i in range(c["B"])]


def _weigh_lens(c):
    """(query lengths, key lengths) of the requests: ragged ones are shorter by up to that share."""
    ql = [max(1, int(round(c["q"] * (1 - c["ragged"] * _fraction(3 * i))))) for i in range(c["B"])]
    kl = [max(1, int(round(c["L"] * (1 - c["ragged"] * _fraction(i))))) for i in range(c["B"])]
    return ql, kl


def _evict_lens(c):
    """(lengths, lengths after) of the requests, the protected counts, the most moves of one head."""
    lens = [max(1, int(round(c["L"] * (1 - c["ragged"] * _fraction(i))))) for i in range(c["B"])]
    keep = [max(1, int(round(n * c["part"]))) for n in lens]
    recent = int(round(c["recent"] * min(lens)))
    return lens, keep, recent, max(min(k, n - k) for n, k in zip(lens, keep))


def _ceil(a, b):
    return -(-a // b)


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
    if op == "prompt":
        lens = _prompt_lens(c)
        return {"bytes": 4 * sum(lens) * (c["hq"] + c["hk"]) * c["D"],
                "flops": 4 * _visible(lens, lens, c["chunk"]) * c["hq"] * c["D"]}
    if op == "weigh":
        ql, kl = _weigh_lens(c)
        old = sum(max(0, k - q) for q, k in zip(ql, kl))
        blocks = sum(_ceil(k, c["bs"]) for k in kl)
        # queries and their log-sum-exp, K codes, old weights of the keys that had some in, new weights out
        n = sum(ql) * c["hq"] * (2 * c["D"] + 4) + c["hk"] * (sum(kl) * (c["D"] + 4) + 4 * old) + 4 * blocks * (c["hk"] + 1)
        return {"bytes": n, "flops": 2 * _visible(ql, kl, c["chunk"]) * c["hq"] * c["D"]}
    lens, keep, _, moves = _evict_lens(c)
    heads = c["layers"] * c["H"]
    if op == "choose":
        return {"bytes": 4 * heads * (sum(lens) + c["B"] * (2 * moves + 1)), "flops": 0}
    # a row that stays is moved when it stood past the new length: about the share of all rows that stay
    moved = sum(int((n - k) * k / n) for n, k in zip(lens, keep))
    row = 2 * c["D"]
    # moved codes, weights and their places in and out; all kept codes in and their values out
    return {"bytes": heads * (moved * (2 * row + 16) + sum(keep) * 3 * row), "flops": 2 * heads * moved * row}


# -------------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(g, layers, lens, H, D, bs, sides=2):
    """A cache that holds `lens` tokens per request in shuffled blocks: codes of normal values and a scale for each block
    and head, per layer; the table."""
    need = [_ceil(n, bs) for n in lens]
    num = sum(need) + 5
    codes = [(torch.randn(layers, num, H, bs, D, generator=g, device=DEV, dtype=torch.float16) * 34).round_()
             .clamp_(-127, 127).to(torch.int8) for _ in range(sides)]
    scales = [torch.exp(0.4 * torch.randn(layers, num, H, generator=g, device=DEV)) / 34 for _ in range(sides)]
    return codes, scales, _table(g, need, num), num


def _table(g, need, num):
    order = torch.randperm(num, generator=g, device=DEV).to(torch.int32)
    start, cols = torch.tensor(_sum0(need)[:-1], device=DEV), torch.arange(max(need), device=DEV)
    at = (start[:, None] + cols).clamp(max=num - 1)
    return torch.where(cols < torch.tensor(need, device=DEV)[:, None], order[at], -1).to(torch.int32).contiguous()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = c["op"]
    if op == "prompt":
        lens, dt = _prompt_lens(c), DTYPES[c["dtype"]]
        T, D = sum(lens), c["D"]
        # q, k and v as column ranges of one projection's output; a few queries look for one key
        qkv = torch.randn(T, c["hq"] + 2 * c["hk"], D, generator=g, device=DEV)
        qkv[::5, :c["hq"]] *= 3
        qkv = qkv.to(dt)
        q, k, v = qkv.split([c["hq"], c["hk"], c["hk"]], 1)
        return dict(op=op, q=q, k=k, v=v, cu=_ints(_sum0(lens)), lens=lens, chunk=c["chunk"])
    if op == "weigh":
        (ql, kl), dt, bs, D = _weigh_lens(c), DTYPES[c["dtype"]], c["bs"], c["D"]
        codes, scales, table, num = _cache(g, 1, kl, c["hk"], D, bs, sides=1)
        q = torch.randn(sum(ql), c["hq"], D, generator=g, device=DEV)
        q[::5] *= 3
        # weights gathered so far: a few keys hold most
        old = torch.exp(1.5 * torch.randn(num, c["hk"], bs, generator=g, device=DEV))
        s = dict(op=op, q=q.to(dt), kc=codes[0][0], ks=scales[0][0], table=table, cu_q=_ints(_sum0(ql)), kv_lens=_ints(kl),
                 fresh=_ints([max(0, k - n) for n, k in zip(ql, kl)]), ql=ql, kl=kl, chunk=c["chunk"], decay=c["decay"],
                 weights=old, out=torch.zeros_like(old))
        s["lse"] = _lse(s)
        return s
    lens, keep, recent, moves = _evict_lens(c)
    num = sum(_ceil(n, c["bs"]) for n in lens) + 5
    # accumulated weights: a few keys hold most, some have none yet
    w = torch.exp(1.5 * torch.randn(c["layers"], num, c["H"], c["bs"], generator=g, device=DEV))
    w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.03, 0.0, w)
    s = dict(op=op, weights=w, lens=_ints(lens), keep=_ints(keep), sink=c["sink"], recent=recent, moves=moves, bs=c["bs"],
             host_lens=lens, host_keep=keep)
    if op == "choose":
        s["table"] = _table(g, [_ceil(n, c["bs"]) for n in lens], num)
        return s
    codes, scales, table, _ = _cache(g, c["layers"], lens, c["H"], c["D"], c["bs"])
    s.update(kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1], table=table, dtype=DTYPES[c["dtype"]])
    s["src"], s["dst"], s["count"] = _plain_choose(s)
    # the slots of the rows that stay, for the reading
    b = torch.repeat_interleave(torch.arange(len(keep), device=DEV), torch.tensor(keep, device=DEV))
    j = torch.arange(sum(keep), device=DEV) - torch.tensor(_sum0(keep)[:-1], device=DEV)[b]
    s["slots"] = (table[b, j // c["bs"]].long() * c["bs"] + j % c["bs"]).to(torch.int32)
    return s


# --------------------------------------------------------------- plain forms
def _limits(first, rows, n, chunk, dev):
    """Keys seen by queries at positions first .. first + rows - 1 of n."""
    pos = torch.arange(first, first + rows, device=dev)
    if not chunk:
        return torch.full_like(pos, n)
    return ((torch.div(pos, chunk, rounding_mode="floor") + 1) * chunk).clamp(0, n)


def _step(n, heads):
    """Query rows to take at a time, so that the scores stay under 2 GB."""
    return max(1, min(4096, 5 * 10 ** 8 // (n * heads)))


def _plain_prompt(s):
    q, chunk = s["q"], s["chunk"]
    T, hq, D = q.shape
    H = s["k"].shape[1]
    out = torch.empty((T, hq, D), dtype=q.dtype, device=q.device)
    at = 0
    for n in s["lens"]:
        k, v = (x[at:at + n].float().permute(1, 0, 2)[:, None] for x in (s["k"], s["v"]))      # [H, 1, n, D]
        step = _step(n, hq)
        for i in range(0, n, step):
            r = min(step, n - i)
            qs = q[at + i:at + i + r].float().reshape(r, H, hq // H, D).permute(1, 2, 0, 3)
            S = (qs @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
            S.masked_fill_(torch.arange(n, device=q.device) >= _limits(i, r, n, chunk, q.device)[:, None], -math.inf)
            p = S.sub_(S.amax(-1, keepdim=True)).exp_()
            o = (p @ v) / p.sum(-1, keepdim=True)
            out[at + i:at + i + r] = o.permute(2, 0, 1, 3).reshape(r, hq, D).to(q.dtype)
        at += n
    return out


def _scores(s, b, i, r, dtype=torch.float32):
    """Scores of queries i .. i + r - 1 of request b over its keys, hidden ones -inf: [H, group, r, n]."""
    q, bs, (_, H, _, D) = s["q"], s["kc"].shape[2], s["kc"].shape
    n, at = s["kl"][b], sum(s["ql"][:b])
    blk = s["table"][b, :_ceil(n, bs)].long()
    k = s["kc"][blk].to(dtype) * s["ks"][blk].to(dtype)[..., None, None]                       # [blocks, H, bs, D]
    k = k.transpose(0, 1).reshape(H, 1, -1, D)[:, :, :n]
    qs = q[at + i:at + i + r].to(dtype).reshape(r, H, -1, D).permute(1, 2, 0, 3)
    S = (qs @ k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    lim = _limits(n - s["ql"][b] + i, r, n, s["chunk"], q.device)
    return S.masked_fill_(torch.arange(n, device=q.device) >= lim[:, None], -math.inf)


def _lse(s):
    """Log-sum-exp of every query's scores, fp32 [hq, tokens], as the attention over the cache gives it."""
    hq = s["q"].shape[1]
    parts = [torch.logsumexp(_scores(s, b, i, min(step, n - i)), -1).reshape(hq, -1)
             for b, n in enumerate(s["ql"]) for step in [_step(s["kl"][b], hq)] for i in range(0, n, step)]
    return torch.cat(parts, 1).contiguous()


def _plain_weigh(s):
    (num, H, bs, _), hq, lse = s["kc"].shape, s["q"].shape[1], s["lse"]
    at = 0
    for b, (nq, n) in enumerate(zip(s["ql"], s["kl"])):
        total = torch.zeros(H, n, device=lse.device)
        step = _step(n, hq)
        for i in range(0, nq, step):
            r = min(step, nq - i)
            e = lse[:, at + i:at + i + r].reshape(H, -1, r, 1)
            e = torch.where(e.isfinite(), e, math.inf)
            total += _scores(s, b, i, r).sub_(e).exp_().sum((1, 2))
        pos = torch.arange(n, device=lse.device)
        blk = s["table"][b, pos // bs].long()
        old = s["weights"][blk, :, pos % bs].t() * s["decay"]                                   # [H, n]
        s["out"][blk, :, pos % bs] = torch.where(pos < s["fresh"][b], total + old, total).t()
        at += nq
    return s["out"]


def _plain_choose(s):
    w, lens, keep, bs, m = s["weights"], s["lens"].long(), s["keep"].long(), s["bs"], s["moves"]
    table, dev = s["table"].long().clamp(min=0), s["weights"].device
    layers, _, H, _ = w.shape
    B, wide = table.shape
    n = max(s["host_lens"])
    big = torch.finfo(torch.float32).max
    # [layers, B, H, positions]
    x = w[:, table].permute(0, 1, 3, 2, 4).reshape(layers, B, H, wide * bs)[..., :n]
    x = torch.where(x.isnan(), -big, x.clamp(-big, big))
    pos, lens, keep = torch.arange(n, device=dev), lens[:, None], torch.minimum(keep, lens)[:, None]
    sink = keep.clamp(max=s["sink"])
    recent = (keep - sink).clamp(max=s["recent"])
    held = (pos < sink) | (pos >= lens - recent)
    x = torch.where(held[:, None], math.inf, x)
    x = torch.where((pos < lens)[:, None], x, -math.inf)
    order = x.sort(dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(x.shape, dtype=torch.bool, device=dev)
    stays.scatter_(-1, order, (pos < keep)[:, None].expand(layers, -1, H, -1))
    hole = ~stays & (pos < keep)[:, None]
    late = stays & (pos >= keep)[:, None]

    def places(mark):
        """Positions of the marks in order, then -1."""
        rank = mark.cumsum(-1) - 1
        to = torch.where(mark, rank, m)
        out = torch.full((*mark.shape[:-1], m + 1), -1, dtype=torch.int64, device=dev)
        return out.scatter_(-1, to, pos.expand(mark.shape))[..., :m].to(torch.int32).contiguous()

    return places(late), places(hole), hole.sum(-1).to(torch.int32)


def _plain_evict(s):
    bs, table, keep = s["bs"], s["table"].long(), s["keep"].long()
    layers, B, H, m = s["src"].shape
    dev = table.device
    l, b, h, i = torch.meshgrid(*(torch.arange(x, device=dev) for x in (layers, B, H, m)), indexing="ij")
    some = (i < s["count"][..., None]).reshape(-1)
    src, dst = s["src"].reshape(-1).long().clamp(min=0), s["dst"].reshape(-1).long().clamp(min=0)
    l, b, h = l.reshape(-1), b.reshape(-1), h.reshape(-1)
    num = s["ks"].shape[1]
    # moves that are none write a spare block
    sb, so = table[b, src // bs], src % bs
    db, do = torch.where(some, table[b, dst // bs], num), dst % bs
    for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        x = codes[l, sb, h, so].float() * scales[l, sb, h][:, None]
        # the spare block takes the padding's rows
        cell = (l * (num + 1) + db) * H + h
        most = torch.zeros(layers * (num + 1) * H, device=dev).scatter_reduce_(0, cell, x.abs().amax(-1), "amax")
        got = torch.zeros(layers * (num + 1) * H, dtype=torch.bool, device=dev)
        got[cell] = True
        most, got = (y.reshape(layers, num + 1, H)[:, :num] for y in (most, got))
        new = torch.where(got, torch.maximum(scales, torch.clamp(most / 127.0, min=SCALE_MIN)), scales)
        inv = 1.0 / new
        kept = (codes.float() * (scales * inv)[..., None, None]).round().clamp(-127, 127)
        kept = torch.where((new != scales)[..., None, None], kept, codes.float())
        kept = torch.nn.functional.pad(kept, (0, 0, 0, 0, 0, 0, 0, 1))
        kept[l, db, h, do] = (x * inv[l, db.clamp(max=num - 1), h][:, None]).round().clamp(-127, 127)
        codes.copy_(kept[:, :num].to(torch.int8))
        scales.copy_(new)
    w = torch.nn.functional.pad(s["weights"], (0, 0, 0, 0, 0, 1))
    w[l, db, h, do] = s["weights"][l, sb, h, so]
    s["weights"].copy_(w[:, :num])
    at = s["slots"].long()
    rows = [torch.stack([c[layer][at // bs, :, at % bs].float() * f[layer][at // bs][..., None]
                         for c, f in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))], 1).to(s["dtype"]).flatten(1)
            for layer in range(layers)]
    return rows, s["ks"], s["vs"], s["weights"]


def run(state):
    s = state
    if not own:
        return {"prompt": _plain_prompt, "weigh": _plain_weigh, "choose": _plain_choose, "evict": _plain_evict}[s["op"]](s)
    from qvggt_b200 import kv_cache
    if s["op"] == "prompt":
        return kv_cache.prompt_attention(s["q"], s["k"], s["v"], s["cu"], max(s["lens"]), causal_chunk=s["chunk"])
    if s["op"] == "weigh":
        return kv_cache.key_weights(s["q"], s["kc"], s["ks"], s["table"], s["cu_q"], s["kv_lens"], s["lse"], s["weights"],
                                    max(s["ql"]), max(s["kl"]), causal_chunk=s["chunk"], fresh_from=s["fresh"],
                                    decay=s["decay"], out=s["out"])
    if s["op"] == "choose":
        p = kv_cache.evict_plan(s["weights"], s["table"], s["lens"], s["keep"], s["sink"], s["recent"], s["moves"],
                                max_len=max(s["host_lens"]))
        return p.src, p.dst, p.counts
    kv_cache.kv_evict(s["kc"], s["vc"], s["ks"], s["vs"], s["weights"], s["table"], s["keep"],
                      kv_cache.EvictPlan(s["src"], s["dst"], s["count"]))
    rows = [kv_cache.kv_gather(s["kc"][i], s["vc"][i], s["ks"][i], s["vs"][i], s["slots"], s["dtype"])
            for i in range(s["kc"].shape[0])]
    return rows, s["ks"], s["vs"], s["weights"]


# ------------------------------------------------------ definitions in 64 bits
def _exact_prompt(s):
    q, k, v, D = s["q"], s["k"], s["v"], s["q"].shape[2]
    group = q.shape[1] // k.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    first = 0
    for n in s["lens"]:
        block = s["chunk"] or n
        rows = slice(first, first + n)
        for h in range(q.shape[1]):
            kd, vd = k[rows, h // group].double(), v[rows, h // group].double()
            for i in range(0, n, 2048):
                qd = q[first + i:first + min(n, i + 2048), h].double()
                # position i sees j where j's block is not after its own
                mine = torch.arange(i, i + qd.shape[0], device=q.device) // block
                theirs = torch.arange(n, device=q.device) // block
                w = torch.where(theirs[None] <= mine[:, None], qd @ kd.t() / math.sqrt(D), -math.inf)
                out[first + i:first + i + qd.shape[0], h] = torch.softmax(w, 1) @ vd
        first += n
    return out


def _exact_weigh(s):
    q, bs, D, H = s["q"], s["kc"].shape[2], s["q"].shape[2], s["kc"].shape[1]
    group, out = q.shape[1] // H, s["out"].double()
    cu = s["cu_q"].tolist()
    for b, n in enumerate(s["kv_lens"].tolist()):
        nq = cu[b + 1] - cu[b]
        ids = s["table"][b, :_ceil(n, bs)].long()
        where = (ids[:, None] * bs + torch.arange(bs, device=q.device)).reshape(-1)[:n]
        block = s["chunk"] or max(n, 1)
        theirs = torch.arange(n, device=q.device) // block
        fresh = int(s["fresh"][b])
        for h in range(H):
            kd = (s["kc"][ids, h].double() * s["ks"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            total = torch.zeros(n, dtype=torch.float64, device=q.device)
            for g in range(h * group, (h + 1) * group):
                for i in range(0, nq, 1024):
                    r = min(1024, nq - i)
                    mine = torch.div(torch.arange(n - nq + i, n - nq + i + r, device=q.device), block, rounding_mode="floor")
                    x = q[cu[b] + i:cu[b] + i + r, g].double() @ kd.t() / math.sqrt(D)
                    x = x - s["lse"][g, cu[b] + i:cu[b] + i + r].double()[:, None]
                    seen = s["lse"][g, cu[b] + i:cu[b] + i + r].isfinite()[:, None].expand(r, n)
                    if s["chunk"]:
                        seen = seen & (theirs[None] <= mine[:, None])
                    total += torch.where(seen, x.exp(), 0.0).sum(0)
            before = s["weights"][:, h].reshape(-1)[where].double() * s["decay"]
            before[fresh:] = 0
            out[where // bs, h, where % bs] = total + before
    return out


def _exact_evict(s):
    bs, out_w = s["bs"], s["weights"].double()
    layers, B, H, _ = s["src"].shape
    res, scales = [], [s["ks"].double(), s["vs"].double()]
    values = [c.double() * f[..., None, None] for c, f in zip((s["kc"], s["vc"]), scales)]
    count = s["count"].tolist()
    for b in range(B):
        ids = s["table"][b, :_ceil(s["host_lens"][b], bs)].long()
        for layer in range(layers):
            for h in range(H):
                m = count[layer][b][h]
                src, dst = s["src"][layer, b, h, :m].long(), s["dst"][layer, b, h, :m].long()
                to, place = torch.unique(dst // bs, return_inverse=True)
                for side in range(2):
                    x = values[side][layer, ids, h].reshape(len(ids) * bs, -1)
                    f = scales[side][layer, ids, h]
                    need = torch.zeros(len(to), dtype=torch.float64, device=x.device)
                    need.index_reduce_(0, place, x[src].abs().amax(1) / 127, "amax")
                    grown = f.clone()
                    grown[to] = torch.maximum(f[to], need.clamp(min=SCALE_MIN))
                    y = x.clone()
                    y[dst] = x[src]
                    y = y.reshape(len(ids), bs, -1)
                    y[to] = (y[to] / grown[to, None, None]).round() * grown[to, None, None]
                    values[side][layer, ids, h] = y
                    scales[side][layer, ids, h] = grown
                line = out_w[layer, ids, h].reshape(-1)
                line[dst] = line[src]
                out_w[layer, ids, h] = line.reshape(-1, bs)
    at = s["slots"].long()
    for layer in range(layers):
        res.append(torch.stack([v[layer][at // bs, :, at % bs] for v in values], 1).flatten(1))
    return res, scales[0], scales[1], out_w


def exact(case, seed):
    op = case["op"]
    if op == "choose":
        return None      # whole numbers only
    return {"prompt": _exact_prompt, "weigh": _exact_weigh, "evict": _exact_evict}[op](prepare(case, seed))
