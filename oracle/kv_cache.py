"""CPU restatement of the streaming K/V cache operators, in 64 bits (test infrastructure).

``append_f32`` is the exception: the codes of the cache are defined by 32-bit
arithmetic, so it restates that, one rounding per operation, and must agree
with the kernels bit for bit.
"""
from __future__ import annotations

import math

import numpy as np
import torch

SCALE_MIN = np.float32(2.0 ** -60)


def rope_pairs(sections, layout):
    """(lo dim, hi dim, axis) of every pair of a head."""
    half, out, base = sum(sections), [], 0
    for axis, n in enumerate(sections):
        for j in range(n):
            i = base + j
            out.append({"axial": (2 * base + j, 2 * base + n + j), "split": (i, i + half),
                        "interleaved": (2 * i, 2 * i + 1)}[layout] + (axis,))
        base += n
    return out


def rope_axes(x, positions, inv_freq, sections, layout="axial", inverse=False):
    """x [T, H, D] (any float type) -> float64 [T, H, D]."""
    x = x.double()
    y = x.clone()
    for j, (lo, hi, axis) in enumerate(rope_pairs(sections, layout)):
        t = positions[axis].double() * inv_freq[j].double() * (-1.0 if inverse else 1.0)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        y[..., lo] = x[..., lo] * c - x[..., hi] * s
        y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def block_plan(cached, target, table, ring, free_range, bs, max_new):
    """Lists and numpy arrays; one request after another.  Returns a dict of the outputs (table and ring as copies)."""
    table, ring = table.copy(), ring.copy()
    B, wide = table.shape
    n = len(ring)
    head, tail = free_range

    def blocks(t):
        return -(-t // bs)

    status = 0
    if any(c < 0 or t < 0 for c, t in zip(cached, target)):
        status = 3
    elif any(blocks(c) > wide or blocks(t) > wide for c, t in zip(cached, target)):
        status = 2
    elif sum(max(0, t - c) for c, t in zip(cached, target)) > max_new:
        status = 4
    elif not 0 <= head <= tail <= head + n or sum(max(0, blocks(c) - blocks(t)) for c, t in zip(cached, target)) > n - (tail - head):
        status = 5
    elif sum(max(0, blocks(t) - blocks(c)) for c, t in zip(cached, target)) > tail - head:
        status = 1
    slots, cu_new, cu_blocks = [], [0], [0]
    lens = list(cached)
    if status == 0:
        for b, (c, t) in enumerate(zip(cached, target)):
            for j in range(blocks(c), blocks(t)):
                table[b, j] = ring[head % n]
                head += 1
        for b, (c, t) in enumerate(zip(cached, target)):
            for j in range(blocks(t), blocks(c)):
                ring[tail % n] = table[b, j]
                tail += 1
            slots += [int(table[b, j // bs]) * bs + j % bs for j in range(c, t)]
            cu_new.append(len(slots))
            cu_blocks.append(cu_blocks[-1] + (len({j // bs for j in range(c, t)})))
            lens[b] = t
    else:
        cu_new, cu_blocks = [0] * (B + 1), [0] * (B + 1)
    slots += [-1] * (max_new - len(slots))
    return dict(table=table, ring=ring, slots=slots, cu_new=cu_new, cu_blocks=cu_blocks, lens=lens,
                free_range=[head, tail], status=status)


def append_f32(x, codes, scales, table, cached, cu_new):
    """New rows x [T, H, D] into codes int8 [nb, H, bs, D] / scales float32 [nb, H] (numpy, updated in place)."""
    f32 = np.float32
    bs = codes.shape[2]
    x = x.float().numpy()
    for b, c in enumerate(cached):
        end = c + cu_new[b + 1] - cu_new[b]
        for j in range(c // bs, -(-end // bs)):
            lo, hi = max(c, j * bs), min(end, (j + 1) * bs)
            if hi <= lo:
                continue
            blk, older = table[b][j], lo - j * bs
            for h in range(codes.shape[1]):
                rows = x[cu_new[b] + lo - c:cu_new[b] + hi - c, h]
                fin = np.where(np.isfinite(rows), np.abs(rows), f32(0))
                before = scales[blk, h] if older else f32(0)
                s = max(before, f32(fin.max() / f32(127)), SCALE_MIN)
                inv = f32(f32(1) / s)
                if older:
                    r = f32(before * inv)
                    codes[blk, h, :older] = np.clip(np.rint(codes[blk, h, :older].astype(f32) * r), -127, 127)
                with np.errstate(over="ignore", invalid="ignore"):
                    q = np.rint(rows * inv)
                q = np.where(np.isnan(q), f32(0), np.clip(q, -127, 127))
                codes[blk, h, older:older + hi - lo] = q.astype(np.int8)
                scales[blk, h] = s


def key_limit(i, ql, n, chunk):
    """Keys that query i of ql sees among n."""
    if not chunk:
        return n
    pos = n - ql + i
    return max(0, min(n, (math.floor(pos / chunk) + 1) * chunk)) if pos >= 0 else 0


def cached_attention(q, kc, vc, ks, vs, table, cu_q, kv_lens, chunk=0, scale=None):
    """-> (out float64 [T, Hq, D], lse float64 [Hq, T], sum of weights times |v| [T, Hq, D]); all on q's device.

    Rows without keys: 0, -inf, 0."""
    dev = q.device
    T, hq, D = q.shape
    bs, hk = kc.shape[2], kc.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, hq, D, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    lse = torch.full((hq, T), -math.inf, dtype=torch.float64, device=dev)
    cu, lens, tab = cu_q.tolist(), kv_lens.tolist(), table.tolist()
    for b, n in enumerate(lens):
        ql = cu[b + 1] - cu[b]
        if n == 0 or ql == 0:
            continue
        blocks = torch.tensor(tab[b][:-(-n // bs)], dtype=torch.long, device=dev)
        k = (kc[blocks].double() * ks[blocks].double()[..., None, None]).permute(1, 0, 2, 3).reshape(hk, -1, D)[:, :n]
        v = (vc[blocks].double() * vs[blocks].double()[..., None, None]).permute(1, 0, 2, 3).reshape(hk, -1, D)[:, :n]
        lim = torch.tensor([key_limit(i, ql, n, chunk) for i in range(ql)], device=dev)
        seen = torch.arange(n, device=dev) < lim[:, None]
        for h in range(hq):
            kh, vh = k[h // (hq // hk)], v[h // (hq // hk)]
            # what no query sees may hold anything
            most = int(lim.max())
            x = (q[cu[b]:cu[b + 1], h].double() @ kh[:most].T) * scale
            x = x.masked_fill(~seen[:, :most], -math.inf)
            if most == 0:
                continue
            m = x.max(1, keepdim=True).values.clamp(min=-1e300)
            w = torch.exp(x - m)
            l = w.sum(1, keepdim=True)
            some = lim > 0
            w = torch.where(some[:, None], w / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(w))
            vm = torch.where(seen[:, :most].any(0)[:, None], vh[:most], torch.zeros_like(vh[:most]))
            out[cu[b]:cu[b + 1], h] = w @ vm
            mag[cu[b]:cu[b + 1], h] = w @ vm.abs()
            lse[h, cu[b]:cu[b + 1]] = torch.where(some, m[:, 0] + torch.log(l[:, 0]),
                                                  torch.full_like(l[:, 0], -math.inf))
    return out, lse, mag
