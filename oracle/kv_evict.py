"""Prompts and a cache of bounded size, restated: attention over packed sequences, gathered key weights, the choice of the
keys that stay (all in 64 bits or whole numbers), and their move (in the 32-bit arithmetic that the codes are defined in).

Test infrastructure: nothing under ``qvggt_b200`` imports it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from .kv_cache import SCALE_MIN, key_limit


def prompt_attention(q, k, v, cu, chunk=0, scale=None):
    """-> (out float64 [T, Hq, D], lse float64 [Hq, T], sum of weights times |v| [T, Hq, D]); rows outside cu are 0.

    A row's sums run over the keys it sees and no others, whatever the others hold."""
    T, hq, D = q.shape
    group = hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, hq, D, dtype=torch.float64, device=q.device)
    mag, lse = torch.zeros_like(out), torch.zeros(hq, T, dtype=torch.float64, device=q.device)
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        step = chunk or max(n, 1)
        for i in range(0, n, step):
            last = min(n, i + step)
            x = torch.einsum("thd,khd->htk", q[a + i:a + last].double(),
                             k[a:a + last].double().repeat_interleave(group, 1)) * scale
            vals = v[a:a + last].double().repeat_interleave(group, 1)
            w = torch.softmax(x, -1)
            out[a + i:a + last] = torch.einsum("htk,khd->thd", w, vals)
            mag[a + i:a + last] = torch.einsum("htk,khd->thd", w, vals.abs())
            lse[:, a + i:a + last] = torch.logsumexp(x, -1)
    return out, lse, mag


def key_weights(q, kc, ks, table, cu_q, kv_lens, lse, weights, chunk=0, scale=None, fresh=None, decay=1.0):
    """-> (weights float64 [nb, H, bs] after the call, a bound of what 32-bit arithmetic may be off by).

    The bound: a score is D products summed in fp32 (D 2^-23 of their magnitudes' sum), its exponent one fma with
    lse log2e (2^-22 of both), the exponential 2^-22; the sum over r rows r 2^-24, decay and addition 2^-23."""
    nb, H, bs, D = kc.shape
    group = q.shape[1] // H
    scale = D ** -0.5 if scale is None else scale
    out, err = weights.double().clone(), torch.zeros_like(weights, dtype=torch.float64)
    cu, lens, tab = cu_q.tolist(), kv_lens.tolist(), table.tolist()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ql = cu[b + 1] - cu[b]
        ids = torch.tensor(tab[b][:-(-n // bs)], dtype=torch.long, device=q.device)
        pos = torch.arange(n, device=q.device)
        lim = torch.tensor([key_limit(i, ql, n, chunk) for i in range(ql)], dtype=torch.long, device=q.device)
        old = weights.double()[ids].permute(1, 0, 2).reshape(H, -1)[:, :n] * decay
        if fresh is not None:
            old = torch.where(pos < int(fresh[b]), old, 0.0)
        for h in range(H):
            k = (kc[ids, h].double() * ks[ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            total, off = torch.zeros(n, dtype=torch.float64, device=q.device), 0.0
            for g in range(h * group, (h + 1) * group):
                e = lse[g, cu[b]:cu[b + 1]].double()
                on = e.isfinite()
                seen = (pos < lim[:, None]) & on[:, None]
                rows = torch.where(on[:, None], q[cu[b]:cu[b + 1], g].double(), 0.0)
                e = torch.where(on, e, 0.0)
                x = rows @ k.t() * scale
                p = torch.where(seen, (x - e[:, None]).exp(), 0.0)
                amp = rows.abs() @ k.abs().t() * scale
                total += p.sum(0)
                off = off + (p * (D * 2.0 ** -23 * amp + 2.0 ** -22 * (e.abs()[:, None] + x.abs() + 1))).sum(0)
            r = ql * group
            at = (ids[pos // bs], h, pos % bs)
            out[at] = old[h] + total
            err[at] = off + total * r * 2.0 ** -24 + (old[h] + total) * 2.0 ** -23 + r * 2.0 ** -126
    return out, err


def evict_plan(weights, table, lens, keep, sink, recent, max_moves):
    """weights numpy float32 [layers, nb, H, bs] -> src, dst int32 [layers, B, H, max_moves], counts [layers, B, H]."""
    layers, _, H, bs = weights.shape
    B, big = len(lens), np.finfo(np.float32).max
    src = np.full((layers, B, H, max_moves), -1, np.int32)
    dst, counts = src.copy(), np.zeros((layers, B, H), np.int32)
    for b, (n, k) in enumerate(zip(lens, keep)):
        if n < 0 or k < 0 or k >= n:
            continue
        first = min(sink, k)
        last = min(recent, k - first)
        for layer in range(layers):
            for h in range(H):
                w = [weights[layer, table[b][j // bs], h, j % bs] for j in range(first, n - last)]
                w = [-big if math.isnan(x) else min(max(float(x), -big), big) for x in w]
                order = sorted(range(len(w)), key=lambda i: (-w[i], i))
                stays = {first + i for i in order[:k - first - last]} | set(range(first)) | set(range(n - last, n))
                holes = [j for j in range(k) if j not in stays]
                late = [j for j in range(k, n) if j in stays]
                assert len(holes) == len(late)
                counts[layer, b, h] = min(len(holes), max_moves)
                m = counts[layer, b, h]
                src[layer, b, h, :m], dst[layer, b, h, :m] = late[:m], holes[:m]
    return src, dst, counts


def kv_evict(codes, scales, table, src, dst, counts):
    """Moves rows of codes int8 [layers, nb, H, bs, D] / scales float32 [layers, nb, H] (numpy, updated in place)."""
    f32 = np.float32
    layers, B, H, _ = src.shape
    bs = codes.shape[3]
    for layer in range(layers):
        for b in range(B):
            for h in range(H):
                m = counts[layer, b, h]
                incoming = {}
                for s, d in zip(src[layer, b, h, :m], dst[layer, b, h, :m]):
                    blk = table[b][s // bs]
                    x = codes[layer, blk, h, s % bs].astype(f32) * scales[layer, blk, h]
                    incoming.setdefault(d // bs, []).append((d % bs, x))
                for j, rows in incoming.items():
                    blk = table[b][j]
                    c = codes[layer, blk, h]
                    before = scales[layer, blk, h]
                    amax = max(np.abs(x).max() for _, x in rows)
                    new = max(before, f32(amax / f32(127)), SCALE_MIN)
                    inv = f32(f32(1) / new)
                    if new != before:
                        c[:] = np.clip(np.rint(c.astype(f32) * f32(before * inv)), -127, 127).astype(np.int8)
                        scales[layer, blk, h] = new
                    for to, x in rows:
                        c[to] = np.clip(np.rint(x * inv), -127, 127).astype(np.int8)


def evict_weights(weights, table, src, dst, counts):
    """The weights' share of the move (numpy [layers, nb, H, bs], in place)."""
    layers, B, H, _ = src.shape
    bs = weights.shape[3]
    for layer in range(layers):
        for b in range(B):
            for h in range(H):
                for i in range(counts[layer, b, h]):
                    s, d = src[layer, b, h, i], dst[layer, b, h, i]
                    weights[layer, table[b][d // bs], h, d % bs] = weights[layer, table[b][s // bs], h, s % bs]
