"""A paged K/V cache in 8 bits and the operators around it, on the sm_100a kernels.

For frames (or camera tokens) that arrive a few at a time: the K/V rows of the
tokens seen so far stay on the GPU as int8 codes with one fp32 scale per
(block of tokens, head), a quarter of the bytes of fp32 and half of fp16, and
new queries attend to them without a dequantised copy.

:func:`rope_axes`         positions with several axes (time, height, width) on q and k
:func:`block_plan`        block tables and slot maps from request lengths, on the GPU
:func:`kv_append`         quantises new K/V rows into their blocks
:func:`kv_gather`         reads rows back as fp16 / bf16 ``[k | v]``
:func:`cached_attention`  attention over the cache, ragged requests, shared heads, block-causal mask
:class:`PagedKVCache`     the buffers of several layers with one block table, and the calls in order

Layout: codes int8 ``[num_blocks, kv_heads, block_size, head_dim]`` (K and V
apart), scales fp32 ``[num_blocks, kv_heads]``; token j of request b is row
``j % block_size`` of block ``block_tables[b, j // block_size]``.

Every call launches on the current stream of its tensors' device and returns
without waiting; CPU tensors, wrong types and shapes raise.  Lengths and tables
live on the GPU, so their contents are checked there: a block id or length
outside its range is skipped and sets the library's status word
(``_lib.device_status()``, 0x201 / 0x202).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from .awq_inference_engine import _Dev, _check_cuda, _check_dtype, _check_shape, _stream

__all__ = ["rope_axes", "block_plan", "BlockPlan", "kv_append", "kv_gather", "cached_attention",
           "attention_scratch_bytes", "PagedKVCache", "PLAN_STATUS"]

_HALF = {torch.float16: 0, torch.bfloat16: 1}      # QVGGT_DTYPE_F16 / _BF16
_LAYOUTS = {"axial": 0, "split": 1, "interleaved": 2}

PLAN_STATUS = {0: "done", 1: "too few free blocks", 2: "a request needs more blocks than its table row holds",
               3: "a negative length", 4: "more new tokens than max_new"}


def _half(name, t, what):
    code = _HALF.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: {what} must be float16 or bfloat16, got {t.dtype}")
    return code


def _rows3(name, t, what):
    """[tokens, heads, head_dim] with unit stride inside a head."""
    if t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name}: {what} {tuple(t.shape)} (strides {t.stride()}) must be [tokens, heads, head_dim] "
                         "with unit stride in head_dim")


def _ints(name, t, what, shape=None):
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise TypeError(f"{name}: {what} must be contiguous int32, got {t.dtype}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)} must be {shape}")


# ---------------------------------------------------------------------- RoPE
def rope_axes(q, k, positions, inv_freq, sections, layout: str = "axial", inverse: bool = False, q_out=None,
              k_out=None):
    """Rotary positions with 1 to 4 axes on q ``[T, Hq, D]`` and k ``[T, Hk, D]`` (or None), in one launch.

    ``positions`` int32 ``[axes, T]``; ``inv_freq`` fp32 ``[R/2]``; ``sections``:
    how many of the R/2 pairs each axis owns, in order.  Pair j turns by
    ``positions[axis_j, t] * inv_freq[j]``.  ``layout``: ``"axial"`` (each
    axis' pairs are the halves of its own slice of the head, as in VGGT's 2-D
    RoPE), ``"split"`` (dims j and j + R/2) or ``"interleaved"`` (2j, 2j + 1);
    dims >= R pass through.  ``inverse`` turns back, which is also the gradient
    of the forward turn.  Any token and head strides; fp16 or bf16; ``q_out`` /
    ``k_out`` may be q / k.  Returns (q, k) turned."""
    name = "rope_axes"
    dev = _check_cuda(name, q, k, positions, inv_freq, q_out, k_out)
    dt = _half(name, q, "q")
    _rows3(name, q, "q")
    T, hq, D = q.shape
    hk = 0
    if k is not None:
        _rows3(name, k, "k")
        _check_dtype(name, k, q.dtype)
        hk = k.shape[1]
        _check_shape(name, k.shape[0] == T and k.shape[2] == D, f"k {tuple(k.shape)} must be [{T}, heads, {D}]")
    if layout not in _LAYOUTS:
        raise ValueError(f"{name}: layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
    axes = len(sections)
    _check_shape(name, 1 <= axes <= 4, f"1 to 4 axes, got {axes}")
    _check_shape(name, inv_freq.dtype == torch.float32 and inv_freq.is_contiguous()
                 and inv_freq.numel() == sum(sections), f"inv_freq must be float32 with {sum(sections)} entries")
    _check_shape(name, positions.dtype == torch.int32 and tuple(positions.shape) == (axes, T)
                 and (positions.stride(1) == 1 or T <= 1),
                 f"positions {tuple(positions.shape)} must be int32 [{axes}, {T}] with unit stride in tokens")
    outs = []
    for x, o, what in ((q, q_out, "q_out"), (k, k_out, "k_out")):
        if x is not None and o is None:
            o = torch.empty(x.shape, dtype=x.dtype, device=dev)
        elif o is not None:
            _rows3(name, o, what)
            _check_dtype(name, o, x.dtype)
            _check_shape(name, o.shape == x.shape, f"{what} {tuple(o.shape)} must be {tuple(x.shape)}")
        outs.append(o)
    qo, ko = outs
    sect = (C.c_int32 * axes)(*sections)
    with _Dev(dev):
        _lib.call("qvggt_rope_axes", q.data_ptr(), q.stride(0), q.stride(1), qo.data_ptr(), qo.stride(0),
                  qo.stride(1), hq, k.data_ptr() if hk else None, k.stride(0) if hk else 0,
                  k.stride(1) if hk else 0, ko.data_ptr() if hk else None, ko.stride(0) if hk else 0,
                  ko.stride(1) if hk else 0, hk, T, D, positions.data_ptr(), positions.stride(0),
                  inv_freq.data_ptr(), sect, axes, _LAYOUTS[layout], 1 if inverse else 0, dt, _stream(q))
    return qo, ko


# -------------------------------------------------------------- block tables
class BlockPlan(NamedTuple):
    """What :func:`block_plan` writes (all on the GPU)."""
    slots: torch.Tensor        # int32 [max_new]: cache row of each new token, then -1
    cu_new: torch.Tensor       # int32 [B + 1]: running sum of the new tokens
    cu_blocks: torch.Tensor    # int32 [B + 1]: running sum of the blocks that get new tokens
    lens: torch.Tensor         # int32 [B]: lengths after the call
    free_range: torch.Tensor   # int64 [2]: the free ring's range after the call
    status: torch.Tensor       # int32 [1]: 0, or why nothing was changed (PLAN_STATUS)


def block_plan(cached_lens, target_lens, block_tables, free_ring, free_range, block_size: int,
               max_new: int) -> BlockPlan:
    """Takes requests from ``cached_lens`` to ``target_lens`` tokens (int32 ``[B]``), on the GPU.

    A request that grows gets blocks from ``free_ring`` (int32
    ``[num_blocks]``, the free ones at positions ``free_range[0]`` to
    ``free_range[1]``, int64 ``[2]``, modulo its size); one that shrinks (0:
    ends) gives its surplus blocks back.  ``block_tables`` (int32 ``[B,
    max_blocks]``) and ``free_ring`` are updated in place, the rest is
    returned; if a request cannot be served nothing is changed and ``status``
    says why.  ``max_new`` bounds the new tokens."""
    name = "block_plan"
    dev = _check_cuda(name, cached_lens, target_lens, block_tables, free_ring, free_range)
    _ints(name, cached_lens, "cached_lens")
    B = cached_lens.numel()
    _ints(name, target_lens, "target_lens", (B,))
    _ints(name, block_tables, "block_tables")
    _ints(name, free_ring, "free_ring")
    _check_shape(name, block_tables.dim() == 2 and block_tables.shape[0] == B,
                 f"block_tables {tuple(block_tables.shape)} must be [{B}, max_blocks]")
    _check_shape(name, free_range.dtype == torch.int64 and free_range.is_contiguous() and free_range.numel() == 2,
                 "free_range must be int64 [2]")
    # one allocation: the 64-bit pair first, then the 32-bit arrays
    buf = torch.empty(4 + 3 * B + 3 + max_new, dtype=torch.int32, device=dev)
    free_out = buf[:4].view(torch.int64)
    cu_new, cu_blocks, lens, status, slots = buf[4:].split_with_sizes([B + 1, B + 1, B, 1, max_new])
    at = buf.data_ptr()
    with _Dev(dev):
        _lib.call("qvggt_block_plan", cached_lens.data_ptr(), target_lens.data_ptr(), B, block_tables.data_ptr(),
                  block_tables.shape[1], free_ring.data_ptr(), free_ring.numel(), free_range.data_ptr(), block_size,
                  max_new, at + 4 * (3 * B + 7), at + 16, at + 4 * (B + 5), at + 4 * (2 * B + 6), at,
                  at + 4 * (3 * B + 6), _stream(cached_lens))
    return BlockPlan(slots, cu_new, cu_blocks, lens, free_out, status)


# --------------------------------------------------------------------- cache
def _check_cache(name, k_cache, v_cache, k_scale, v_scale):
    """Cache tensors -> (num_blocks, kv_heads, block_size, head_dim)."""
    if k_cache.dim() != 4 or k_cache.dtype != torch.int8 or v_cache.dtype != torch.int8:
        raise TypeError(f"{name}: the caches must be int8 [num_blocks, kv_heads, block_size, head_dim]")
    nb, h, bs, d = k_cache.shape
    inner = (bs * d, d, 1)
    if v_cache.shape != k_cache.shape or k_cache.stride()[1:] != inner or v_cache.stride() != k_cache.stride():
        raise ValueError(f"{name}: K and V caches must have the same shape and strides, dense inside a block")
    for s, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if s.dtype != torch.float32 or tuple(s.shape) != (nb, h) or not s.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous float32 [{nb}, {h}]")
    return nb, h, bs, d


def kv_append(k, v, k_cache, v_cache, k_scale, v_scale, block_tables, cached_lens, cu_new, cu_blocks,
              max_units: int | None = None):
    """Quantises new rows k, v ``[tokens, kv_heads, head_dim]`` (fp16 / bf16, requests packed as ``cu_new`` says, any
    16-byte aligned token and head strides) into the cache.

    ``cu_new`` and ``cu_blocks`` come from :func:`block_plan`, ``cached_lens``
    are the lengths before.  A block's scale grows when its new rows need it,
    and its earlier codes are rounded to the new scale.  ``max_units``: a
    bound of ``cu_blocks[-1]`` if one tighter than ``tokens // block_size + 2
    * B`` is known."""
    name = "kv_append"
    dev = _check_cuda(name, k, v, k_cache, v_cache, k_scale, v_scale, block_tables, cached_lens, cu_new, cu_blocks)
    nb, h, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    dt = _half(name, k, "k")
    _check_dtype(name, v, k.dtype)
    _rows3(name, k, "k")
    _rows3(name, v, "v")
    T = k.shape[0]
    _check_shape(name, tuple(k.shape) == (T, h, d) and v.shape == k.shape,
                 f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {h}, {d}]")
    B = cached_lens.numel()
    _ints(name, block_tables, "block_tables")
    _ints(name, cached_lens, "cached_lens")
    _ints(name, cu_new, "cu_new", (B + 1,))
    _ints(name, cu_blocks, "cu_blocks", (B + 1,))
    _check_shape(name, block_tables.dim() == 2 and block_tables.shape[0] == B,
                 f"block_tables {tuple(block_tables.shape)} must be [{B}, max_blocks]")
    if max_units is None:
        max_units = T // bs + 2 * B
    with _Dev(dev):
        _lib.call("qvggt_kv_append", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                  T, dt, k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(),
                  v_scale.data_ptr(), nb, h, bs, d, block_tables.data_ptr(), block_tables.shape[1],
                  cached_lens.data_ptr(), cu_new.data_ptr(), cu_blocks.data_ptr(), B, max_units, _stream(k))


def kv_gather(k_cache, v_cache, k_scale, v_scale, slots, dtype=torch.float16, out=None):
    """The cache rows of ``slots`` (int32 ``[n]``) as ``[n, 2 * kv_heads * head_dim]`` rows ``[k | v]``, the layout
    :func:`~qvggt_b200.awq_inference_engine.attention` reads; a negative slot gives zeros."""
    name = "kv_gather"
    dev = _check_cuda(name, k_cache, v_cache, k_scale, v_scale, slots, out)
    nb, h, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    _ints(name, slots, "slots")
    n = slots.numel()
    if out is None:
        out = torch.empty(n, 2 * h * d, dtype=dtype, device=dev)
    _check_shape(name, out.dim() == 2 and tuple(out.shape) == (n, 2 * h * d) and out.stride(1) == 1,
                 f"out {tuple(out.shape)} must be [{n}, {2 * h * d}]")
    dt = _half(name, out, "out")
    with _Dev(dev):
        _lib.call("qvggt_kv_gather", k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(),
                  v_scale.data_ptr(), nb, h, bs, d, slots.data_ptr(), n, out.data_ptr(), out.stride(0), dt,
                  _stream(slots))
    return out


# ----------------------------------------------------------------- attention
def attention_scratch_bytes(tokens: int, q_heads: int, kv_heads: int, requests: int, max_q: int, max_kv: int,
                            head_dim: int) -> int:
    """Scratch :func:`cached_attention` needs for these sizes on the current device."""
    nb = C.c_int64(0)
    _lib.call("qvggt_cached_attention_scratch", tokens, q_heads, kv_heads, requests, max_q, max_kv, head_dim,
              C.byref(nb))
    return int(nb.value)


def cached_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens, max_q: int, max_kv: int,
                     causal_chunk: int = 0, scale: float | None = None, out=None, lse=None, scratch=None):
    """``softmax(scale q k^T + mask) v`` over the 8-bit cache, for requests of any lengths.

    q ``[tokens, Hq, head_dim]`` fp16 / bf16: request b's queries are rows
    ``cu_q[b]`` to ``cu_q[b + 1]`` (at most ``max_q``), its keys the first
    ``kv_lens[b]`` tokens of table row b (``max_kv``: about the longest; it
    sets how the work is split).  ``Hq`` is a multiple of the cache's heads.
    Query i of ql sits at position ``kv_len - ql + i``.  ``causal_chunk`` 0:
    every query sees every key; 1: causal; the tokens of a frame: its own and
    all earlier frames.  A query that sees no key gives 0 (and ``lse`` -inf).
    ``scale`` defaults to ``head_dim ** -0.5``.  ``lse``: fp32 ``[Hq, tokens]``
    to be filled.  ``scratch``: uint8, at least :func:`attention_scratch_bytes`
    (allocated here if None).  Returns ``out`` ``[tokens, Hq, head_dim]``."""
    name = "cached_attention"
    dev = _check_cuda(name, q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens, out, lse, scratch)
    nb, hk, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    dt = _half(name, q, "q")
    _rows3(name, q, "q")
    T, hq, dq = q.shape
    _check_shape(name, dq == d, f"q has head_dim {dq}, the cache {d}")
    B = kv_lens.numel()
    _ints(name, block_tables, "block_tables")
    _ints(name, cu_q, "cu_q", (B + 1,))
    _ints(name, kv_lens, "kv_lens")
    _check_shape(name, block_tables.dim() == 2 and block_tables.shape[0] == B,
                 f"block_tables {tuple(block_tables.shape)} must be [{B}, max_blocks]")
    if out is None:
        out = torch.empty((T, hq, d), dtype=q.dtype, device=dev)
    else:
        _rows3(name, out, "out")
        _check_dtype(name, out, q.dtype)
        _check_shape(name, out.shape == q.shape, f"out {tuple(out.shape)} must be {tuple(q.shape)}")
    if lse is not None:
        _check_shape(name, lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == (hq, T),
                     f"lse must be contiguous float32 [{hq}, {T}]")
    with _Dev(dev):
        nbytes = attention_scratch_bytes(T, hq, hk, B, max_q, max_kv, d)
        if scratch is None:
            if nbytes:
                scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        else:
            _check_shape(name, scratch.dtype == torch.uint8 and scratch.is_contiguous() and scratch.numel() >= nbytes,
                         f"scratch must be a contiguous uint8 tensor of >= {nbytes} bytes")
        _lib.call("qvggt_cached_attention", q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0),
                  out.stride(1), None if lse is None else lse.data_ptr(), T, hq, dt, k_cache.data_ptr(),
                  v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(), v_scale.data_ptr(), nb, hk, bs, d,
                  block_tables.data_ptr(), block_tables.shape[1], cu_q.data_ptr(), kv_lens.data_ptr(), B, max_q,
                  max_kv, causal_chunk, d ** -0.5 if scale is None else float(scale),
                  None if scratch is None else scratch.data_ptr(), 0 if scratch is None else scratch.numel(),
                  _stream(q))
    return out


class PagedKVCache:
    """The 8-bit K/V of several layers behind one set of block tables.

    ``num_blocks`` blocks of ``block_size`` tokens are shared by up to
    ``requests`` requests of at most ``max_len`` tokens.  A step::

        plan = cache.plan(target_lens, max_new)        # once: lengths after this step, on the GPU
        for layer in ...:
            cache.append(layer, k, v, plan)            # the new tokens' rows
            o = cache.attend(layer, q, plan, max_q, max_kv, causal_chunk)
        cache.commit(plan)                             # the plan's lengths become the cache's

    Nothing waits for the GPU; :meth:`check` does, and raises if the plan
    could not be served.  One stream at a time."""

    def __init__(self, layers: int, num_blocks: int, kv_heads: int, head_dim: int, requests: int, max_len: int,
                 block_size: int = 64, device="cuda"):
        if block_size not in (32, 64, 128) or head_dim not in (64, 128):
            raise ValueError("PagedKVCache: block_size must be 32, 64 or 128 and head_dim 64 or 128")
        dev = torch.device(device)
        self.block_size = block_size
        shape = (layers, num_blocks, kv_heads, block_size, head_dim)
        self.k = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.v = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.k_scale = torch.ones(shape[:3], dtype=torch.float32, device=dev)
        self.v_scale = torch.ones(shape[:3], dtype=torch.float32, device=dev)
        self.block_tables = torch.full((requests, -(-max_len // block_size)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free_ring = torch.arange(num_blocks, dtype=torch.int32, device=dev)
        self.free_range = torch.tensor([0, num_blocks], dtype=torch.int64, device=dev)
        self._scratch = None

    def plan(self, target_lens, max_new: int) -> BlockPlan:
        """Blocks and slots for ``target_lens`` (int32 ``[requests]`` on the GPU; 0 ends a request)."""
        return block_plan(self.lens, target_lens, self.block_tables, self.free_ring, self.free_range, self.block_size,
                          max_new)

    def append(self, layer: int, k, v, plan: BlockPlan) -> None:
        """Writes the new tokens' k and v ``[tokens, kv_heads, head_dim]`` of one layer."""
        kv_append(k, v, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.block_tables,
                  self.lens, plan.cu_new, plan.cu_blocks)

    def attend(self, layer: int, q, plan: BlockPlan, max_q: int, max_kv: int, causal_chunk: int = 0, out=None):
        """The new tokens' queries over everything the layer holds, the new tokens among it."""
        need = attention_scratch_bytes(q.shape[0], q.shape[1], self.k.shape[2], self.lens.numel(), max_q, max_kv,
                                       self.k.shape[4])
        if need and (self._scratch is None or self._scratch.numel() < need):
            self._scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
        return cached_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                self.block_tables, plan.cu_new, plan.lens, max_q, max_kv, causal_chunk, out=out,
                                scratch=self._scratch if need else None)

    def gather(self, layer: int, slots, dtype=torch.float16):
        """Rows of one layer back as ``[k | v]`` (see :func:`kv_gather`)."""
        return kv_gather(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], slots, dtype)

    def commit(self, plan: BlockPlan) -> None:
        """Adopts the plan's lengths and free blocks."""
        self.lens, self.free_range = plan.lens, plan.free_range

    def check(self, plan: BlockPlan) -> None:
        """Waits for the plan and raises if it could not be served."""
        st = int(plan.status.item())
        if st:
            raise RuntimeError(f"PagedKVCache: {PLAN_STATUS.get(st, st)}; the cache is unchanged")
