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
live on the GPU, so their contents are checked there: what a block id or length
outside its range names is skipped, and the library's status word is set
(``_lib.device_status()``, 0x201 / 0x202); :func:`block_plan` refuses lengths
in its own status.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

from . import _lib
from .awq_inference_engine import _Dev, _check_cuda, _check_dtype, _check_shape, _stream

__all__ = ["rope_axes", "block_plan", "BlockPlan", "kv_append", "kv_gather", "cached_attention",
           "attention_scratch_bytes", "PagedKVCache", "PLAN_STATUS"]

_HALF = {torch.float16: 0, torch.bfloat16: 1}      # QVGGT_DTYPE_F16 / _BF16
_LAYOUTS = {"axial": 0, "split": 1, "interleaved": 2}
_I32, _F32 = torch.int32, torch.float32

PLAN_STATUS = {0: "done", 1: "too few free blocks", 2: "a request needs more blocks than its table row holds",
               3: "a negative length", 4: "more new tokens than max_new",
               5: "the free range is no range of the ring, or more blocks come back than are out"}

# The argument structures of include/qvggt_b200.h: 64-bit fields only.  Packed
# in one go: converting some thirty ctypes arguments took longer than the rest
# of a call.
_ROPE = struct.Struct("=27q").pack
_PLAN = struct.Struct("=16q").pack
_APPEND = struct.Struct("=24q").pack
_GATHER = struct.Struct("=14q").pack
_ATTEND = struct.Struct("=27qd2q").pack

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_functions: dict = {}


def _run(name, dev, t, args):
    """The C call `name` on the current stream of the tensor t's device (index dev)."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.load(), name)
    if _current_device() == dev:
        rc = fn(args, _stream(t))
    else:
        with _Dev(t.device):
            rc = fn(args, _stream(t))
    if rc:
        raise _lib.QvggtError(name, rc, _lib.load().qvggt_last_error().decode(errors="replace"))


def _half(name, t, what):
    code = _HALF.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: {what} must be float16 or bfloat16, got {t.dtype}")
    return code


def _rows3(name, t, what):
    """[tokens, heads, head_dim] with unit stride inside a head; returns its strides."""
    st = t.stride()
    if len(st) != 3 or (st[2] != 1 and t.shape[2] > 1):
        raise ValueError(f"{name}: {what} {tuple(t.shape)} (strides {st}) must be [tokens, heads, head_dim] "
                         "with unit stride in head_dim")
    return st


def _ints(name, t, what, shape=None):
    if t.dtype is not _I32 or not t.is_contiguous():
        raise TypeError(f"{name}: {what} must be contiguous int32, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)} must be {shape}")


def _table(name, t, B):
    _ints(name, t, "block_tables")
    shape = t.shape
    if len(shape) != 2 or shape[0] != B:
        raise ValueError(f"{name}: block_tables {tuple(shape)} must be [{B}, max_blocks]")
    return shape[1]


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
    dev = q.get_device()
    if dev < 0 or not dev == positions.get_device() == inv_freq.get_device():
        _check_cuda(name, q, k, positions, inv_freq)
    dt = _half(name, q, "q")
    sq = _rows3(name, q, "q")
    T, hq, D = q.shape
    axes = len(sections)
    if layout not in _LAYOUTS:
        raise ValueError(f"{name}: layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
    if not 1 <= axes <= 4:
        raise ValueError(f"{name}: 1 to 4 axes, got {axes}")
    if inv_freq.dtype is not _F32 or not inv_freq.is_contiguous() or inv_freq.numel() != sum(sections):
        raise ValueError(f"{name}: inv_freq must be float32 with {sum(sections)} entries")
    sp = positions.stride()
    if positions.dtype is not _I32 or positions.shape != (axes, T) or (sp[1] != 1 and T > 1):
        raise ValueError(f"{name}: positions {tuple(positions.shape)} must be int32 [{axes}, {T}] with unit stride in "
                         "tokens")
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        so = (hq * D, D)
    else:
        so = _out3(name, q_out, q, dev, "q_out")
    if k is None:
        tail = (0,) * 7
        k_out = None
    else:
        if k.get_device() != dev:
            _check_cuda(name, q, k)
        sk = _rows3(name, k, "k")
        _check_dtype(name, k, q.dtype)
        Tk, hk, Dk = k.shape
        if Tk != T or Dk != D:
            raise ValueError(f"{name}: k {tuple(k.shape)} must be [{T}, heads, {D}]")
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
            sko = (hk * D, D)
        else:
            sko = _out3(name, k_out, k, dev, "k_out")
        tail = (k.data_ptr(), sk[0], sk[1], k_out.data_ptr(), sko[0], sko[1], hk)
    _run("qvggt_rope_axes", dev, q,
         _ROPE(q.data_ptr(), sq[0], sq[1], q_out.data_ptr(), so[0], so[1], hq, *tail, T, D, positions.data_ptr(), sp[0],
               inv_freq.data_ptr(), *sections, *(0,) * (4 - axes), axes, _LAYOUTS[layout], 1 if inverse else 0, dt))
    return q_out, k_out


def _out3(name, out, like, dev, what):
    """Strides of a given output that has to match `like`."""
    if out.get_device() != dev:
        _check_cuda(name, like, out)
    st = _rows3(name, out, what)
    _check_dtype(name, out, like.dtype)
    if out.shape != like.shape:
        raise ValueError(f"{name}: {what} {tuple(out.shape)} must be {tuple(like.shape)}")
    return st


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
    returned; if a request cannot be served, or the lengths and the free range
    do not fit the pool, nothing is changed and ``status`` says why.  Block ids
    are handed on as they stand; one outside the pool sets the status word
    (0x201) and its tokens get the slot -1.  ``max_new`` bounds the new tokens."""
    name = "block_plan"
    dev = cached_lens.get_device()
    if dev < 0 or not (dev == target_lens.get_device() == block_tables.get_device() == free_ring.get_device()
                       == free_range.get_device()):
        _check_cuda(name, cached_lens, target_lens, block_tables, free_ring, free_range)
    _ints(name, cached_lens, "cached_lens")
    B = cached_lens.numel()
    _ints(name, target_lens, "target_lens", (B,))
    wide = _table(name, block_tables, B)
    _ints(name, free_ring, "free_ring")
    if free_range.dtype is not torch.int64 or not free_range.is_contiguous() or free_range.numel() != 2:
        raise ValueError(f"{name}: free_range must be int64 [2]")
    # one allocation: the 64-bit pair first, then the 32-bit arrays
    buf = cached_lens.new_empty(3 * B + 7 + max_new)
    free_out, cu_new, cu_blocks, lens, status, slots = buf.split_with_sizes([4, B + 1, B + 1, B, 1, max_new])
    at = buf.data_ptr()
    _run("qvggt_block_plan", dev, buf,
         _PLAN(cached_lens.data_ptr(), target_lens.data_ptr(), B, block_tables.data_ptr(), wide, free_ring.data_ptr(),
               free_ring.numel(), free_range.data_ptr(), block_size, max_new, at + 12 * B + 28, at + 16,
               at + 4 * B + 20, at + 8 * B + 24, at, at + 12 * B + 24))
    return BlockPlan(slots, cu_new, cu_blocks, lens, free_out.view(torch.int64), status)


# --------------------------------------------------------------------- cache
def _check_cache(name, k_cache, v_cache, k_scale, v_scale):
    """Cache tensors -> (num_blocks, kv_heads, block_size, head_dim)."""
    shape, st = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or k_cache.dtype is not torch.int8 or v_cache.dtype is not torch.int8:
        raise TypeError(f"{name}: the caches must be int8 [num_blocks, kv_heads, block_size, head_dim]")
    nb, h, bs, d = shape
    if v_cache.shape != shape or st[1:] != (bs * d, d, 1) or v_cache.stride() != st:
        raise ValueError(f"{name}: K and V caches must have the same shape and strides, dense inside a block")
    if (k_scale.dtype is not _F32 or v_scale.dtype is not _F32 or k_scale.shape != (nb, h) or v_scale.shape != (nb, h)
            or not k_scale.is_contiguous() or not v_scale.is_contiguous()):
        raise ValueError(f"{name}: k_scale and v_scale must be contiguous float32 [{nb}, {h}]")
    return nb, h, bs, d


def kv_append(k, v, k_cache, v_cache, k_scale, v_scale, block_tables, cached_lens, cu_new, cu_blocks,
              max_units: int | None = None):
    """Quantises new rows k, v ``[tokens, kv_heads, head_dim]`` (fp16 / bf16, requests packed as ``cu_new`` says, any
    16-byte aligned token and head strides) into the cache.

    ``cu_new`` and ``cu_blocks`` come from :func:`block_plan`, ``cached_lens``
    are the lengths before.  A block's scale grows when its new rows need it,
    and its earlier codes are rounded to the new scale.  ``max_units``: a
    bound of ``cu_blocks[-1]`` if one tighter than ``tokens // block_size + 2
    * B`` is known; blocks past it are not written, and the status word says so."""
    name = "kv_append"
    dev = k.get_device()
    if dev < 0 or not (dev == v.get_device() == k_cache.get_device() == v_cache.get_device() == k_scale.get_device()
                       == v_scale.get_device() == block_tables.get_device() == cached_lens.get_device()
                       == cu_new.get_device() == cu_blocks.get_device()):
        _check_cuda(name, k, v, k_cache, v_cache, k_scale, v_scale, block_tables, cached_lens, cu_new, cu_blocks)
    nb, h, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    dt = _half(name, k, "k")
    _check_dtype(name, v, k.dtype)
    sk, sv = _rows3(name, k, "k"), _rows3(name, v, "v")
    shape = k.shape
    T = shape[0]
    if shape != (T, h, d) or v.shape != shape:
        raise ValueError(f"{name}: k {tuple(shape)} and v {tuple(v.shape)} must be [tokens, {h}, {d}]")
    B = cached_lens.numel()
    wide = _table(name, block_tables, B)
    _ints(name, cached_lens, "cached_lens")
    _ints(name, cu_new, "cu_new", (B + 1,))
    _ints(name, cu_blocks, "cu_blocks", (B + 1,))
    if max_units is None:
        max_units = T // bs + 2 * B
    _run("qvggt_kv_append", dev, k,
         _APPEND(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(), v_scale.data_ptr(), nb,
                 h, bs, d, k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], T, dt, block_tables.data_ptr(), wide,
                 cached_lens.data_ptr(), cu_new.data_ptr(), cu_blocks.data_ptr(), B, max_units))


def kv_gather(k_cache, v_cache, k_scale, v_scale, slots, dtype=torch.float16, out=None):
    """The cache rows of ``slots`` (int32 ``[n]``) as ``[n, 2 * kv_heads * head_dim]`` rows ``[k | v]``, the layout
    :func:`~qvggt_b200.awq_inference_engine.attention` reads; a negative slot gives zeros."""
    name = "kv_gather"
    dev = slots.get_device()
    if dev < 0 or not (dev == k_cache.get_device() == v_cache.get_device() == k_scale.get_device()
                       == v_scale.get_device()):
        _check_cuda(name, k_cache, v_cache, k_scale, v_scale, slots)
    nb, h, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    _ints(name, slots, "slots")
    n = slots.numel()
    if out is None:
        out = slots.new_empty((n, 2 * h * d), dtype=dtype)
    elif out.get_device() != dev:
        _check_cuda(name, slots, out)
    if out.shape != (n, 2 * h * d) or out.stride()[1] != 1:
        raise ValueError(f"{name}: out {tuple(out.shape)} must be [{n}, {2 * h * d}]")
    dt = _half(name, out, "out")
    _run("qvggt_kv_gather", dev, slots,
         _GATHER(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(), v_scale.data_ptr(), nb,
                 h, bs, d, slots.data_ptr(), n, out.data_ptr(), out.stride(0), dt))
    return out


# ----------------------------------------------------------------- attention
@functools.lru_cache(maxsize=1024)
def _scratch_bytes(dev, *sizes):
    nb = C.c_int64(0)
    with torch.cuda.device(dev):
        _lib.call("qvggt_cached_attention_scratch", *sizes, C.byref(nb))
    return int(nb.value)


def attention_scratch_bytes(tokens: int, q_heads: int, kv_heads: int, requests: int, max_q: int, max_kv: int,
                            head_dim: int) -> int:
    """Scratch :func:`cached_attention` needs for these sizes on the current device."""
    return _scratch_bytes(_current_device(), tokens, q_heads, kv_heads, requests, max_q, max_kv, head_dim)


def cached_attention(q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens, max_q: int, max_kv: int,
                     causal_chunk: int = 0, scale: float | None = None, out=None, lse=None, scratch=None):
    """``softmax(scale q k^T + mask) v`` over the 8-bit cache, for requests of any lengths.

    q ``[tokens, Hq, head_dim]`` fp16 / bf16: request b's queries are rows
    ``cu_q[b]`` to ``cu_q[b + 1]`` (at most ``max_q``), its keys the first
    ``kv_lens[b]`` tokens of table row b (``max_kv``: about the longest; it
    sets how the work is split).  ``Hq`` is a multiple of the cache's heads.
    Query i of ql sits at position ``kv_len - ql + i``.  ``causal_chunk`` 0:
    every query sees every key; 1: causal; the tokens of a frame: its own and
    all earlier frames.  A query that sees no key gives 0 (and ``lse`` -inf);
    rows outside ``cu_q``, and those of a request that is skipped for its
    lengths (status word 0x202), are left as they are.  ``scale``: positive
    (more than 1e-30, at most 1e30), ``head_dim ** -0.5`` by default.  The V
    scales of one request's blocks may lie 2^80 apart.  ``lse``: fp32 ``[Hq, tokens]``
    to be filled.  ``scratch``: uint8, at least :func:`attention_scratch_bytes`
    (allocated here if None).  Returns ``out`` ``[tokens, Hq, head_dim]``."""
    name = "cached_attention"
    dev = q.get_device()
    if dev < 0 or not (dev == k_cache.get_device() == v_cache.get_device() == k_scale.get_device()
                       == v_scale.get_device() == block_tables.get_device() == cu_q.get_device()
                       == kv_lens.get_device()):
        _check_cuda(name, q, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens)
    nb, hk, bs, d = _check_cache(name, k_cache, v_cache, k_scale, v_scale)
    dt = _half(name, q, "q")
    sq = _rows3(name, q, "q")
    T, hq, dq = q.shape
    if dq != d:
        raise ValueError(f"{name}: q has head_dim {dq}, the cache {d}")
    B = kv_lens.numel()
    wide = _table(name, block_tables, B)
    _ints(name, cu_q, "cu_q", (B + 1,))
    _ints(name, kv_lens, "kv_lens")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        so = (hq * d, d)
    else:
        so = _out3(name, out, q, dev, "out")
    if lse is None:
        lse_at = 0
    else:
        if lse.get_device() != dev:
            _check_cuda(name, q, lse)
        _check_shape(name, lse.dtype is _F32 and lse.is_contiguous() and lse.shape == (hq, T),
                     f"lse must be contiguous float32 [{hq}, {T}]")
        lse_at = lse.data_ptr()
    nbytes = _scratch_bytes(dev, T, hq, hk, B, max_q, max_kv, d)
    scratch_at = scratch_len = 0
    if scratch is not None:
        if scratch.get_device() != dev:
            _check_cuda(name, q, scratch)
        scratch_len = scratch.numel()
        _check_shape(name, scratch.dtype is torch.uint8 and scratch.is_contiguous() and scratch_len >= nbytes,
                     f"scratch must be a contiguous uint8 tensor of >= {nbytes} bytes")
        scratch_at = scratch.data_ptr()
    elif nbytes:
        scratch = q.new_empty(nbytes, dtype=torch.uint8)
        scratch_at, scratch_len = scratch.data_ptr(), nbytes
    _run("qvggt_cached_attention", dev, q,
         _ATTEND(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0), k_scale.data_ptr(), v_scale.data_ptr(), nb,
                 hk, bs, d, q.data_ptr(), sq[0], sq[1], out.data_ptr(), so[0], so[1], lse_at, T, hq, dt,
                 block_tables.data_ptr(), wide, cu_q.data_ptr(), kv_lens.data_ptr(), B, max_q, max_kv, causal_chunk,
                 d ** -0.5 if scale is None else scale, scratch_at, scratch_len))
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
    could not be served (its tokens then have no place: :meth:`append` writes
    nothing and :meth:`attend` leaves its output as allocated).  One stream at
    a time.  :meth:`commit` takes the plan's tensors for the cache's, so a step
    captured in a CUDA graph would start from the same lengths at each replay."""

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
