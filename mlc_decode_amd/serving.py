"""A serving step around the paged decode: the torch-facing entry points.

* ``reserve_pages(pool, block_table, cache_seqlens, new_lens, num_tokens)`` ->
  ``Reservation(slots, positions, cu_new, granted)``: pages, block tables and the slot map of a step's new
  tokens, from the request lengths, on the GPU; ``release_pages(pool, block_table, cache_seqlens,
  keep_lens)`` shortens sequences (rejected drafts, finished requests) and returns their pages.
* ``rope_plan(...)`` -> ``Rope`` and ``apply_rope(x, positions, rope)``: rotary positions.
* ``kv_append_slots(kv_new, kv_cache, slots, positions, rope, q_pe, q)``: the step's tokens, packed and
  ragged, into the cache rows a slot map names, rotated on the way, together with the queries' rope parts.
* ``kv_gather(kv_cache, slots)``: cached tokens as rows (what a chunked prefill attends to).

A decode step is ``reserve_pages`` -> ``kv_append_slots`` -> ``get_mla_metadata`` ->
``flash_mla_with_kvcache`` (the last two per step and per layer, api.py).  Every cache format the decode
takes is taken here.  Calls are queued on torch's current stream of the tensors' device, synchronise
nothing, and can be captured in a HIP graph.  The reference decodes a pre-filled cache with rotated inputs
and has no counterpart of these.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import (MLA_DIM_QK, MLA_DIM_V, MLA_DTYPE_BF16, MLA_DTYPE_F16, MLA_DTYPE_F32, MLA_KV_NATIVE, MLA_ROPE_HALF,
                   MLA_ROPE_INTERLEAVED, MlaAppendSlotsArgs, MlaKvCache, MlaPagePool, MlaRope, MlaRopeArgs, check)
from .api import _cache_format, _check_coded_cache, _launch, _require_gpu, _split_kv

_DTYPES = {torch.bfloat16: MLA_DTYPE_BF16, torch.float16: MLA_DTYPE_F16, torch.float32: MLA_DTYPE_F32}
_LAYOUTS = {"interleaved": MLA_ROPE_INTERLEAVED, "half": MLA_ROPE_HALF}
_ROPE_DIM = MLA_DIM_QK - MLA_DIM_V
_PAGE = _lib.MLA_PAGE_TOKENS
_FLT_MAX = 3.4028234663852886e38

# filled by one struct.pack each, like the decode's arguments (api.py)
_CACHE = struct.Struct("=4i3Q6q")
_ROPE = struct.Struct("=Q2ifi")
_ROPE_ARGS = struct.Struct("=2Q4qQ6i")
_APPEND = struct.Struct("=Qq4Q4q2i")
_POOL = struct.Struct("=2Q2iQ2iQ")
for _s, _c in ((_CACHE, MlaKvCache), (_ROPE, MlaRope), (_ROPE_ARGS, MlaRopeArgs), (_APPEND, MlaAppendSlotsArgs), (_POOL, MlaPagePool)):
    assert _s.size == ctypes.sizeof(_c)


def _require(t: torch.Tensor, name: str, device: Optional[torch.device] = None) -> None:
    at = t.get_device()  # -1: not on a GPU
    if at < 0:
        _require_gpu(t, name)
    if device is not None and at != device.index:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _require_int32(t: torch.Tensor, name: str, n: int, device: torch.device) -> None:
    if t.get_device() != device.index:
        _require(t, name, device)
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] int32 tensor")


# ---------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------
class Rope(NamedTuple):
    """A rotation plan: ``freqs`` float64 ``[dim / 2]`` on the GPU, turns per position of each pair; ``layout``
    "interleaved" (pairs 2i, 2i + 1) or "half" (pairs i, i + dim / 2); ``amp`` multiplies cosine and sine.
    Made by :func:`rope_plan`, or from frequencies of one's own."""
    freqs: torch.Tensor
    layout: str = "interleaved"
    amp: float = 1.0


def rope_frequencies(dim: int = _ROPE_DIM, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                     original_max: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, mscale: float = 1.0,
                     mscale_all_dim: float = 0.0):
    """``(turns per position [dim / 2], amp)`` of :func:`rope_plan`, in Python floats (64 bits)."""
    if dim < 2 or dim % 2:
        raise ValueError("dim must be even and at least 2")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError("base must be above 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if scaling is not None and not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling takes dim >= 4")
        base *= factor ** (dim / (dim - 2))
    turns = [base ** (-2 * i / dim) / (2 * math.pi) for i in range(dim // 2)]
    amp = 1.0
    if scaling == "linear":
        turns = [t / factor for t in turns]
    elif scaling == "yarn":
        if not (original_max > 0 and beta_fast > 0 and beta_slow > 0):
            raise ValueError("yarn scaling takes positive original_max, beta_fast and beta_slow")
        # the (fractional) pair that turns `beta` times over the original context
        edge = lambda beta: dim * math.log(original_max / (beta * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(edge(beta_fast)), 0), min(math.ceil(edge(beta_slow)), dim - 1)
        span = max(high - low, 0.001)
        for i, t in enumerate(turns):
            ramp = min(1.0, max(0.0, (i - low) / span))
            turns[i] = t / factor * ramp + t * (1.0 - ramp)
        grow = lambda m: 0.1 * m * math.log(factor) + 1.0  # noqa: E731
        amp = grow(mscale) / grow(mscale_all_dim)
    return turns, amp


def rope_plan(dim: int = _ROPE_DIM, base: float = 10000.0, layout: str = "interleaved", scaling: Optional[str] = None,
              factor: float = 1.0, original_max: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
              mscale: float = 1.0, mscale_all_dim: float = 0.0, device="cuda") -> Rope:
    """The rotation of ``dim`` dims with pair i at ``base ** (-2i / dim)`` radians per position; made once.

    ``scaling`` for contexts longer than trained on: "linear" (positions divided by ``factor``), "ntk" (the
    base grown so that the slowest pair slows by ``factor``), "yarn" (pairs that turn more than
    ``beta_fast`` times over ``original_max`` positions keep their speed, those below ``beta_slow`` are
    slowed by ``factor``, a linear ramp between; cosine and sine times
    ``(0.1 mscale ln factor + 1) / (0.1 mscale_all_dim ln factor + 1)``)."""
    if layout not in _LAYOUTS:
        raise ValueError("layout must be 'interleaved' or 'half'")
    turns, amp = rope_frequencies(dim, base, scaling, factor, original_max, beta_fast, beta_slow, mscale, mscale_all_dim)
    return Rope(torch.tensor(turns, dtype=torch.float64, device=device), layout, amp)


def _rope_struct(rope: Rope, device: torch.device) -> MlaRope:
    freqs, layout, amp = rope
    _require(freqs, "rope.freqs", device)
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or freqs.numel() < 1 or not freqs.is_contiguous():
        raise ValueError("rope.freqs must be a contiguous 1-D float64 tensor")
    if layout not in _LAYOUTS:
        raise ValueError("rope.layout must be 'interleaved' or 'half'")
    amp = float(amp)
    if not abs(amp) <= _FLT_MAX:
        raise ValueError("rope.amp must be finite")
    return MlaRope.from_buffer_copy(_ROPE.pack(freqs.data_ptr(), 2 * freqs.numel(), _LAYOUTS[layout], amp, 0))


def _rows(x: torch.Tensor):
    """``(tokens, heads, token stride, head stride)`` of ``[..., H, D]``: the leading dims as one."""
    if x.dim() == 3:
        tokens, heads, _ = x.shape
        stride, head_stride, _ = x.stride()
        return tokens, heads, stride if tokens > 1 else 0, head_stride if heads > 1 else 0
    tokens, stride = 1, 0
    for n, s in zip(reversed(x.shape[:-2]), reversed(x.stride()[:-2])):
        if n == 1:
            continue
        if tokens == 1:
            stride = s
        elif s != tokens * stride:
            return None
        tokens *= n
    return tokens, x.shape[-2], stride, x.stride(-2) if x.shape[-2] > 1 else 0


def apply_rope(x: torch.Tensor, positions: torch.Tensor, rope: Rope, first: Optional[int] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate dims ``[first, first + dim)`` of every head of ``x [..., H, D]`` (bf16, fp16 or fp32) by its token's
    position -> ``out`` of the same shape and dtype, the other dims copied.

    ``positions`` int32 of shape ``x.shape[:-2]`` (a negative one leaves its row unrotated); ``first`` defaults to
    ``D - dim``, the last dims, where MLA keeps them; ``out`` defaults to a new tensor, and may be ``x``
    itself (in place); it may not overlap it otherwise.  Heads may be strided, a head's dims are contiguous;
    the token dims of each must be one stride apart."""
    _require(x, "x")
    device = x.device
    if x.dtype not in _DTYPES:
        raise ValueError("x must be bfloat16, float16 or float32")
    if x.dim() < 3:
        raise ValueError("x must be [..., H, D]")
    if positions.shape != x.shape[:-2]:
        raise ValueError("positions must have x's shape without its last two dims")
    _require(positions, "positions", device)
    if positions.dtype != torch.int32 or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 tensor")
    r = _rope_struct(rope, device)
    D = x.shape[-1]
    if first is None:
        first = D - r.dim
    if not 0 <= first <= D - r.dim:
        raise ValueError("the rotated dims [first, first + dim) must lie in the head")
    fresh = out is None
    if fresh:
        out = torch.empty(x.shape, dtype=x.dtype, device=device)
    else:
        _require(out, "out", device)
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("out must have x's shape and dtype")
    if x.numel() == 0:
        return out
    xr = _rows(x)
    if xr is not None:
        tokens, heads, x_t, x_h = xr
        orr = (tokens, heads, heads * D, D) if fresh else _rows(out)
    if xr is None or orr is None or (D > 1 and (x.stride(-1) != 1 or out.stride(-1) != 1)):
        raise ValueError("x and out must have unit stride in their last dim and token dims one stride apart")
    o_t, o_h = orr[2:]
    x_ptr, o_ptr = x.data_ptr(), out.data_ptr()
    if not fresh:
        if _rows_meet((o_t, o_h), (tokens, heads), D):
            raise ValueError("out's rows overlap")
        if not _apart_or_same(x_ptr, (x_t, x_h), o_ptr, (o_t, o_h), (tokens, heads), D, x.element_size()):
            raise ValueError("out overlaps x without being x")
    a = MlaRopeArgs.from_buffer_copy(_ROPE_ARGS.pack(
        x_ptr, o_ptr, x_t, x_h, o_t, o_h, positions.data_ptr(), tokens, heads, D, first, _DTYPES[x.dtype], 0))
    _launch("mla_apply_rope", _lib.load().mla_apply_rope, device, ctypes.byref(r), ctypes.byref(a))
    return out


def _rows_meet(strides, counts, width: int, shift: int = 0) -> bool:
    """Whether any two of ``counts[0] * counts[1]`` rows of ``width`` elements at these strides overlap; with a ``shift``,
    whether a row and one of the same rows that many elements on do."""
    (st, sh), (t, h), d = strides, counts, abs(shift)
    if (d == 0 or d >= width) and (h == 1 or sh >= d + width) and (t == 1 or st >= (h - 1) * sh + d + width):
        return False  # the usual layouts: heads side by side, token after token
    (s0, n0), (s1, n1) = sorted((s if n > 1 else 0, n) for s, n in zip(strides, counts))
    if shift == 0 and ((n0 > 1 and s0 < width) or (n1 > 1 and s1 < width)):
        return True
    reach = 0 if s1 == 0 else min(n1 - 1, ((n0 - 1) * s0 + abs(shift) + width) // s1)
    for k1 in range(-reach, reach + 1):  # as far as the other stride's rows reach
        at = shift + k1 * s1
        near = 0 if s0 == 0 else -at // s0
        for k0 in (near, near + 1):
            k0 = min(max(k0, 1 - n0), n0 - 1)
            if abs(at + k0 * s0) < width and (shift or k0 or k1):
                return True
    return False


def _apart_or_same(x_ptr: int, xs, o_ptr: int, os, counts, width: int, es: int) -> bool:
    """Whether two sets of rows of ``width`` elements at the given strides are the same memory, row for row, or do
    not meet: apart, or parts of the same wider rows (``w[..., :a]`` and ``w[..., a:]``)."""
    if x_ptr == o_ptr:
        return xs == os
    t, h = counts[0] - 1, counts[1] - 1
    if x_ptr >= o_ptr + es * (t * os[0] + h * os[1] + width) or o_ptr >= x_ptr + es * (t * xs[0] + h * xs[1] + width):
        return True
    return xs == os and not _rows_meet(xs, counts, width, (o_ptr - x_ptr) // es)


# ---------------------------------------------------------------------------------------
# appending and reading by slot
# ---------------------------------------------------------------------------------------
def _cache_struct(kv_cache, device: Optional[torch.device]) -> tuple:
    """``(mla_kv_cache, dtype, device)`` of a cache in any of its forms."""
    fmt = _cache_format(kv_cache)
    rope_offset, scale_args = 0, (0, 0, 0)
    others = ()
    if fmt != MLA_KV_NATIVE:
        latent, scale, rope = _check_coded_cache(kv_cache)
        dtype = torch.bfloat16
        page, block, _ = scale.stride()
        scale_args = (scale.data_ptr(), page, block)
        others = (scale, rope)
    else:
        if isinstance(kv_cache, (tuple, list)):
            latent, rope = _split_kv(kv_cache)
            others = (rope,)
        else:
            latent = rope = kv_cache
            if kv_cache.shape[-1] != MLA_DIM_QK:
                raise ValueError(f"kv_cache last dim must be {MLA_DIM_QK}")
            rope_offset = 2 * MLA_DIM_V
        dtype = latent.dtype
        for t in (latent, *others):
            if t.dtype not in (torch.bfloat16, torch.float16) or t.dtype != dtype:
                raise ValueError("the cache must be bfloat16 or float16")
            if t.dim() != 4 or t.shape[1] != _PAGE or t.shape[2] != 1 or t.stride(-1) != 1:
                raise ValueError("kv cache must be [num_blocks, 64, 1, D] with unit stride in D")
        if latent.shape[0] != rope.shape[0]:
            raise ValueError("the cache's halves have different page counts")
    if device is None:
        device = latent.device
    for t in (latent, *others):
        if t.get_device() != device.index or device.index is None:
            _require(t, "kv_cache", device)
    (sp, st, *_), (rp, rt, *_) = latent.stride(), rope.stride()
    c = MlaKvCache.from_buffer_copy(_CACHE.pack(
        fmt, _DTYPES[dtype], latent.shape[0], 0, latent.data_ptr(), rope.data_ptr() + rope_offset, scale_args[0],
        sp, st, rp, rt, scale_args[1], scale_args[2]))
    return c, dtype, device


def kv_append_slots(kv_new: torch.Tensor, kv_cache, slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
                    rope: Optional[Rope] = None, q_pe: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None) -> None:
    """Write ``kv_new [T, 576]`` (latent, then rope dims; the cache's dtype, bf16 for the coded caches) to cache
    rows ``slots [T]`` (int32, page * 64 + row), the rope dims rotated by ``positions [T]`` (int32) if a ``rope``
    of 64 dims is given.

    With ``q_pe [T, H, 64]``, the rope parts of the step's queries, they are rotated into the last 64 dims of
    ``q [T, H, 576]``, the decode's query buffer (``q_pe`` may be those dims themselves), in the same launch.  A slot outside the cache (-1: a row not
    granted, or behind the last sequence) names no row: nothing is written for that token, in the cache or in
    ``q``.  No two rows may have the same slot.  Unlike ``kv_append`` this takes any number of tokens per
    sequence, and does not advance lengths (``reserve_pages`` did)."""
    _require(kv_new, "kv_new")
    device = kv_new.device
    c, dtype, _ = _cache_struct(kv_cache, device)
    if kv_new.dim() != 2 or kv_new.shape[1] != MLA_DIM_QK or kv_new.dtype != dtype or kv_new.stride(1) != 1:
        raise ValueError(f"kv_new must be a [T, {MLA_DIM_QK}] tensor in the cache's dtype ({dtype}) with unit stride in its rows")
    T = kv_new.shape[0]
    _require_int32(slots, "slots", T, device)
    r = None
    if rope is not None:
        if positions is None:
            raise ValueError("a rope needs positions")
        r = _rope_struct(rope, device)
        if r.dim != _ROPE_DIM:
            raise ValueError(f"the rope must rotate {_ROPE_DIM} dims")
    if positions is not None:
        _require_int32(positions, "positions", T, device)
    heads, q_args = 0, (0, 0, 0, 0, 0, 0)
    if (q_pe is None) != (q is None):
        raise ValueError("q_pe and q come together")
    if q_pe is not None:
        if rope is None:
            raise ValueError("q_pe is rotated: it needs a rope")
        _require(q_pe, "q_pe", device)
        _require(q, "q", device)
        heads = q_pe.shape[1] if q_pe.dim() == 3 else 0
        if q_pe.dim() != 3 or q_pe.shape != (T, heads, _ROPE_DIM) or q_pe.dtype != dtype or (q_pe.numel() and q_pe.stride(2) != 1):
            raise ValueError(f"q_pe must be a [T, H, {_ROPE_DIM}] tensor in the cache's dtype with unit stride in its heads")
        if q.shape != (T, heads, MLA_DIM_QK) or q.dtype != dtype or (q.numel() and q.stride(2) != 1):
            raise ValueError(f"q must be a [T, H, {MLA_DIM_QK}] tensor like q_pe with unit stride in its heads")
        (_, _, pe_t, pe_h), (_, _, q_t, q_h) = _rows(q_pe), _rows(q)
        if T * heads and _rows_meet((q_t, q_h), (T, heads), MLA_DIM_QK):
            raise ValueError("q's rows overlap")
        pe_ptr, q_ptr = q_pe.data_ptr(), q.data_ptr() + 2 * MLA_DIM_V
        if T * heads and not _apart_or_same(pe_ptr, (pe_t, pe_h), q_ptr, (q_t, q_h), (T, heads), _ROPE_DIM, 2):
            raise ValueError("q's rope dims overlap q_pe without being it")
        q_args = (pe_ptr, q_ptr, pe_t, pe_h, q_t, q_h)
    a = MlaAppendSlotsArgs.from_buffer_copy(_APPEND.pack(
        kv_new.data_ptr(), kv_new.stride(0) if T > 1 else 0, slots.data_ptr(),
        positions.data_ptr() if positions is not None else 0, *q_args, T, heads))
    _launch("mla_kv_append_slots", _lib.load().mla_kv_append_slots, device, ctypes.byref(c),
            ctypes.byref(r) if r is not None else None, ctypes.byref(a))


def kv_gather(kv_cache, slots: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The cached tokens ``slots [T]`` (int32, page * 64 + row) as rows ``[T, 576]`` in the cache's dtype.  The coded caches
    give bf16, exactly: a code times its scale fits it, up to its range (an fp8 block whose largest latent is
    ``1.9375 * 2**127`` or more can hold a code past it, which reads as an infinity; the 4-bit appends store none).
    A slot outside the cache gives a row of zeros."""
    c, dtype, device = _cache_struct(kv_cache, None)
    if slots.dim() != 1:
        raise ValueError("slots must be a 1-D int32 tensor")
    T = slots.shape[0]
    _require_int32(slots, "slots", T, device)
    if out is None:
        out = torch.empty(T, MLA_DIM_QK, dtype=dtype, device=device)
    else:
        _require(out, "out", device)
        if out.shape != (T, MLA_DIM_QK) or out.dtype != dtype or out.stride(1) != 1:
            raise ValueError(f"out must be a [T, {MLA_DIM_QK}] tensor in the cache's dtype with unit stride in its rows")
    _launch("mla_kv_gather", _lib.load().mla_kv_gather, device, ctypes.byref(c), slots.data_ptr(), T, out.data_ptr(),
            out.stride(0) if T > 1 else MLA_DIM_QK)
    return out


# ---------------------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------------------
class PagePool(NamedTuple):
    """The free pages of a cache, a stack: the first ``count[0]`` entries of ``free_pages`` (int32 ``[num_blocks]``) are
    free and the last of them is taken next; ``count`` int32 ``[1]``.  Made by :func:`page_pool`."""
    free_pages: torch.Tensor
    count: torch.Tensor


class Reservation(NamedTuple):
    """What :func:`reserve_pages` gives: ``slots [T]`` and ``positions [T]`` of the step's packed rows (-1: a row not
    granted, or behind the last sequence), ``cu_new [B + 1]`` (sequence b's rows start at ``cu_new[b]``) and
    ``granted [B]`` (1 or 0), all int32."""
    slots: torch.Tensor
    positions: torch.Tensor
    cu_new: torch.Tensor
    granted: torch.Tensor


def page_pool(num_blocks: int, device="cuda") -> PagePool:
    """A pool of ``num_blocks`` free pages; page 0 is taken first."""
    if num_blocks < 1:
        raise ValueError("num_blocks must be at least 1")
    return PagePool(torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device),
                    torch.full((1,), num_blocks, dtype=torch.int32, device=device))


def _pool_struct(pool: PagePool, block_table: torch.Tensor, cache_seqlens: torch.Tensor):
    _require(block_table, "block_table")
    device = block_table.device
    if block_table.dtype is not torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be a [B, P] int32 tensor with unit column stride")
    (B, P), (stride, unit) = block_table.shape, block_table.stride()
    if P > 1 and unit != 1:
        raise ValueError("block_table must be a [B, P] int32 tensor with unit column stride")
    if P < 1 or (B > 1 and stride < P):
        raise ValueError("block_table must have columns, and rows that do not overlap")
    _require_int32(cache_seqlens, "cache_seqlens", B, device)
    free, count = pool
    pages = free.numel()
    _require_int32(free, "pool.free_pages", pages, device)
    _require_int32(count, "pool.count", 1, device)
    if B <= 1:
        stride = P
    if stride >= 2 ** 31:
        raise ValueError("block_table's row stride must be below 2^31")
    s = MlaPagePool.from_buffer_copy(_POOL.pack(
        free.data_ptr(), count.data_ptr(), pages, B, block_table.data_ptr(), stride, P, cache_seqlens.data_ptr()))
    return s, B, device


def reserve_pages(pool: PagePool, block_table: torch.Tensor, cache_seqlens: torch.Tensor, new_lens: torch.Tensor,
                  num_tokens: int) -> Reservation:
    """Room in the cache for ``new_lens[b]`` more tokens of every sequence (int32 ``[B]``; 0 or less: none): takes the
    pages they need from ``pool``, writes them into ``block_table [B, P]``, advances ``cache_seqlens [B]``, all in
    place, and maps the step's ``num_tokens`` packed rows (the sum of ``new_lens``, or more: a captured step's
    size) to cache slots and positions.

    Requests are served in order.  One whose table row or token rows are too short, or for which the pool runs
    out, gets nothing (``granted[b] = 0``, slots -1, its length and table as they were), and neither does any
    later one that needs a page the earlier requests, granted or not, asked for first.  Which pages are taken
    depends only on the inputs.  Calls on one pool must be ordered."""
    s, B, device = _pool_struct(pool, block_table, cache_seqlens)
    _require_int32(new_lens, "new_lens", B, device)
    num_tokens = int(num_tokens)
    if not 0 <= num_tokens < 2 ** 31:
        raise ValueError("num_tokens must be in [0, 2^31)")
    buf = torch.empty(2 * num_tokens + 3 * B + 2, dtype=torch.int32, device=device)
    slots = buf.data_ptr()
    positions, cu_new = slots + 4 * num_tokens, slots + 8 * num_tokens
    granted, scratch = cu_new + 4 * (B + 1), cu_new + 4 * (2 * B + 1)
    _launch("mla_reserve_pages", _lib.load().mla_reserve_pages, device, ctypes.byref(s), new_lens.data_ptr(), num_tokens, slots,
            positions, cu_new, granted, scratch)
    return Reservation(*buf.split_with_sizes((num_tokens, num_tokens, B + 1, B, B + 1))[:4])


def release_pages(pool: PagePool, block_table: torch.Tensor, cache_seqlens: torch.Tensor, keep_lens: torch.Tensor) -> None:
    """Shorten every sequence to ``keep_lens[b]`` tokens (int32 ``[B]``; 0: it is done, its length or more: nothing
    changes) and return the pages it no longer needs to ``pool``, in place.  The pages go back in the order they
    came: releasing what ``reserve_pages`` took restores the stack.  ``block_table`` keeps stale entries; one that is no
    page of the pool is not put back."""
    s, B, device = _pool_struct(pool, block_table, cache_seqlens)
    _require_int32(keep_lens, "keep_lens", B, device)
    _launch("mla_release_pages", _lib.load().mla_release_pages, device, ctypes.byref(s), keep_lens.data_ptr())
