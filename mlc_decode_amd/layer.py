"""Around the attention in a layer: the torch-facing entry points.

* ``rms_norm(x, weight, eps, residual)``: the residual's addition and the root-mean-square norm, to rows in x's dtype or
  to 8-bit rows with scales (``Fp8Rows``).
* ``linear_fp4(x, w)``: a projection of few rows, 16-bit or 8-bit ones, by 4-bit weights (``Fp4Weight``) that
  ``quantize_w_fp4(w)`` makes from a matrix and ``pack_w_fp4(codes, scale)`` from codes at hand; ``mla_decode_absorbed``
  takes one as its ``w_o``.

Calls are queued on torch's current stream of the tensors' device, synchronise nothing, and can be captured in a HIP graph.
The reference starts at rotated, projected inputs and has no counterpart of these.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import MLA_DTYPE_BF16, MLA_DTYPE_F16, MLA_DTYPE_F32, MlaLinearArgs, MlaRmsNormArgs
from .api import _launch, _stream_ptr, _workspace, new_tensor
from .serving import _FLT_MAX, _apart_or_same, _require, _rows_meet

_DTYPES = {torch.bfloat16: MLA_DTYPE_BF16, torch.float16: MLA_DTYPE_F16, torch.float32: MLA_DTYPE_F32}
_NORM = struct.Struct("=6Q4q4ifi")
_LINEAR = struct.Struct("@6Q3q6iQq")
assert _NORM.size == ctypes.sizeof(MlaRmsNormArgs) and _LINEAR.size == ctypes.sizeof(MlaLinearArgs)
GROUP = 32  # dims that share a scale


class Fp8Rows(NamedTuple):
    """Rows in 8 bits: ``codes`` uint8 ``[..., D]`` (OCP e4m3) and ``scale`` uint8 ``[..., D / 32]``: value d of a row is
    ``e4m3(codes[d]) * 2**(scale[d // 32] - 127)``, scale bytes 1 .. 254 (255: the block holds a NaN or an infinity).
    Made by ``rms_norm(..., quantize=True)``."""
    codes: torch.Tensor
    scale: torch.Tensor


def _token_rows(t: torch.Tensor) -> Optional[Tuple[int, int]]:
    """``(tokens, stride)`` of ``[..., D]``: the leading dims as one; None where they are not one stride apart."""
    if t.dim() == 2:
        n = t.shape[0]
        return n, t.stride(0) if n > 1 else 0
    if 0 in t.shape:
        return 0, 0
    tokens, stride = 1, 0
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if tokens == 1:
            stride = s
        elif s != tokens * stride:
            return None
        tokens *= n
    return tokens, stride


def _norm_rows(t: torch.Tensor, name: str, x: torch.Tensor) -> int:
    """The row stride of a tensor shaped like ``x``, checked."""
    if t.get_device() != x.get_device():
        _require(t, name, x.device)
    if t.shape != x.shape or t.dtype is not x.dtype or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must have x's shape and dtype, and unit stride in its rows")
    rows = _token_rows(t)
    if rows is None:
        raise ValueError(f"{name} must have token dims one stride apart")
    return rows[1]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
             quantize: bool = False) -> Union[torch.Tensor, Fp8Rows, Tuple[Union[torch.Tensor, Fp8Rows], torch.Tensor]]:
    """``y = h / sqrt(mean(h**2) + eps) * weight`` over the last dim of ``h = x`` or ``h = x + residual`` -> ``y``, or with a
    ``residual`` ``(y, h)``.

    ``x [..., D]`` in bf16, fp16 or fp32, ``residual`` like it, ``weight [D]`` in x's dtype or fp32.  ``h`` is added, squared
    and summed in fp32 (a row whose squares add up past its range gives zeros); y is of h as added, and both are rounded once, to x's dtype.  With ``quantize`` y is
    :class:`Fp8Rows`, rounded from fp32 (D a multiple of 32), what ``linear_fp4`` reads.  ``out`` and ``residual_out``
    default to new tensors; each may be ``x`` or ``residual`` itself (in place), and may not overlap them otherwise, nor
    each other, nor ``weight``.  Rows may be strided (the latent part of ``kv [T, 576]`` before it is appended); the token dims of each
    tensor must be one stride apart."""
    index = x.get_device()
    if index < 0:
        _require(x, "x")
    device, dtype, shape = x.device, x.dtype, x.shape
    kind = _DTYPES.get(dtype)
    if kind is None:
        raise ValueError("x must be bfloat16, float16 or float32")
    if len(shape) < 2 or shape[-1] < 1:
        raise ValueError("x must be [..., D], D at least 1")
    D = shape[-1]
    rows = _token_rows(x)
    if rows is None or (D > 1 and x.stride(-1) != 1):
        raise ValueError("x must have unit stride in its rows, and token dims one stride apart")
    tokens, x_t = rows
    if tokens >= 2 ** 24:
        raise ValueError("x must have fewer than 2**24 rows")
    if weight.get_device() != index:
        _require(weight, "weight", device)
    if weight.shape != (D,) or not weight.is_contiguous() or weight.dtype not in (dtype, torch.float32):
        raise ValueError(f"weight must be a contiguous [{D}] tensor in x's dtype or float32")
    eps = float(eps)
    if not 0.0 <= eps <= _FLT_MAX:
        raise ValueError("eps must be finite in fp32 and at least 0")
    r_ptr, r_t, h, h_ptr, h_t = 0, 0, None, 0, 0
    if residual is not None:
        r_ptr, r_t = residual.data_ptr(), _norm_rows(residual, "residual", x)
        h = residual_out
        if h is None:
            h, h_t = torch.empty_like(x, memory_format=torch.contiguous_format), D
        else:
            h_t = _norm_rows(h, "residual_out", x)
        h_ptr = h.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out is the sum with a residual: it needs one")
    scale, scale_ptr = None, 0
    if quantize:
        if out is not None:
            raise ValueError("8-bit rows are new tensors: no out")
        if D % GROUP:
            raise ValueError(f"8-bit rows take a D that is a multiple of {GROUP}")
        y = new_tensor(shape, torch.uint8, device)
        scale = new_tensor((*shape[:-1], D // GROUP), torch.uint8, device)
        y_t, scale_ptr = D, scale.data_ptr()
    elif out is None:
        y, y_t = torch.empty_like(x, memory_format=torch.contiguous_format), D
    else:
        y, y_t = out, _norm_rows(out, "out", x)
    y_ptr = y.data_ptr()
    if tokens and (out is not None or residual_out is not None):
        _norm_overlaps(x, residual, weight, out, h if residual_out is not None else None, (tokens, D), (x_t, r_t, y_t, h_t))
    a = MlaRmsNormArgs.from_buffer_copy(_NORM.pack(
        x.data_ptr(), r_ptr, weight.data_ptr(), y_ptr, scale_ptr, h_ptr, x_t, r_t, y_t, h_t, tokens, D, kind,
        _DTYPES[weight.dtype], eps, 0))
    _launch("mla_rms_norm", _lib.load().mla_rms_norm, device, ctypes.byref(a))
    if quantize:
        y = Fp8Rows(y, scale)
    return y if residual is None else (y, h)


def _norm_overlaps(x, residual, weight, out, residual_out, rows, strides) -> None:
    """Refuses outputs of the caller's own whose rows overlap each other's, or an input's without being it."""
    (tokens, D), (x_t, r_t, y_t, h_t), es = rows, strides, x.element_size()
    counts = (tokens, 1)
    for o, name, o_t in ((out, "out", y_t), (residual_out, "residual_out", h_t)):
        if o is None:
            continue
        if _rows_meet((o_t, 0), counts, D):
            raise ValueError(f"{name}'s rows overlap")
        w_ptr, o_ptr = weight.data_ptr(), o.data_ptr()
        if w_ptr < o_ptr + es * ((tokens - 1) * o_t + D) and o_ptr < w_ptr + weight.element_size() * D:
            raise ValueError(f"{name} overlaps weight")
        for t, other, t_t in ((x, "x", x_t), (residual, "residual", r_t)):
            if t is not None and not _apart_or_same(t.data_ptr(), (t_t, 0), o.data_ptr(), (o_t, 0), counts, D, es):
                raise ValueError(f"{name} overlaps {other} without being it")
    if out is not None and residual_out is not None:
        if out.data_ptr() == residual_out.data_ptr() or not _apart_or_same(
                out.data_ptr(), (y_t, 0), residual_out.data_ptr(), (h_t, 0), counts, D, es):
            raise ValueError("out and residual_out overlap")


# ---------------------------------------------------------------------------------------
# projections by 4-bit weights
# ---------------------------------------------------------------------------------------
class Fp4Weight(NamedTuple):
    """Weights ``[n, k]`` in 4 bits, as ``linear_fp4`` reads them: ``codes`` uint8 ``[ceil(n / 16), ceil(k / 128), 64, 16]``
    (OCP e2m1), ``scale`` uint8 ``[ceil(n / 16), ceil(k / 128), 64]`` (a power of two per output and 32 inputs) and ``top``
    uint8 ``[16 * ceil(n / 16)]``, each output's largest scale (255, a NaN block's, as 1).  Made by :func:`quantize_w_fp4` or :func:`pack_w_fp4`."""
    codes: torch.Tensor
    scale: torch.Tensor
    top: torch.Tensor
    n: int
    k: int


def pack_w_fp4(codes: torch.Tensor, scale: torch.Tensor) -> Fp4Weight:
    """The weights ``codes`` uint8 ``[n, k / 2]`` (OCP e2m1, two a byte, the lower input in the low half) with ``scale`` uint8
    ``[n, k / 32]`` (value ``e2m1(code) * 2**(scale - 127)``, bytes 1 .. 254, 0 taken as 1, 255 a NaN), laid out for the
    matrix unit.  Done once per weight."""
    if codes.dim() != 2 or scale.dim() != 2 or codes.dtype != torch.uint8 or scale.dtype != torch.uint8:
        raise ValueError("codes and scale must be 2-D uint8 tensors")
    n, k = codes.shape[0], 2 * codes.shape[1]
    if n < 1 or k < GROUP or k % GROUP or scale.shape != (n, k // GROUP) or scale.device != codes.device:
        raise ValueError(f"codes must be [n, k / 2] and scale [n, k / {GROUP}] on one device, k a multiple of {GROUP}")
    tiles, chunks = -(-n // 16), -(-k // 128)
    c = torch.zeros(16 * tiles, 64 * chunks, dtype=torch.uint8, device=codes.device)
    c[:n, :k // 2] = codes
    s = torch.full((16 * tiles, 4 * chunks), 127, dtype=torch.uint8, device=codes.device)
    s[:n, :k // GROUP] = scale.clamp(min=1)
    top = torch.full((16 * tiles,), 127, dtype=torch.uint8, device=codes.device)
    top[:n] = torch.where(s == 255, 1, s)[:n, :k // GROUP].amax(1)
    return Fp4Weight(c.view(tiles, 16, chunks, 4, 16).permute(0, 2, 3, 1, 4).contiguous().view(tiles, chunks, 64, 16),
                     s.view(tiles, 16, chunks, 4).permute(0, 2, 3, 1).contiguous().view(tiles, chunks, 64), top, n, k)


def quantize_w_fp4(w: torch.Tensor) -> Fp4Weight:
    """A weight matrix ``[n, k]`` (any float type, k a multiple of 32) in 4 bits: per output and 32 inputs the smallest power
    of two that brings them to 6 at most, values to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, as
    the 4-bit cache holds its latents (a block with a NaN or an infinity becomes NaN).  Done once per weight."""
    if w.dim() != 2 or not w.is_floating_point() or w.shape[0] < 1 or w.shape[1] < GROUP or w.shape[1] % GROUP:
        raise ValueError(f"w must be a float [n, k] tensor, k a multiple of {GROUP}")
    parts = [_to_fp4(p) for p in w.split(4096)]
    return pack_w_fp4(torch.cat([c for c, _ in parts]), torch.cat([s for _, s in parts]))


def _to_fp4(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes [n, k / 2], scale bytes [n, k / 32])`` of float rows."""
    b = w.float().unflatten(-1, (-1, GROUP))
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    b = torch.where(bad[..., None], 0, b.clamp(-1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127))
    m, e = torch.frexp(b.abs().amax(-1))  # amax = m * 2^e, m in [0.5, 1); 6 = 0.75 * 2^3
    k = torch.where(m == 0, torch.zeros_like(e), torch.where(m <= 0.75, e - 3, e - 2).clamp(-126, 127))
    v = torch.ldexp(b, -k[..., None])
    a = v.abs()
    n = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    n = (n | torch.signbit(v).to(torch.uint8) << 3).flatten(-2).unflatten(-1, (-1, 2))
    return n[..., 0] | n[..., 1] << 4, torch.where(bad, 255, k + 127).to(torch.uint8)


@functools.lru_cache(maxsize=4096)
def _linear_workspace(tokens: int, n: int, k: int) -> int:
    return _lib.load().mla_linear_workspace_bytes(tokens, n, k)


def linear_fp4(x: Union[torch.Tensor, Fp8Rows], w: Fp4Weight, out: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y [..., n] = x [..., k] . w^T`` for few rows: decode steps, drafted tokens.

    ``x`` in bf16 or fp16, or :class:`Fp8Rows` (from :func:`rms_norm`).  Sums are fp32, rounded once to ``dtype`` (bf16 or
    fp16; x's by default, bf16 of 8-bit rows).  8-bit rows are taken as bf16 values, exactly inside bf16's range; bf16 and
    8-bit rows take the weights exactly; with fp16 rows weights below ``2**-35`` of the largest of their output are lost.  The leading dims must be one stride apart; rows that do not
    start on 16 bytes are copied first.  ``out`` (unit stride in its rows) may not overlap ``x`` or ``w``.  Memory gives the weights
    once for up to 64 rows, so a few rows cost little more than one; it takes up to 2**20."""
    coded = isinstance(x, Fp8Rows)
    rows = x.codes if coded else x
    index = rows.get_device()
    if index < 0:
        _require(rows, "x")
    device, shape, n, k = rows.device, rows.shape, w.n, w.k
    if len(shape) < 2 or shape[-1] != k:
        raise ValueError(f"x must be [..., {k}]")
    if coded:
        if rows.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise ValueError("8-bit rows have uint8 (or float8_e4m3fn) codes")
        kind = MLA_DTYPE_BF16
        if dtype is None:
            dtype = torch.bfloat16 if out is None else out.dtype
    else:
        kind = _DTYPES.get(rows.dtype)
        if kind is None or kind == MLA_DTYPE_F32:
            raise ValueError("x must be bfloat16 or float16, or 8-bit rows")
        if dtype is None:
            dtype = rows.dtype if out is None else out.dtype
    y_kind = _DTYPES.get(dtype)
    if y_kind is None or y_kind == MLA_DTYPE_F32:
        raise ValueError("dtype must be bfloat16 or float16")
    codes, scale, top = w.codes, w.scale, w.top
    tiles, chunks = -(-n // 16), -(-k // 128)
    u8 = torch.uint8
    if not (codes.get_device() == scale.get_device() == top.get_device() == index and codes.dtype is scale.dtype is top.dtype is u8
            and codes.shape == (tiles, chunks, 64, 16) and scale.shape == (tiles, chunks, 64) and top.shape == (16 * tiles,)
            and codes.is_contiguous() and scale.is_contiguous() and top.is_contiguous()):
        for t, name, want in ((codes, "w.codes", (tiles, chunks, 64, 16)), (scale, "w.scale", (tiles, chunks, 64)), (top, "w.top", (16 * tiles,))):
            if t.get_device() != index:
                _require(t, name, device)
            if t.dtype is not u8 or t.shape != want or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 {list(want)} tensor (see pack_w_fp4)")
    if codes.data_ptr() % 16:
        raise ValueError("w.codes must be 16-byte aligned")
    at = _token_rows(rows)
    if at is None or rows.stride(-1) != 1:
        raise ValueError("x must have unit stride in its rows and token dims one stride apart")
    tokens, x_t = at
    if tokens > 2 ** 20:
        raise ValueError("x must have at most 2**20 rows")
    size = rows.element_size()
    if rows.data_ptr() % 16 or x_t * size % 16:
        rows = rows.contiguous().clone()
        x_t = k
    s_ptr, s_t = 0, 0
    if coded:
        xs = x.scale
        if xs.get_device() != index:
            _require(xs, "x.scale", device)
        s_at = _token_rows(xs)
        if xs.dtype is not torch.uint8 or xs.shape != (*shape[:-1], k // GROUP) or s_at is None or (k > GROUP and xs.stride(-1) != 1):
            raise ValueError(f"x.scale must be a uint8 [..., {k // GROUP}] tensor with unit stride in its rows")
        s_ptr, s_t = xs.data_ptr(), s_at[1]
    if out is None:
        y, y_t = new_tensor((*shape[:-1], n), dtype, device), n
    else:
        y = out
        if y.get_device() != index:
            _require(y, "out", device)
        y_at = _token_rows(y)
        if y.shape != (*shape[:-1], n) or y.dtype is not dtype or y_at is None or (n > 1 and y.stride(-1) != 1):
            raise ValueError(f"out must be a {dtype} [..., {n}] tensor with unit stride in its rows")
        y_t = y_at[1]
        if tokens and _rows_meet((y_t, 0), (tokens, 1), n):
            raise ValueError("out's rows overlap")
        y_ptr, x_ptr = y.data_ptr(), rows.data_ptr()
        y_end = y_ptr + 2 * ((tokens - 1) * y_t + n)
        if tokens and y_ptr < x_ptr + size * ((tokens - 1) * x_t + k) and x_ptr < y_end:
            raise ValueError("out overlaps x")
        if tokens and coded and y_ptr < s_ptr + (tokens - 1) * s_t + k // GROUP and s_ptr < y_end:
            raise ValueError("out overlaps x.scale")
        if tokens and any(y_ptr < t.data_ptr() + t.numel() and t.data_ptr() < y_end for t in (codes, scale, top)):
            raise ValueError("out overlaps w")
    need = _linear_workspace(tokens, n, k)
    ws_ptr = ws = 0
    if need:
        _, ws_ptr, ws = _workspace(device, _stream_ptr(device), need)
    a = MlaLinearArgs.from_buffer_copy(_LINEAR.pack(
        rows.data_ptr(), s_ptr, codes.data_ptr(), scale.data_ptr(), top.data_ptr(), y.data_ptr(), x_t, s_t, y_t,
        tokens, n, k, kind, y_kind, 0, ws_ptr, ws))
    _launch("mla_linear_fp4", _lib.load().mla_linear_fp4, device, ctypes.byref(a))
    return y
