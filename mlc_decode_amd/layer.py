"""Around the attention in a layer: the torch-facing entry points.

* ``rms_norm(x, weight, eps, residual)``: the residual's addition and the root-mean-square norm, to rows in x's dtype or
  to 8-bit rows with scales (``Fp8Rows``).

Calls are queued on torch's current stream of the tensors' device, synchronise nothing, and can be captured in a HIP graph.
The reference starts at rotated, projected inputs and has no counterpart of these.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import MLA_DTYPE_BF16, MLA_DTYPE_F16, MLA_DTYPE_F32, MlaRmsNormArgs
from .api import _launch
from .serving import _apart_or_same, _require, _rows_meet

_DTYPES = {torch.bfloat16: MLA_DTYPE_BF16, torch.float16: MLA_DTYPE_F16, torch.float32: MLA_DTYPE_F32}
_NORM = struct.Struct("=6Q4q4ifi")
assert _NORM.size == ctypes.sizeof(MlaRmsNormArgs)
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
    and summed in fp32; y is of h as added, and both are rounded once, to x's dtype.  With ``quantize`` y is
    :class:`Fp8Rows`, rounded from fp32 (D a multiple of 32), what ``linear_fp4`` reads.  ``out`` and ``residual_out``
    default to new tensors; each may be ``x`` or ``residual`` itself (in place), and may not overlap them otherwise, nor
    each other.  Rows may be strided (the latent part of ``kv [T, 576]`` before it is appended); the token dims of each
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
    x_t = _norm_rows(x, "x", x)
    tokens = x.numel() // D
    if weight.get_device() != index:
        _require(weight, "weight", device)
    if weight.shape != (D,) or not weight.is_contiguous() or weight.dtype not in (dtype, torch.float32):
        raise ValueError(f"weight must be a contiguous [{D}] tensor in x's dtype or float32")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be finite and at least 0")
    r_ptr, r_t, h, h_ptr, h_t = 0, 0, None, 0, 0
    if residual is not None:
        r_ptr, r_t = residual.data_ptr(), _norm_rows(residual, "residual", x)
        h = residual_out
        if h is None:
            h, h_t = torch.empty(shape, dtype=dtype, device=device), D
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
        y = torch.empty(shape, dtype=torch.uint8, device=device)
        scale = torch.empty(*shape[:-1], D // GROUP, dtype=torch.uint8, device=device)
        y_t, scale_ptr = D, scale.data_ptr()
    elif out is None:
        y, y_t = torch.empty(shape, dtype=dtype, device=device), D
    else:
        y, y_t = out, _norm_rows(out, "out", x)
    y_ptr = y.data_ptr()
    if tokens and (out is not None or residual_out is not None):
        _norm_overlaps(x, residual, out, h if residual_out is not None else None, (tokens, D), (x_t, r_t, y_t, h_t))
    a = MlaRmsNormArgs.from_buffer_copy(_NORM.pack(
        x.data_ptr(), r_ptr, weight.data_ptr(), y_ptr, scale_ptr, h_ptr, x_t, r_t, y_t, h_t, tokens, D, kind,
        _DTYPES[weight.dtype], eps, 0))
    _launch("mla_rms_norm", _lib.load().mla_rms_norm, device, ctypes.byref(a))
    if quantize:
        y = Fp8Rows(y, scale)
    return y if residual is None else (y, h)


def _norm_overlaps(x, residual, out, residual_out, rows, strides) -> None:
    """Refuses outputs of the caller's own whose rows overlap each other's, or an input's without being it."""
    (tokens, D), (x_t, r_t, y_t, h_t), es = rows, strides, x.element_size()
    counts = (tokens, 1)
    for o, name, o_t in ((out, "out", y_t), (residual_out, "residual_out", h_t)):
        if o is None:
            continue
        if _rows_meet((o_t, 0), counts, D):
            raise ValueError(f"{name}'s rows overlap")
        for t, other, t_t in ((x, "x", x_t), (residual, "residual", r_t)):
            if t is not None and not _apart_or_same(t.data_ptr(), (t_t, 0), o.data_ptr(), (o_t, 0), counts, D, es):
                raise ValueError(f"{name} overlaps {other} without being it")
    if out is not None and residual_out is not None:
        if out.data_ptr() == residual_out.data_ptr() or not _apart_or_same(
                out.data_ptr(), (y_t, 0), residual_out.data_ptr(), (h_t, 0), counts, D, es):
            raise ValueError("out and residual_out overlap")
