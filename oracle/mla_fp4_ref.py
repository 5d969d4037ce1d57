"""CPU restatement of the 4-bit latent-cache format -- test infrastructure only.

The reference has no such cache.  This file defines the format the 4-bit append and decode implement:

  * ``e2m1_decode`` / ``e2m1_encode`` -- the 4-bit element of the OCP Microscaling Formats Specification
    v1.0 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), rounded to nearest, ties
    to the even code, saturating at 6;
  * ``scale_byte`` -- the scale of 32 dims: 2^k as the byte k + 127, k the smallest with amax <= 6 * 2^k
    (-126 at least; 0 for zeros), byte 255 where the block holds a NaN or an infinity;
  * ``LARGEST`` -- 1.5 * 2^127, the largest value that e2m1 codes and bf16 both hold: larger ones are stored as it
    (the next code, 4 * 2^126 = 2^128, is no bf16 or fp32 number);
  * ``quantize_latent`` / ``dequantize_latent`` / ``dequantize_pages`` / ``append_paged_fp4`` as in
    ``mla_fp8_ref``: dim 2i of a token is the low half of byte i.

Pinning (tests/test_oracle_fp4.py): decode against the fields' definition, encode against a nearest-value
search in rationals, the scale rule against a brute force over all exponents.
"""
from __future__ import annotations

import numpy as np
import torch

LATENT, ROPE, BLOCK, PAGE = 512, 64, 32, 64
NBLK = LATENT // BLOCK
E2M1_MAX = 6.0
LARGEST = 1.5 * 2.0 ** 127
NAN_BYTE = 255


def e2m1_decode(codes: np.ndarray) -> np.ndarray:
    """4-bit codes -> values: exponent field 0 is m / 2, else (1 + m / 2) * 2^(e - 1)."""
    c = np.asarray(codes).astype(np.int64)
    e, m = (c >> 1) & 3, c & 1
    v = np.where(e == 0, m / 2.0, (1.0 + m / 2.0) * np.exp2(e - 1.0))
    return np.where(c & 8, -v, v)


def e2m1_encode(x: np.ndarray) -> np.ndarray:
    """Finite values -> 4-bit codes; the sign of a value that rounds to zero is kept."""
    a = np.abs(np.asarray(x, dtype=np.float64))
    step = np.where(a < 2.0, 0.5, np.where(a < 4.0, 1.0, 2.0))
    r = np.minimum(np.rint(a / step) * step, E2M1_MAX)  # a binade's last tie goes up to a power of two: even
    e = np.where(r < 1.0, 0, np.floor(np.log2(np.maximum(r, 1.0))).astype(np.int64) + 1)
    m = np.where(r < 1.0, r * 2, (r / np.exp2(e - 1.0) - 1.0) * 2).astype(np.int64)
    return ((np.signbit(x).astype(np.int64) << 3) | (e << 1) | m).astype(np.uint8)


def scale_byte(amax: np.ndarray) -> np.ndarray:
    """amax of each block (fp32 holding a bf16 value; NaN and infinity allowed) -> byte."""
    a = np.asarray(amax, dtype=np.float64)
    bad = ~np.isfinite(a)
    m, e = np.frexp(np.where(bad, 0.0, a))     # a = m * 2^e, m in [0.5, 1); 6 = 0.75 * 2^3
    k = np.where(m <= 0.75, e - 3, e - 2)
    k = np.where((a == 0) | bad, 0, np.maximum(k, -126))
    return np.where(bad, NAN_BYTE, k + 127).astype(np.uint8)


def quantize_latent(latent: torch.Tensor):
    """latent [n, 512] (bf16) -> (codes uint8 [n, 256], scale bytes uint8 [n, 16])."""
    x = latent.to(torch.bfloat16).float().numpy().astype(np.float64).reshape(-1, NBLK, BLOCK)
    amax = np.where(np.isfinite(x).all(-1), np.abs(x).max(-1), np.inf)
    byte = scale_byte(amax)
    bad = byte == NAN_BYTE
    v = np.clip(np.where(bad[..., None], 0.0, x), -LARGEST, LARGEST) / np.exp2(np.where(bad, 0, byte.astype(np.int64) - 127))[..., None]
    c = np.where(bad[..., None], 0, e2m1_encode(v)).astype(np.uint8).reshape(-1, LATENT // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), byte


def dequantize_latent(codes: np.ndarray, byte: np.ndarray) -> np.ndarray:
    """codes [n, 256], bytes [n, 16] -> float64 [n, 512] (NaN blocks as NaN)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(-1, NBLK, BLOCK)
    s = np.where(byte == NAN_BYTE, np.nan, np.exp2(byte.astype(np.float64) - 127))
    with np.errstate(invalid="ignore"):
        return (e2m1_decode(c) * s.reshape(-1, NBLK, 1)).reshape(-1, LATENT)


def quantize_pages(kv_cache: torch.Tensor):
    """bf16 cache [nb, 64, 1, 576] -> (codes [nb, 64, 256], bytes [nb, 64, 16], rope [nb, 64, 64])."""
    nb = kv_cache.shape[0]
    flat = kv_cache.reshape(nb * PAGE, LATENT + ROPE)
    codes, byte = quantize_latent(flat[:, :LATENT])
    return (codes.reshape(nb, PAGE, LATENT // 2), byte.reshape(nb, PAGE, NBLK),
            flat[:, LATENT:].to(torch.bfloat16).reshape(nb, PAGE, ROPE).contiguous())


def dequantize_pages(codes: np.ndarray, byte: np.ndarray, rope: torch.Tensor) -> torch.Tensor:
    """-> float64 [nb, 64, 1, 576]: the cache the 4-bit decode must agree with."""
    nb = codes.shape[0]
    lat = dequantize_latent(codes.reshape(nb * PAGE, -1), byte.reshape(nb * PAGE, -1))
    return torch.cat([torch.from_numpy(lat).reshape(nb, PAGE, LATENT), rope.double()], -1).reshape(nb, PAGE, 1, -1)


def append_paged_fp4(codes, byte, rope, block_table, cache_seqlens, kv_new):
    """As mla_fp8_ref.append_paged_fp8, in the 4-bit format; a sequence whose pages do not hold its new
    tokens is left as it was.  Returns (codes, bytes, rope, lengths, skipped)."""
    codes, byte, rope, lens, skipped = codes.copy(), byte.copy(), rope.clone(), cache_seqlens.clone(), []
    B, n, _ = kv_new.shape
    c, s = quantize_latent(kv_new[..., :LATENT].reshape(B * n, LATENT))
    for b in range(B):
        L = int(cache_seqlens[b])
        cols = [(L + t) // PAGE for t in range(n)]
        if L < 0 or any(i >= block_table.shape[1] or not 0 <= int(block_table[b, i]) < codes.shape[0] for i in cols):
            skipped.append(b)
            continue
        for t, i in enumerate(cols):
            pg, row = int(block_table[b, i]), (L + t) % PAGE
            codes[pg, row], byte[pg, row], rope[pg, row] = c[b * n + t], s[b * n + t], kv_new[b, t, LATENT:]
        lens[b] = L + n
    return codes, byte, rope, lens, skipped
