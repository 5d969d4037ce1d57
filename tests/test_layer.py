"""Host checks of the operators around the attention, without a GPU: struct layouts and refusals."""
import ctypes
import math
import shutil

import pytest
import torch

import mlc_decode_amd as M
from mlc_decode_amd import _lib
from test_capi import _c_layout

BASE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc to lay out the header's structs")
@pytest.mark.parametrize("cls,name", [(_lib.MlaRmsNormArgs, "mla_rms_norm_args"), (_lib.MlaLinearArgs, "mla_linear_args")])
def test_struct_layouts(tmp_path, cls, name):
    fields = [f for f, _ in cls._fields_]
    c = _c_layout(tmp_path, name, fields)
    assert c[0] == ctypes.sizeof(cls) and c[1:] == [getattr(cls, f).offset for f in fields]


def test_norm_refusals(lib):
    def norm(**kw):
        a = _lib.MlaRmsNormArgs()
        a.x, a.residual, a.weight, a.out, a.residual_out = BASE, 2 * BASE, 3 * BASE, 4 * BASE, 5 * BASE
        a.x_stride = a.residual_stride = a.out_stride = a.residual_out_stride = 64
        a.tokens, a.dim, a.eps = 4, 64, 1e-6
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mla_rms_norm(ctypes.byref(a), None), lib.mla_last_error()

    for kw, code, needle in [
            (dict(dtype=3), 1, b"dtype"), (dict(weight_dtype=1), 1, b"weight_dtype"), (dict(tokens=-1), 1, b"tokens"), (dict(dim=0), 1, b"dim"),
            (dict(reserved=1), 1, b"reserved"), (dict(eps=-1.0), 1, b"eps"), (dict(eps=math.nan), 1, b"eps"), (dict(eps=math.inf), 1, b"eps"),
            (dict(scale=BASE, dim=48), 1, b"multiple of 32"), (dict(tokens=1 << 24), 4, b"2^24"), (dict(dim=(1 << 24) + 1), 4, b"2^24"),
            (dict(x=None), 1, b"NULL"), (dict(weight=None), 1, b"NULL"), (dict(out=None), 1, b"NULL"), (dict(residual=None), 1, b"residual"),
            (dict(x=BASE + 1), 1, b"aligned"), (dict(weight_dtype=2, weight=BASE + 2), 1, b"aligned"), (dict(scale=BASE, out=BASE + 4), 1, b"8-byte"),
            (dict(scale=BASE, out_stride=68), 1, b"8-byte"), (dict(out_stride=-1), 1, b"strides")]:
        rc, msg = norm(**kw)
        assert rc == code and needle in msg, (kw, rc, msg)
    assert norm(tokens=0)[0] == 0 and lib.mla_rms_norm(None, None) == 1


def test_python_refuses_cpu_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    with pytest.raises(ValueError, match="GPU"):
        M.rms_norm(x, w)


def test_linear_refusals(lib):
    def linear(**kw):
        a = _lib.MlaLinearArgs()
        a.x, a.codes, a.scale, a.top, a.y = BASE, 2 * BASE, 3 * BASE, 4 * BASE, 5 * BASE
        a.x_stride, a.y_stride, a.tokens, a.n, a.k = 256, 64, 4, 64, 256
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mla_linear_fp4(ctypes.byref(a), None), lib.mla_last_error()

    for kw, code, needle in [
            (dict(tokens=-1), 1, b"tokens"), (dict(tokens=(1 << 20) + 1), 1, b"tokens"), (dict(n=0), 1, b"n in"), (dict(n=(1 << 22) + 1), 1, b"n in"),
            (dict(k=0), 1, b"multiple of 32"), (dict(k=48), 1, b"multiple of 32"), (dict(y_dtype=2), 1, b"y_dtype"), (dict(x_dtype=2), 1, b"x_dtype"), (dict(reserved=1), 1, b"reserved"),
            (dict(x=None), 1, b"NULL"), (dict(top=None), 1, b"NULL"), (dict(y=None), 1, b"NULL"), (dict(x=BASE + 8), 1, b"16-byte"), (dict(codes=BASE + 8), 1, b"16-byte"),
            (dict(x_stride=260), 1, b"strides"), (dict(x_scale=BASE, x_stride=264), 1, b"strides"), (dict(x_scale_stride=-1), 1, b"strides"), (dict(y_stride=-2), 1, b"strides"),
            (dict(tokens=64, k=16384, n=4096), 2, b"workspace"), (dict(tokens=64, k=16384, n=4096, workspace=BASE, workspace_bytes=100, x_stride=16384), 2, b"workspace"),
            (dict(tokens=64, k=16384, n=4096, workspace=BASE + 8, workspace_bytes=1 << 40), 2, b"aligned")]:
        rc, msg = linear(**kw)
        assert rc == code and needle in msg, (kw, rc, msg)
    assert linear(tokens=0)[0] == 0 and lib.mla_linear_fp4(None, None) == 1
    assert lib.mla_linear_workspace_bytes(16, 512, 8192) == 0 and lib.mla_linear_workspace_bytes(64, 512, 48) == 0
    n = lib.mla_linear_workspace_bytes(64, 4096, 16384)
    assert n > 0 and n % (64 * 4096 * 4) == 0 and lib.mla_linear_workspace_bytes(64, 512, 2048) == 0


def test_weights_against_the_format():
    """Quantised as the 4-bit cache's oracle says, and every code and scale where the layout says."""
    import numpy as np
    from mlc_decode_amd.layer import _to_fp4
    from oracle import mla_fp4_ref as F
    g = torch.Generator().manual_seed(1)
    n, k = 37, 544
    w = torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-30, 30, (n, k), generator=g).float())
    w[3, 40], w[4, 0], w[5, :32], w[6, 32:64] = math.nan, 3e38, 0.0, 2.0 ** -140
    codes, scale = _to_fp4(w)
    b = w.double().numpy().reshape(n, k // 32, 32)
    amax = np.abs(b).max(-1)
    byte = F.scale_byte(np.where(amax > F.LARGEST, F.LARGEST, amax))
    assert (byte == scale.numpy()).all()
    bad = byte == F.NAN_BYTE
    v = np.where(bad[..., None], 0.0, np.clip(np.nan_to_num(b), -F.LARGEST, F.LARGEST) / np.exp2(np.where(bad, 127, byte) - 127.0)[..., None])
    want = F.e2m1_encode(v).reshape(n, k)
    got = np.stack([codes.numpy() & 15, codes.numpy() >> 4], -1).reshape(n, k)
    assert (want == got).all()
    p = M.quantize_w_fp4(w)
    assert p[3:] == (n, k) and p.codes.shape == (3, 5, 64, 16) and p.scale.shape == (3, 5, 64) and p.top.shape == (48,)
    for m in range(48):
        for c in range(5):
            for q in range(4):
                at = (m // 16, c, 16 * q + m % 16)
                j = 128 * c + 32 * q
                if m < n and j < k:
                    assert p.codes[at].tolist() == codes[m, j // 2:j // 2 + 16].tolist() and p.scale[at] == scale[m, j // 32]
                else:
                    assert not p.codes[at].any() and p.scale[at] == 127
    assert p.top[4] == scale[4].max() and p.top[3] == scale[3][scale[3] != 255].max()
    assert M.pack_w_fp4(torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8)).scale[0, 0, 0] == 1
    for args in [(codes.int(), scale), (codes, scale[:, :3]), (codes[:, :8], scale[:, :1]), (codes[0], scale[0])]:
        with pytest.raises(ValueError):
            M.pack_w_fp4(*args)
    for m in (torch.zeros(4, 48), torch.zeros(4), torch.zeros(4, 64, dtype=torch.int32)):
        with pytest.raises(ValueError):
            M.quantize_w_fp4(m)
    with pytest.raises(ValueError, match="GPU"):
        M.linear_fp4(torch.zeros(2, k, dtype=torch.bfloat16), p)
