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
@pytest.mark.parametrize("cls,name", [(_lib.MlaRmsNormArgs, "mla_rms_norm_args")])
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
