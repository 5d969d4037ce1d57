"""Host checks of the serving step's entry points, without a GPU: struct layouts, refusals of the C ABI (before any HIP
call) and of the Python layer, the rotation plan's frequencies."""
import ctypes
import math
import shutil

import pytest
import torch

import mlc_decode_amd as M
from mlc_decode_amd import _lib
from mlc_decode_amd.serving import _apart_or_same, rope_frequencies
from test_capi import _c_layout, _valid_args

BASE = 1 << 20  # fake, aligned device addresses: validation fails before any use


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc to lay out the header's structs")
@pytest.mark.parametrize("cls,name", [(_lib.MlaKvCache, "mla_kv_cache"), (_lib.MlaRope, "mla_rope"), (_lib.MlaRopeArgs, "mla_rope_args"),
                                      (_lib.MlaAppendSlotsArgs, "mla_append_slots_args"), (_lib.MlaPagePool, "mla_page_pool")])
def test_struct_layouts(tmp_path, cls, name):
    fields = [f for f, _ in cls._fields_]
    c = _c_layout(tmp_path, name, fields)
    assert c[0] == ctypes.sizeof(cls) and c[1:] == [getattr(cls, f).offset for f in fields]


def cache_desc(fmt=0, **kw):
    c = _lib.MlaKvCache()
    c.format, c.dtype, c.num_blocks = fmt, 0, 8
    c.nope, c.rope, c.scale = BASE, BASE, BASE
    c.stride_page, c.stride_tok, c.rope_stride_page, c.rope_stride_tok = 64 * 576, 576, 64 * 576, 576
    c.scale_stride_page, c.scale_stride_blk = 1024, 16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rope_desc(**kw):
    r = _lib.MlaRope()
    r.freqs, r.dim, r.layout, r.amp = BASE, 64, 0, 1.0
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("changes,code,needle", [
    (dict(dtype=1), 4, b"bf16"),
    (dict(block_table=None), 4, b"paged"),
    (dict(kv_scale=None), 1, b"kv_scale"),
    (dict(kv_scale=BASE + 8), 1, b"kv_scale"),
    (dict(kv_scale_stride_blk=20), 1, b"kv_scale"),
    (dict(kv_scale_stride_page=-16), 1, b"kv_scale"),
    (dict(kv_scale_stride_blk=1 << 24), 4, b"2^24"),
    (dict(kv_stride_tok=264), 1, b"16 bytes"),
    (dict(kv_stride_page=64 * 256 + 8), 1, b"16 bytes"),
    (dict(), 2, b"workspace"),  # valid up to the workspace
])
def test_decode_refuses_bad_fp4_args(lib, changes, code, needle):
    a = _valid_args()
    a.kv_format, a.kv_scale, a.kv_scale_stride_page, a.kv_scale_stride_blk = 4, BASE, 1024, 16
    a.kv_stride_tok, a.kv_stride_page = 256, 64 * 256
    for k, v in changes.items():
        setattr(a, k, v)
    assert lib.mla_decode_fwd(ctypes.byref(a), None) == code
    assert needle in lib.mla_last_error()


@pytest.mark.parametrize("changes,code,needle", [
    (dict(dtype=1), 4, b"bf16"), (dict(kv_scale=None), 1, b"kv_scale"), (dict(kv_stride_tok=264), 1, b"16 bytes"), (dict(kv_format=3), 1, b"kv_format")])
def test_append_refuses_bad_fp4_args(lib, changes, code, needle):
    a = _lib.MlaKvAppendArgs()
    a.batch, a.n_new, a.num_blocks, a.kv_new, a.new_stride_b, a.new_stride_t = 1, 1, 4, BASE, 576, 576
    a.kv_nope = a.kv_rope = a.kv_scale = a.block_table = a.cache_seqlens = BASE
    a.kv_stride_page, a.kv_stride_tok, a.kv_rope_stride_page, a.kv_rope_stride_tok = 64 * 256, 256, 64 * 64, 64
    a.kv_format, a.kv_scale_stride_page, a.kv_scale_stride_blk, a.block_table_stride, a.max_pages = 4, 1024, 16, 4, 4
    for k, v in changes.items():
        setattr(a, k, v)
    assert lib.mla_kv_append(ctypes.byref(a), None) == code
    assert needle in lib.mla_last_error()


def test_num_parts_by_format(lib):
    for rows, want in ((16, 512), (17, 256), (32, 256), (33, 512), (64, 512), (65, 256), (128, 256), (129, 128), (65536, 1)):
        for pages in (0, 65536, 2 ** 40):
            assert lib.mla_num_parts_for(4, 1, rows, 1, 256, 4, pages) == want
            assert lib.mla_num_parts_for(4, 1, rows, 1, 256, 0, pages) == lib.mla_num_parts(4, 1, rows, 1, 256)
    for rows, pages, want in ((64, 1536, 128), (64, 1537, 512), (128, 768, 64), (128, 769, 256), (8192, 8, 1), (1, 6144, 512)):
        assert lib.mla_num_parts_for(4, 1, rows, 1, 256, 4, pages) == want  # few pages: 512 workgroups of 16 rows
    assert lib.mla_num_parts_for(4, 1, 16, 1, 256, 2, 0) == -1 and b"kv_format" in lib.mla_last_error()
    assert lib.mla_num_parts_for(4, 1, 16, 1, 256, 4, -1) == -1 and b"max_pages" in lib.mla_last_error()
    assert lib.mla_num_parts_for(0, 1, 16, 1, 256, 4, 0) == -1


@pytest.mark.parametrize("fmt,changes,code,needle", [
    (2, {}, 1, b"kv_format"),
    (0, dict(dtype=2), 1, b"dtype"),
    (1, dict(dtype=1), 4, b"bf16"),
    (0, dict(reserved=1), 1, b"reserved"),
    (0, dict(num_blocks=0), 1, b"num_blocks"),
    (0, dict(num_blocks=1 << 26), 1, b"num_blocks"),
    (0, dict(nope=BASE + 8), 1, b"16-byte"),
    (0, dict(rope=None), 1, b"16-byte"),
    (0, dict(stride_tok=580), 1, b"strides"),
    (0, dict(rope_stride_page=-8), 1, b"strides"),
    (4, dict(stride_tok=264), 1, b"16 bytes"),
    (4, dict(scale=None), 1, b"kv_scale"),
    (4, dict(scale_stride_blk=24), 1, b"kv_scale"),
    (1, dict(scale=BASE + 4), 1, b"kv_scale"),
    (1, dict(scale_stride_blk=65), 1, b"kv_scale"),
])
def test_cache_descriptor_refusals(lib, fmt, changes, code, needle):
    c = cache_desc(fmt, **changes)
    assert lib.mla_kv_gather(ctypes.byref(c), BASE, 4, BASE, 576, None) == code
    assert needle in lib.mla_last_error()


def test_gather_and_append_refusals(lib):
    c, r = cache_desc(), rope_desc()
    assert lib.mla_kv_gather(None, BASE, 4, BASE, 576, None) == 1
    for args, needle in [((BASE, -1, BASE, 576), b"tokens"), ((None, 4, BASE, 576), b"NULL"), ((BASE, 4, BASE + 8, 576), b"16-byte"),
                         ((BASE, 4, BASE, 568), b"576"), ((BASE, 4, BASE, 580), b"576")]:
        assert lib.mla_kv_gather(ctypes.byref(c), *args, None) == 1 and needle in lib.mla_last_error()
    assert lib.mla_kv_gather(ctypes.byref(c), None, 0, None, 0, None) == 0  # nothing to do

    def append(rope=r, **kw):
        a = _lib.MlaAppendSlotsArgs()
        a.kv_new, a.new_stride, a.slots, a.positions, a.tokens = BASE, 576, BASE, BASE, 4
        a.q_pe, a.q_rope, a.heads = BASE, BASE, 2
        a.pe_stride_t, a.pe_stride_h, a.q_stride_t, a.q_stride_h = 128, 64, 1152, 576
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mla_kv_append_slots(ctypes.byref(c), ctypes.byref(rope) if rope else None, ctypes.byref(a), None), lib.mla_last_error()

    for kw, needle in [(dict(tokens=-1), b"tokens"), (dict(slots=None), b"NULL"), (dict(positions=None), b"NULL"), (dict(kv_new=BASE + 2), b"16-byte"),
                       (dict(new_stride=577), b"multiple of 8"), (dict(q_rope=None), b"16-byte"), (dict(q_stride_h=580), b"multiples of 8"),
                       (dict(rope=None), b"rope"), (dict(rope=rope_desc(dim=32)), b"64"), (dict(rope=rope_desc(layout=2)), b"layout"),
                       (dict(rope=rope_desc(freqs=None)), b"freqs"), (dict(rope=rope_desc(amp=math.inf)), b"amp")]:
        rc, msg = append(**kw)
        assert rc == 1 and needle in msg, (kw, msg)
    assert append(tokens=0)[0] == 0


def test_rope_refusals(lib):
    def rope(r=None, **kw):
        a = _lib.MlaRopeArgs()
        a.x, a.out, a.positions, a.tokens, a.heads, a.dim, a.first = BASE, 2 * BASE, BASE, 4, 2, 64, 0
        a.x_stride_t, a.x_stride_h, a.o_stride_t, a.o_stride_h = 128, 64, 128, 64
        for k, v in kw.items():
            setattr(a, k, v)
        r = r or rope_desc()
        return lib.mla_apply_rope(ctypes.byref(r), ctypes.byref(a), None), lib.mla_last_error()

    for kw, code, needle in [(dict(dtype=3), 1, b"dtype"), (dict(tokens=-1), 1, b"tokens"), (dict(dim=0), 1, b"dim"), (dict(first=1), 1, b"first"),
                             (dict(first=-1), 1, b"first"), (dict(x=None), 1, b"NULL"), (dict(x=BASE + 1), 1, b"aligned"), (dict(x_stride_h=-1), 1, b"strides"),
                             (dict(out=BASE, o_stride_t=256), 1, b"in place"), (dict(heads=1 << 20), 4, b"2^22"), (dict(reserved=1), 1, b"reserved"),
                             (dict(r=rope_desc(dim=63)), 1, b"even"), (dict(r=rope_desc(dim=1026), dim=2000), 1, b"1024")]:
        rc, msg = rope(**kw)
        assert rc == code and needle in msg, (kw, rc, msg)
    assert rope(tokens=0)[0] == 0 and rope(heads=0)[0] == 0


def test_pool_refusals(lib):
    def pool(**kw):
        p = _lib.MlaPagePool()
        p.free_pages = p.count = p.block_table = p.cache_seqlens = BASE
        p.num_blocks, p.batch, p.block_table_stride, p.block_table_width = 8, 2, 4, 4
        for k, v in kw.items():
            setattr(p, k, v)
        return ctypes.byref(p)

    for kw, needle in [(dict(free_pages=None), b"free_pages"), (dict(num_blocks=0), b"num_blocks"), (dict(num_blocks=1 << 26), b"num_blocks"),
                       (dict(block_table_width=5), b"width"), (dict(block_table_width=0), b"width"), (dict(cache_seqlens=None), b"cache_seqlens"),
                       (dict(batch=0), b"batch"), (dict(batch=16385), b"batch")]:
        assert lib.mla_reserve_pages(pool(**kw), BASE, 4, BASE, BASE, BASE, BASE, BASE, None) == 1 and needle in lib.mla_last_error()
        assert lib.mla_release_pages(pool(**kw), BASE, None) == 1 and needle in lib.mla_last_error()
    assert lib.mla_reserve_pages(pool(), BASE, -1, BASE, BASE, BASE, BASE, BASE, None) == 1
    assert lib.mla_reserve_pages(pool(), None, 4, BASE, BASE, BASE, BASE, BASE, None) == 1
    assert lib.mla_reserve_pages(pool(), BASE, 4, None, BASE, BASE, BASE, BASE, None) == 1
    assert lib.mla_release_pages(pool(), None, None) == 1


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pos = torch.zeros(4, dtype=torch.int32)
    rope = M.Rope(torch.zeros(32, dtype=torch.float64))
    kv = torch.zeros(2, 64, 1, 576, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pool = M.page_pool(4, device="cpu")
    assert pool.free_pages.tolist() == [3, 2, 1, 0] and pool.count.tolist() == [4]
    for call in (lambda: M.apply_rope(x, pos, rope), lambda: M.kv_append_slots(torch.zeros(4, 576, dtype=torch.bfloat16), kv, pos),
                 lambda: M.kv_gather(kv, pos), lambda: M.reserve_pages(pool, table, lens, lens, 4), lambda: M.release_pages(pool, table, lens, lens),
                 lambda: M.quantize_kv_cache(kv, bits=4), lambda: M.kv_gather(M.fp4_kv_cache(2, device="cpu"), pos)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: M.quantize_kv_cache(kv, bits=3), lambda: M.page_pool(0, device="cpu")):
        with pytest.raises(ValueError):
            call()


def test_fp4_cache_factory():
    c = M.fp4_kv_cache(3, device="cpu")
    assert c.latent.shape == (3, 64, 256) and c.scale.shape == (3, 64, 16) and c.rope.shape == (3, 64, 64)
    assert (c.scale == 127).all() and not c.latent.any()


def test_rope_frequencies():
    f, amp = rope_frequencies(64, 10000.0)
    assert amp == 1.0 and [abs(v * 2 * math.pi - 10000.0 ** (-2 * i / 64)) < 1e-15 for i, v in enumerate(f)] == [True] * 32
    g, _ = rope_frequencies(64, 10000.0, "linear", factor=4.0)
    assert g == [v / 4 for v in f]
    n, _ = rope_frequencies(64, 10000.0, "ntk", factor=8.0)
    assert n[0] == f[0] and abs(n[-1] * 8 / f[-1] - 1) < 1e-12  # the slowest pair slows by the factor
    y, amp = rope_frequencies(64, 10000.0, "yarn", factor=40.0, original_max=4096, mscale=1.0, mscale_all_dim=0.0)
    assert abs(amp - (0.1 * math.log(40.0) + 1)) < 1e-15
    turns = [v * 4096 for v in f]  # over the original context
    for v, w, t in zip(y, f, turns):
        if t > 40:
            assert v == w
        if t < 0.7:
            assert abs(v - w / 40) < 1e-18
        assert w / 40 * (1 - 1e-12) <= v <= w
    assert rope_frequencies(64, 10000.0, "yarn", factor=40.0, mscale=1.0, mscale_all_dim=1.0)[1] == 1.0


@pytest.mark.parametrize("kw", [dict(dim=63), dict(dim=0), dict(base=1.0), dict(base=math.inf), dict(scaling="other"), dict(scaling="linear", factor=0.5),
                                dict(scaling="ntk", factor=2.0, dim=2), dict(scaling="yarn", factor=2.0, original_max=0)])
def test_rope_plan_refusals(kw):
    with pytest.raises(ValueError):
        rope_frequencies(**kw)
    with pytest.raises(ValueError):
        M.rope_plan(layout="sideways", device="cpu")


def test_overlap_rule():
    same = dict(counts=(4, 2), width=64, es=2)
    assert _apart_or_same(0, (128, 64), 0, (128, 64), **same)            # in place
    assert not _apart_or_same(0, (128, 64), 0, (256, 64), **same)        # in place, other strides
    assert _apart_or_same(0, (128, 64), 1024, (128, 64), **same)         # one after the other
    assert not _apart_or_same(0, (128, 64), 1022, (128, 64), **same)     # by one element
    assert _apart_or_same(0, (1152, 576), 1024, (1152, 576), **same)     # parts of one row
    assert not _apart_or_same(0, (1152, 576), 1152 - 64, (1152, 576), **same)  # into the next head
    assert not _apart_or_same(0, (128, 64), 64, (128, 64), **same)
