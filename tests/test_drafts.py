"""Host checks of the operators on drafted tokens, without a GPU: struct layout, refusals, and the oracle on small trees."""
import ctypes
import shutil

import pytest
import torch

import mlc_decode_amd as M
from mlc_decode_amd import _lib
from oracle import mla_tree_ref as T
from test_capi import _c_layout, _valid_args
from test_serving import cache_desc

BASE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc to lay out the header's structs")
def test_struct_layout(tmp_path):
    cls = _lib.MlaTreePlanArgs
    fields = [f for f, _ in cls._fields_]
    c = _c_layout(tmp_path, "mla_tree_plan_args", fields)
    assert c[0] == ctypes.sizeof(cls) and c[1:] == [getattr(cls, f).offset for f in fields]


def test_workspace(lib):
    pad = lambda x: -(-x // 256) * 256  # noqa: E731
    slots, rows = 2 * 3 + 40, 5 * 16
    assert lib.mla_tree_workspace_bytes(3, 5, 16, 40) == pad(4 * 4) + pad(slots * rows * 4) + pad(slots * rows * 16) + slots * rows * 1024
    assert lib.mla_tree_workspace_bytes(0, 5, 16, 40) == 0


def tree_args(**kw):
    a = _valid_args()
    a.s_q, a.workspace_bytes = 4, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("changes,mask,code,needle", [
    ({}, None, 1, b"mask"), ({}, BASE + 4, 1, b"mask"), (dict(s_q=65), BASE, 4, b"s_q"), (dict(batch=65536), BASE, 4, b"65535"),
    (dict(s_q=1, indices=BASE, topk=4, indices_stride=4), BASE, 4, b"paged"), (dict(block_table=None), BASE, 4, b"paged"),
    (dict(workspace_bytes=0), BASE, 2, b"mla_tree_workspace_bytes"), (dict(sm_scale=-1.0), BASE, 1, b"sm_scale"), (dict(kv_format=4, dtype=1), BASE, 4, b"bf16")])
def test_decode_refusals(lib, changes, mask, code, needle):
    assert lib.mla_tree_decode_fwd(tree_args(**changes), mask, None) == code
    assert needle in lib.mla_last_error()
    assert lib.mla_tree_absorb_fwd(tree_args(**changes), mask, BASE, BASE, None) == code


def test_absorb_refusals(lib):
    assert lib.mla_tree_absorb_fwd(tree_args(), BASE, None, BASE, None) == 1 and b"w_uv_blk" in lib.mla_last_error()
    assert lib.mla_tree_decode_fwd(None, BASE, None) == 1 and b"NULL" in lib.mla_last_error()


def test_takes_pages(lib):
    """Few pages and rows, room in the workspace; nothing of a call that the decode would refuse."""
    f = lib.mla_tree_takes_pages
    for fmt in (0, 1, 4):
        assert f(1, 8, 16, 256, fmt, 33) == 1 and f(1, 1, 1, 256, fmt, 1) == 1
        assert f(1, 8, 16, 256, fmt, 258) == 0 and f(64, 8, 128, 256, fmt, 2) == 0  # slots; tiles
        assert f(1, 8, 16, 256, fmt, 2 ** 24) == 0 and f(65535, 64, 1024, 256, fmt, 2 ** 24) == 0
    assert f(1, 1, 1, 256, 2, 1) == 0 and f(0, 1, 1, 256, 0, 1) == 0 and f(1, 1, 1, 256, 0, 0) == 0 and f(1, 1, 1, 0, 0, 1) == 0


def test_plan_accept_keep_refusals(lib):
    def plan(**kw):
        a = _lib.MlaTreePlanArgs()
        for f in ("parents", "cache_seqlens", "block_table", "mask", "positions", "slots", "prefix_lens"):
            setattr(a, f, BASE)
        a.block_table_stride, a.block_table_width, a.batch, a.s_q = 4, 4, 2, 8
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mla_tree_plan(ctypes.byref(a), None), lib.mla_last_error()

    for kw, needle in [(dict(s_q=0), b"s_q"), (dict(s_q=65), b"s_q"), (dict(batch=-1), b"batch"), (dict(batch=(1 << 20) + 1), b"batch"), (dict(parents=None), b"NULL"),
                       (dict(slots=None), b"NULL"), (dict(mask=BASE + 4), b"8-byte"), (dict(block_table_width=5), b"width"), (dict(block_table_width=0), b"width")]:
        rc, msg = plan(**kw)
        assert rc == 1 and needle in msg, (kw, msg)
    assert plan(batch=0)[0] == 0 and lib.mla_tree_plan(None, None) == 1

    def accept(mask=BASE, tokens=BASE, wide=0, batch=2, s_q=8, nxt=BASE):
        return lib.mla_tree_accept(mask, BASE, tokens, BASE, wide, batch, s_q, BASE, BASE, nxt, BASE, None), lib.mla_last_error()

    for kw, needle in [(dict(mask=None), b"NULL"), (dict(mask=BASE + 4), b"aligned"), (dict(tokens=BASE + 4, wide=1), b"aligned"), (dict(nxt=BASE + 2), b"aligned"),
                       (dict(wide=2), b"wide"), (dict(s_q=65), b"s_q"), (dict(batch=-1), b"batch")]:
        rc, msg = accept(**kw)
        assert rc == 1 and needle in msg, (kw, msg)
    assert accept(batch=0)[0] == 0

    c = cache_desc()
    assert lib.mla_kv_keep_path(ctypes.byref(c), BASE, BASE, 0, 8, None) == 0
    assert lib.mla_kv_keep_path(None, BASE, BASE, 2, 8, None) == 1
    for args, needle in [((None, BASE, 2, 8), b"NULL"), ((BASE, None, 2, 8), b"NULL"), ((BASE, BASE, 2, 65), b"s_q"), ((BASE, BASE, -1, 8), b"batch")]:
        assert lib.mla_kv_keep_path(ctypes.byref(c), *args, None) == 1 and needle in lib.mla_last_error()
    bad = cache_desc(num_blocks=0)
    assert lib.mla_kv_keep_path(ctypes.byref(bad), BASE, BASE, 2, 8, None) == 1 and b"num_blocks" in lib.mla_last_error()


def test_python_refusals():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    p = M.TreePlan(torch.zeros(2, 4, dtype=torch.int64), i32(2, 4), i32(2, 4), i32(2))
    q, kv = torch.zeros(2, 4, 8, 576, dtype=torch.bfloat16), torch.zeros(2, 64, 1, 576, dtype=torch.bfloat16)
    for call in (lambda: M.tree_plan(i32(2, 4), i32(2), i32(2, 4)), lambda: M.tree_accept(p, i32(2, 4), i32(2, 4)),
                 lambda: M.kv_keep_path(kv, i32(2, 4), i32(2, 4)), lambda: M.flash_mla_with_kvcache(q, kv, i32(2, 4), None, 512, i32(4, 8), i32(3), tree=p)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_oracle_on_a_small_tree():
    #      0
    #     1  2        5 has a dropped parent, 6 hangs below it
    #    3    4
    parents = [-1, 0, 0, 1, 2, -2, 5, 9]
    mask, pos, slots, prefix = T.plan([parents], [70], [[3, 1]])
    assert prefix == [62] and mask[0] == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 2, 4}, set(), set(), set()]
    assert pos[0] == [62, 63, 63, 64, 64, -1, -1, -1] and slots[0] == [254, 255, 64, 65, 66, 67, 68, 69]
    tok, tgt = [7, 5, 6, 1, 2, 0, 0, 0], [6, 1, 2, 0, 9, 0, 0, 0]
    assert T.accept(mask, prefix, [tok], [tgt]) == ([[0, 2, 4, -1, -1, -1, -1, -1]], [3], [9], [65])
    assert T.plan([parents], [7], [[3, 1]])[0][0] == [set()] * 8  # shorter than its tree
    assert T.bits({63}) == -(1 << 63) and T.bits({0, 2}) == 5
