"""GPU tests of the 4-bit cache where its decode's three forms (16, 64 and 128 rows a workgroup) could part: references that
move, NaN blocks that some rows do not see, page ids that name no page, segments of many pages, queries with
outliers, the largest latents, and the projections on top of it."""
import math

import pytest
import torch

from mlc_decode_amd import (flash_mla_with_kvcache, get_mla_metadata, kv_gather, mla_decode_absorbed, mla_decode_with_kvcache,
                            prepare_w_uv, quantize_kv_cache)
from oracle import mla_fp4_ref as F4
from oracle import mla_ref as R
from test_gpu_fp4 import SCALE, assert_cache, assert_decode, exact, problem, say, table_for, to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("splits", [1, 2])
def test_rising_and_falling_scores(gpu, H, splits):
    """Each page's scores pass the last one's by far, so that the running reference moves with nearly every stage, for
    every row tile; and the other way round, where it never moves again.  Rows of one tile move apart: odd
    heads rise where even ones fall."""
    q, cache, table, lens, _ = problem(3, [1500, 1500, 1500], H, 1)
    codes, byte, rope = cache.latent.cpu().numpy(), cache.scale.cpu().numpy(), cache.rope.cpu()
    q[..., 512:] = q[..., 512:].abs() + 0.5
    q[2, :, 1::2, 512:] *= -1
    for b in range(3):
        for i in range(24):
            rope[int(table[b, i])] = 0.5 * (23 - i if b == 1 else i)
    cache = cache._replace(rope=rope.cuda())
    table = table_for(table, H, False)
    say(f"rising H={H} splits={splits}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), num_splits=splits)
    torch.cuda.synchronize()
    assert_decode(out, lse, q, F4.dequantize_pages(codes, byte, rope), table, lens, True, f"rising H={H} splits={splits}")


@pytest.mark.parametrize("H", [16, 20, 64, 128])
@pytest.mark.parametrize("splits", [1, 2])
def test_nan_block_in_each_form(gpu, H, splits):
    q, cache, table, lens, kv = problem(44, [100, 100, 700], H, 1)
    cache.scale[int(table[0, 0]), 7, 3] = 255
    cache.scale[int(table[2, 9]), 63, 15] = 255
    table = table_for(table, H, False)
    say(f"NaN block H={H} splits={splits}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), num_splits=splits)
    torch.cuda.synchronize()
    assert torch.isnan(out[::2]).all() and (lse[::2] == -math.inf).all()
    assert_decode(out[1:2], lse[1:2], q[1:2], kv, table[1:2], lens[1:2], True, f"beside NaNs H={H}")


@pytest.mark.parametrize("H,s_q", [(8, 2), (1, 3), (16, 2), (16, 4), (64, 2), (33, 4), (128, 2)])
@pytest.mark.parametrize("splits", [None, 1, 2])
def test_nan_block_of_a_hidden_token(gpu, H, s_q, splits):
    """A NaN block in each sequence's last token: the last query's rows are NaN, every other row, and a row that sees no
    token, is as without it."""
    q, cache, table, lens, kv = problem(H + s_q, [1, 2, 64, 65, 96, 130, 800], H, s_q)
    for b, n in enumerate(lens.tolist()):
        cache.scale[int(table[b, (n - 1) // 64]), (n - 1) % 64, b] = 255
    table = table_for(table, H * s_q, False)
    say(f"hidden NaN H={H} s_q={s_q} splits={splits}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), num_splits=splits, causal=True)
    torch.cuda.synchronize()
    assert torch.isnan(out[:, -1]).all() and (lse[..., -1] == -math.inf).all()
    # without the last query the last token is seen by nobody: L - 1 tokens, s_q - 1 queries
    assert_decode(out[:, :-1], lse[..., :-1], q[:, :-1], kv, table, lens - 1, True, f"hidden NaN H={H} s_q={s_q}")


@pytest.mark.parametrize("H", [16, 64, 128])
def test_cut_at_the_table_and_foreign_pages(gpu, H):
    """Page ids that name no page are clamped into the pool, in the first, a middle and the last page that is read."""
    q, cache, table, lens, kv = problem(12, [640, 300, 64 * 90], H, 1, poison=False)
    table = table_for(table, H, False).clone()
    table[0, 0], table[0, 5], table[1, 4] = -3, 10 ** 6, 2 ** 31 - 1
    table[2, 0], table[2, 70], table[2, 89] = 2 ** 31 - 1, -2 ** 31, kv.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    say(f"foreign pages H={H}")
    for parts in (None, 1):
        sched, splits = get_mla_metadata(lens.cuda(), H, 1, parts)
        out, lse = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), 512, sched, splits, status=status)
        torch.cuda.synchronize()
        assert status.item() == 0
        assert_decode(out, lse, q, kv, table, lens, False, f"foreign H={H} parts={parts}")
    long = lens + 64 * table.shape[1]  # every sequence is cut
    sched, splits = get_mla_metadata(long.cuda(), H, 1)
    flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), long.cuda(), 512, sched, splits, status=status)
    torch.cuda.synchronize()
    assert status.item() == 1


@pytest.mark.parametrize("H", [16, 64, 128])
def test_many_pages_in_one_segment(gpu, H):
    """More than two wavefronts' worth of pages in one part, a ragged last one, and ids that name no page."""
    q, cache, table, lens, kv = problem(77, [64 * 150 + 7, 64 * 129], H, 1, poison=False)
    table = table_for(table, H, False)
    table[0, 63], table[0, 64], table[0, 127], table[0, 128], table[1, 64] = -1, 10 ** 9, 10 ** 6, -2 ** 31, 2 ** 31 - 1
    say(f"many pages H={H}")
    for parts in (1, 2):
        sched, splits = get_mla_metadata(lens.cuda(), H, 1, parts)
        out, lse = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), 512, sched, splits)
        torch.cuda.synchronize()
        assert_decode(out, lse, q, kv, table, lens, False, f"many pages H={H} parts={parts}")


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("kind", ["blocks", "outliers", "tiny", "huge"])
def test_queries_of_unequal_size(gpu, H, kind):
    """Blocks of 32 dims that differ by up to 2^12, one dim of each block 1024 times its neighbours, queries at both ends of
    bf16 (scores of huge ones are kept finite by a zero query elsewhere and a tiny scale)."""
    q, cache, table, lens, kv = problem(H, [700, 64, 1], H, 1)
    g = torch.Generator().manual_seed(5)
    x = q.float()
    scale = SCALE
    if kind == "blocks":
        x[..., :512] *= torch.exp2(-torch.randint(0, 13, x.shape[:3] + (16,), generator=g).float()).repeat_interleave(32, -1)
    elif kind == "outliers":
        x[..., 7:512:32] *= 1024.0
        x /= 64.0
    elif kind == "tiny":
        x *= 2.0 ** -60
    else:
        x *= 2.0 ** 100
        scale = SCALE * 2.0 ** -100
    q = x.to(torch.bfloat16)
    table = table_for(table, H, False)
    say(f"unequal queries H={H} {kind}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), sm_scale=scale)
    torch.cuda.synchronize()
    if kind == "huge":
        q = (q.double() * 2.0 ** -100)  # the same scores
    assert_decode(out, lse, q, kv, table, lens, True, f"unequal H={H} {kind}")


@pytest.mark.parametrize("H", [16, 64, 128])
def test_outlier_queries_within_the_decodes_bar(gpu, H):
    """One query dim of every 32 a thousand times its neighbours: the decode's own bar (outputs 1e-2, lse
    1e-3), against the exact attention of the same inputs.  Above 32 rows the query is two e4m3 parts, which drop at
    most 2^-15 of a block's largest value a: a logit is off by at most 2^-15 sum_d a_d |k_d| / 24, and by the root of
    that sum of squares over sqrt(3) where the dropped bits are even.  Here a = 16, |k_d| about 1: 2^-15 * 16 * sqrt(512) /
    (24 sqrt(3)) = 2.7e-4."""
    q, cache, table, lens, kv = problem(H + 1, [900, 300, 65, 1], H, 1)
    x = q.float() / 64.0
    x[..., 7:512:32] *= 1024.0
    q = x.to(torch.bfloat16)
    table = table_for(table, H, False)
    say(f"outliers within the bar H={H}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda())
    torch.cuda.synchronize()
    for b, n in enumerate(lens.tolist()):
        keys = R.gather(kv[:, :, 0], table[b], n)
        o, l, _, _ = exact(q[b], kv, keys, [n])
        assert (out[b].double().cpu() - o).abs().max() <= 1e-2 and (lse[b].double().cpu() - l).abs().max() <= 1e-3


def test_largest_latents(gpu):
    """Up to the largest bf16 value: what is stored reads back finite, to the nearest value that the format and bf16 hold,
    and a single token's decode gives it back."""
    g = torch.Generator().manual_seed(1)
    top = 3.3895313892515355e38
    kv = torch.randn(3, 64, 1, 576, generator=g)
    kv[..., 480:512] = 0.0
    kv[0, :, 0, 480:512] = torch.linspace(0.5, 1.0, 64)[:, None] * torch.linspace(-1, 1, 32) * top
    kv[0, 5, 0, 480:512] = top
    kv[1, 0, 0, 480:512] = -top
    kv = kv.to(torch.bfloat16)
    assert torch.isfinite(kv).all()
    say("largest latents")
    cache = quantize_kv_cache(kv.cuda(), bits=4)
    rows = kv_gather(cache, torch.arange(192, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 1, 128, 576, generator=g)
    q[..., 480:512] = 0.0
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    out, _ = mla_decode_with_kvcache(q.to(torch.bfloat16).cuda(), cache, one.reshape(1, 1), one)
    torch.cuda.synchronize()
    assert_cache(cache, *F4.quantize_pages(kv), "largest")
    got, want = rows[:, 480:512].double().cpu(), kv.reshape(192, 576)[:, 480:512].double()
    assert torch.isfinite(rows).all()
    # e2m1 is off by at most a quarter of the value or of the smallest step of its block; what lies past the largest
    # value, 1.5 * 2^127 (bf16 ends below 2^128), by a quarter too
    k = torch.exp2(torch.ceil(torch.log2(want.abs().amax(-1, keepdim=True) / 6)))
    assert ((got - want).abs() <= torch.maximum(want.abs() * 0.25, 0.25 * k)).all()
    assert torch.equal(out[0, 0, 0].cpu().double(), rows[64, :512].cpu().double()) and (out[0, 0, :, 480:] == -1.5 * 2.0 ** 127).all()


@pytest.mark.parametrize("H", [16, 24, 64, 128])
@pytest.mark.parametrize("sparse", [False, True])
def test_absorbed(gpu, H, sparse):
    q, cache, table, lens, _ = problem(5 + H, [400, 64, 1, 900], H, 1)
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(H, 512, 128, generator=g) * 512 ** -0.5).to(torch.bfloat16)
    wb = prepare_w_uv(w.cuda())
    say(f"absorbed H={H} sparse={sparse}")
    if sparse:
        nb = cache.latent.shape[0]
        cache = to_gpu(*F4.quantize_pages(torch.randn(nb, 64, 1, 576, generator=g).to(torch.bfloat16)))
        idx = torch.randint(0, nb * 64, (4, 1, 200), generator=g, dtype=torch.int32)
        idx[1, 0, ::3], idx[2] = -1, -1
        meta = get_mla_metadata(torch.zeros(4, dtype=torch.int32, device="cuda"), H, 1, topk=200, kv_cache=cache)
        out, lse = flash_mla_with_kvcache(q.cuda(), cache, None, None, 512, *meta, indices=idx.cuda())
        v, lse2 = mla_decode_absorbed(q.cuda(), cache, None, None, *meta, wb, indices=idx.cuda())
    else:
        d = (q.cuda(), cache, table_for(table, H, False).cuda(), lens.cuda())
        meta = get_mla_metadata(d[3], H, 1, kv_cache=cache)
        out, lse = flash_mla_with_kvcache(*d, 512, *meta, causal=True)
        v, lse2 = mla_decode_absorbed(*d, *meta, wb, causal=True)
    torch.cuda.synchronize()
    assert torch.equal(lse, lse2)
    o = out.double().cpu()
    want = torch.stack([o[:, :, h] @ w[h].double() for h in range(H)], 2)
    mag = torch.stack([o[:, :, h].abs() @ w[h].double().abs() for h in range(H)], 2)
    # v's own rounding (2^-8) and fp32 sums of 512 products
    assert ((v.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * mag).all()


@pytest.mark.parametrize("H", [40, 128, 200])
def test_a_schedule_for_few_pages_is_taken_with_a_wide_table(gpu, H):
    """The longest length that the host knows decides, not the table's width: the same workgroups, bit for bit."""
    q, cache, table, lens, kv = problem(H, [700, 64, 0, 333, 1], H, 1)
    wide = torch.nn.functional.pad(table, (0, 2000))
    ld = lens.cuda()
    say(f"few pages, wide table H={H}")
    meta = get_mla_metadata(ld, H, 1, kv_cache=cache, max_seqlen=700)
    out, lse = flash_mla_with_kvcache(q.cuda(), cache, wide.cuda(), ld, 512, *meta)
    want = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), ld, 512, *meta)
    torch.cuda.synchronize()
    assert_decode(out, lse, q, kv, wide, lens, False, f"wide table H={H}")
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
