"""GPU parity of the 4-bit latent cache: the quantizing append bit-exact against the format's oracle, and the decode
against the 64-bit attention of the dequantised cache, within a bound derived from the kernel's roundings."""
import math
import sys

import numpy as np
import pytest
import torch

from mlc_decode_amd import (Fp4KVCache, flash_mla_with_kvcache, fp4_kv_cache, get_mla_metadata, kv_append,
                            mla_decode_absorbed, mla_decode_with_kvcache, prepare_w_uv, quantize_kv_cache)
from mlc_decode_amd import _lib, api
from oracle import mla_fp4_ref as F4
from oracle import mla_ref as R

pytestmark = pytest.mark.gpu

SCALE = 576 ** -0.5


def say(msg):
    print(f"[gpu-fp4] {msg}", flush=True)
    sys.stdout.flush()


def varied_cache(nb, seed):
    """bf16 pages whose 32-dim blocks span many scales, with zero, tiny, huge and odd blocks."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(nb, 64, 1, 576, generator=g)
    mag = torch.exp2(torch.randint(-20, 20, (nb, 64, 1, 16), generator=g).float())
    kv[..., :512] = (kv[..., :512].reshape(nb, 64, 1, 16, 32) * mag[..., None]).reshape(nb, 64, 1, 512)
    kv[0, 3, 0, 32:64] = 0.0
    kv[0, 4, 0, :32] = 1e-38
    kv[0, 4, 0, 32:64] = 2.0 ** -133
    kv[0, 5, 0, 480:512] = 6.0
    kv[0, 6, 0, 480:512] = -3.0e38
    kv[0, 7, 0, 64] = float("nan")
    kv[0, 8, 0, 511] = float("inf")
    return kv.to(torch.bfloat16)


def to_gpu(codes, byte, rope):
    return Fp4KVCache(torch.from_numpy(codes).cuda(), torch.from_numpy(byte).cuda(), rope.cuda())


def assert_cache(c, codes, byte, rope, what):
    assert np.array_equal(c.scale.cpu().numpy(), byte), f"{what}: scales differ"
    bad = np.argwhere(c.latent.cpu().numpy() != codes)
    assert bad.size == 0, f"{what}: {len(bad)} code bytes differ, first {bad[:4].tolist()}"
    assert torch.equal(c.rope.cpu().view(torch.int16), rope.view(torch.int16)), f"{what}: rope differs"


def test_quantize_matches_oracle(gpu):
    kv = varied_cache(5, 0)
    say("quantize bits=4")
    got = quantize_kv_cache(kv.cuda(), bits=4)
    torch.cuda.synchronize()
    assert_cache(got, *F4.quantize_pages(kv), "quantize")


def test_every_bf16_value_rounds_alike(gpu):
    """All finite bf16 patterns against a block maximum of 6 * 2^e: the conversion's ties, signs and tiny values."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    v = bits.to(torch.int16).view(torch.bfloat16).float()
    e = torch.floor(torch.log2(v.clamp(min=2.0 ** -126)))
    x = torch.zeros(bits.numel(), 32)
    x[:, 0] = v
    x[:, 1] = -v
    x[:, 2] = (6.0 * torch.exp2((e + torch.arange(bits.numel()) % 5).clamp(max=125.0))).clamp(min=v)
    n = -(-bits.numel() // 16)
    rows = torch.zeros(n * 16, 32)
    rows[:bits.numel()] = x
    lat = rows.reshape(n, 512).to(torch.bfloat16)
    nb = -(-n // 64)
    kv = torch.zeros(nb * 64, 576, dtype=torch.bfloat16)
    kv[:n, :512] = lat
    kv = kv.reshape(nb, 64, 1, 576)
    say("every bf16 value")
    got = quantize_kv_cache(kv.cuda(), bits=4)
    torch.cuda.synchronize()
    assert_cache(got, *F4.quantize_pages(kv), "every value")


@pytest.mark.parametrize("n_new", [1, 2, 5, 17, 64])
def test_append_matches_oracle(gpu, n_new):
    g = torch.Generator().manual_seed(10 + n_new)
    nb, B = 24, 6
    codes, byte, rope = F4.quantize_pages(varied_cache(nb, n_new))
    table = torch.randperm(nb, generator=g).reshape(B, 4).to(torch.int32)
    table[4, 2] = nb  # a page outside the cache
    lens = torch.tensor([0, 63, 64, 150, 128, 255], dtype=torch.int32)  # the last runs past its table
    new = varied_cache(B, 100 + n_new).reshape(B, 64, 576)[:, :n_new].contiguous()
    cache, lens_d = to_gpu(codes, byte, rope), lens.cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    say(f"append n_new={n_new}")
    kv_append(new.cuda(), cache, table.cuda(), lens_d, status=status)
    torch.cuda.synchronize()
    codes2, byte2, rope2, lens2, skipped = F4.append_paged_fp4(codes, byte, rope, table, lens, new)
    assert 4 in skipped and (n_new == 1 or 5 in skipped)
    assert torch.equal(lens_d.cpu(), lens2) and status.item() == 1
    assert_cache(cache, codes2, byte2, rope2, f"append n_new={n_new}")


# ---------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------
def bound(q, k, see, o, lse):
    """Per-element bounds of one query's heads: q [H, 576], k [see, 576] in 64 bits, o, lse the exact result.

    Scores: hi holds q's block of 32 in a window that the MFMA adds exactly; lo is off by at most 2^-15 of the
    block's amax a, and its products (at most 2^-4 a |k|) may lose what lies 13 bits below their group's
    largest, at most 8 * 2^-17 a max|k| a group of eight: together below 2^-13 sum_d a_d |k_d|.  Adding 576
    products in fp32 is below 2^-14 of them with that.  Weights: bf16, half a step 2^-8, in numerator and
    denominator; a logit's error d is e^d - 1 of both.  Partials: fp16 with a scale per 128 dims, 2^-11 of
    the chunk's largest value.  The output's own rounding, 2^-8.  lse: the score bound, and fp32 logarithms
    and sums (2^-17 of the sum for up to 2^15 keys in any order)."""
    a = q[:, :512].reshape(-1, 16, 32).abs().amax(-1).repeat_interleave(32, -1)
    mag = torch.cat([a, q[:, 512:].abs()], -1)
    d = SCALE * (2.0 ** -13 + 2.0 ** -14) * (mag @ k.abs().T).amax(-1) + 2.0 ** -18 * (1 + lse.abs())
    w = torch.softmax(q @ k.T * SCALE, -1)
    A = w @ k[:, :512].abs()
    tol = 2.0 ** -8 * o.abs() + (2 * 2.0 ** -8 + 2 * d[:, None]) * A * 1.01 + 2.0 ** -11 * k[:, :512].abs().amax()
    return tol, d + 2.0 ** -17


def exact(q, kv, keys, visible):
    """Attention in 64 bits of one sequence: q [s_q, H, 576], its keys [L, 576], visible [s_q] counts."""
    s_q, H, _ = q.shape
    o, t = torch.zeros(s_q, H, 512, dtype=torch.float64), torch.zeros(s_q, H, 512, dtype=torch.float64)
    l, lt = torch.full((H, s_q), -math.inf, dtype=torch.float64), torch.zeros(H, s_q, dtype=torch.float64)
    for i, n in enumerate(visible):
        if n > 0:
            qi, k = q[i].double(), keys[:n]
            s = qi @ k.T * SCALE
            l[:, i] = torch.logsumexp(s, -1)
            o[i] = torch.softmax(s, -1) @ k[:, :512]
            t[i], lt[:, i] = bound(qi, k, n, o[i], l[:, i])
    return o, l, t, lt


def assert_decode(out, lse, q, kv, table, lens, causal, what, indices=None):
    out, lse = out.double().cpu(), lse.double().cpu()
    flat = kv.reshape(-1, 576)
    for b in range(q.shape[0]):
        if indices is not None:
            ids = indices[b]
            keys = flat[ids[(ids >= 0) & (ids < flat.shape[0])].long()]
            visible = [keys.shape[0]]
        else:
            L = max(0, min(int(lens[b]), 64 * table.shape[1]))
            keys = R.gather(kv[:, :, 0], table[b].clamp(0, kv.shape[0] - 1), L)
            visible = [L - (q.shape[1] - 1 - i if causal else 0) for i in range(q.shape[1])]
        o, l, t, lt = exact(q[b], kv, keys, visible)
        err = (out[b] - o).abs()
        assert (err <= t).all(), f"{what} seq {b}: out off by {err.max():.3e}, bound {t.flatten()[err.argmax()]:.3e}"
        fin = torch.isfinite(l)
        assert torch.equal(torch.isfinite(lse[b]), fin), f"{what} seq {b}: lse of empty rows"
        assert ((lse[b] - l).abs()[fin] <= lt[fin]).all(), f"{what} seq {b}: lse off by {(lse[b] - l).abs()[fin].max():.3e}"


def problem(seed, lens, H, s_q, sigma=1.0, spare=1, poison=True):
    """Queries, a 4-bit cache with poisoned rows behind every sequence's end, table, lengths, and the exact cache."""
    g = torch.Generator().manual_seed(seed)
    pages = [(n + 63) // 64 for n in lens]
    nb = sum(pages) + spare
    kv = (torch.randn(nb, 64, 1, 576, generator=g) * sigma).to(torch.bfloat16)
    codes, byte, rope = F4.quantize_pages(kv)
    table = torch.zeros(len(lens), max(max(pages), 1), dtype=torch.int32)
    order, at = torch.randperm(nb, generator=g), 0
    exactkv = F4.dequantize_pages(codes, byte, rope)
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
        if poison and lens[b] % 64:
            pg, row = int(table[b, n - 1]), lens[b] % 64
            byte[pg, row:], rope[pg, row:] = 255, float("nan")
            codes[pg, row:] = 0x77
    q = (torch.randn(len(lens), s_q, H, 576, generator=g) * sigma).to(torch.bfloat16)
    return q, to_gpu(codes, byte, rope), table, torch.tensor(lens, dtype=torch.int32), exactkv


FEW = 6144  # table columns times row tiles of 16 up to which the decode takes workgroups of 16 rows


def table_for(table, rows, few):
    """The table as it is (few pages), or with columns behind it that make the decode take its forms for many."""
    tiles = (rows + 15) // 16
    if few:
        assert table.numel() * tiles <= FEW
        return table
    return torch.nn.functional.pad(table, (0, FEW // (tiles * table.shape[0]) + 1))


LENS = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700]


@pytest.mark.parametrize("H,s_q", [(1, 1), (8, 1), (16, 1), (17, 1), (32, 1), (40, 1), (64, 1), (100, 1), (128, 1), (16, 2), (5, 3), (64, 2), (128, 2), (40, 4)])
@pytest.mark.parametrize("few", [False, True])
def test_decode_rows(gpu, H, s_q, few):
    q, cache, table, lens, kv = problem(H * 8 + s_q, LENS, H, s_q)
    table = table_for(table, H * s_q, few)
    d = (q.cuda(), cache, table.cuda(), lens.cuda())
    say(f"decode H={H} s_q={s_q}")
    for splits in (None, 1, 3):
        out, lse = mla_decode_with_kvcache(*d, num_splits=splits, causal=True)
        torch.cuda.synchronize()
        assert_decode(out, lse, q, kv, table, lens, True, f"H={H} s_q={s_q} splits={splits}")


@pytest.mark.parametrize("H", [16, 32, 128])
@pytest.mark.parametrize("few", [False, True])
def test_decode_without_mask_and_scales(gpu, H, few):
    q, cache, table, lens, kv = problem(7, [5, 200, 64], H, 2, sigma=3.0)
    table = table_for(table, 2 * H, few)
    say(f"decode no mask H={H}")
    out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), causal=False)
    torch.cuda.synchronize()
    assert_decode(out, lse, q, kv, table, lens, False, f"no mask H={H}")


@pytest.mark.parametrize("H", [16, 24, 64, 128])
@pytest.mark.parametrize("parts", [1, 2, 7, 64])
@pytest.mark.parametrize("few", [False, True])
def test_decode_schedules(gpu, H, parts, few):
    """Any schedule: parts that span sequences, sequences that span parts, parts with nothing to do."""
    q, cache, table, lens, kv = problem(50 + H, [300, 1, 0, 2000, 64, 65], H, 1)
    table = table_for(table, H, few)
    say(f"decode parts={parts} H={H}")
    ld = lens.cuda()
    sched, splits = get_mla_metadata(ld, H, 1, num_parts=parts)
    out, lse = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), ld, 512, sched, splits)
    torch.cuda.synchronize()
    assert_decode(out, lse, q, kv, table, lens, False, f"parts={parts} H={H}")


def test_decode_long_and_rising_scores(gpu):
    """Each page's scores pass the last one's by far: the running reference moves with nearly every page; and the
    other way round, where it never moves again."""
    H = 16
    q, cache, table, lens, _ = problem(3, [1500, 1500], H, 1)
    codes, byte = cache.latent.cpu().numpy(), cache.scale.cpu().numpy()
    rope = cache.rope.cpu()
    for b in range(2):
        for i in range(24):
            r = i if b == 0 else 23 - i
            rope[int(table[b, i])] = (q[b, 0, 0, 512:].float().sign() * 0.5 * r).to(torch.bfloat16)
    cache = cache._replace(rope=rope.cuda())
    kv = F4.dequantize_pages(codes, byte, rope)
    say("decode rising scores")
    for splits in (1, 2):
        out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), num_splits=splits)
        torch.cuda.synchronize()
        assert_decode(out, lse, q, kv, table, lens, True, f"rising splits={splits}")


@pytest.mark.parametrize("H", [16, 48, 128])
def test_decode_strides_and_views(gpu, H):
    """Padded pages and rows of the cache, queries that are a view, an output with padded heads, a wider table."""
    q, cache, table, lens, kv = problem(90, [130, 64, 1], H, 1)
    nb = cache.latent.shape[0]
    lat = torch.full((nb, 70, 288), 0x77, dtype=torch.uint8, device="cuda")
    sc = torch.full((nb, 66, 32), 255, dtype=torch.uint8, device="cuda")
    rp = torch.full((nb, 65, 72), float("nan"), dtype=torch.bfloat16, device="cuda")
    lat[:, :64, :256], sc[:, :64, :16], rp[:, :64, :64] = cache
    wide = Fp4KVCache(lat[:, :64, :256], sc[:, :64, :16], rp[:, :64, :64])
    qw = torch.full((3, 1, H, 640), float("nan"), dtype=torch.bfloat16, device="cuda")
    qw[..., :576] = q.cuda()
    tw = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    tw[:, :table.shape[1]] = table.cuda()
    out = torch.full((3, 1, H, 520), 9.0, dtype=torch.bfloat16, device="cuda")
    say(f"decode strides H={H}")
    sched, splits = get_mla_metadata(lens.cuda(), H, 1, kv_cache=wide)
    got, lse = flash_mla_with_kvcache(qw[..., :576], wide, tw, lens.cuda(), 512, sched, splits, out=out[..., :512])
    torch.cuda.synchronize()
    assert_decode(got, lse, q, kv, table, lens, False, f"strides H={H}")
    assert (out[..., 512:] == 9.0).all()


def test_decode_cut_at_the_table_and_foreign_pages(gpu):
    H = 16
    q, cache, table, lens, kv = problem(12, [640, 100], H, 1, poison=False)
    short = table[:, :4].clone()
    short[1, 0] = 10 ** 6  # clamped into the pool, as with the other formats
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    say("decode cut at the table")
    sched, splits = get_mla_metadata(lens.cuda(), H, 1)
    out, lse = flash_mla_with_kvcache(q.cuda(), cache, short.cuda(), lens.cuda(), 512, sched, splits, status=status)
    torch.cuda.synchronize()
    assert status.item() == 1
    assert_decode(out, lse, q, kv, short, lens, False, "cut")


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("few", [False, True])
def test_decode_far_pages(gpu, H, few):
    """Pages past 4 GiB from the pool's start."""
    nb, gap = 72, 1 << 26
    buf = torch.empty(nb * gap, dtype=torch.uint8, device="cuda")
    q, cache, table, lens, kv = problem(33, [200, 64 * 60 + 3], H, 1, spare=nb - 65)
    table = table_for(table, H, few)
    far = buf.as_strided((nb, 64, 256), (gap, 256, 1))
    far.copy_(cache.latent)
    sc = buf.as_strided((nb, 64, 16), (gap, 16, 1), 1 << 20)
    sc.copy_(cache.scale)
    say(f"decode far pages H={H}")
    out, lse = mla_decode_with_kvcache(q.cuda(), Fp4KVCache(far, sc, cache.rope), table.cuda(), lens.cuda())
    torch.cuda.synchronize()
    assert_decode(out, lse, q, kv, table, lens, True, f"far H={H}")


def test_decode_nan_block_stays_with_its_sequence(gpu):
    H = 20
    q, cache, table, lens, kv = problem(44, [100, 100], H, 1)
    cache.scale[int(table[0, 0]), 7, 3] = 255
    say("decode NaN block")
    for splits in (1, 2):  # a NaN row's lse is -inf, as with the other formats
        out, lse = mla_decode_with_kvcache(q.cuda(), cache, table.cuda(), lens.cuda(), num_splits=splits)
        torch.cuda.synchronize()
        assert torch.isnan(out[0]).all() and (lse[0] == -math.inf).all()
        assert_decode(out[1:], lse[1:], q[1:], kv, table[1:], lens[1:], True, f"beside a NaN, splits={splits}")


@pytest.mark.parametrize("H", [16, 32, 64, 128])
@pytest.mark.parametrize("topk", [1, 63, 64, 200, 2048])
@pytest.mark.parametrize("parts", [None, 512])  # 512: more than the form for few pages is taken with
def test_sparse(gpu, H, topk, parts):
    g = torch.Generator().manual_seed(topk + H)
    nb, B = 40, 3
    kv = torch.randn(nb, 64, 1, 576, generator=g).to(torch.bfloat16)
    codes, byte, rope = F4.quantize_pages(kv)
    idx = torch.randint(0, nb * 64, (B, topk), generator=g, dtype=torch.int32)
    idx[1, ::3] = -1
    idx[1, 1::7] = nb * 64 + 5
    idx[2] = -1
    q = torch.randn(B, 1, H, 576, generator=g).to(torch.bfloat16)
    cache = to_gpu(codes, byte, rope)
    say(f"sparse H={H} topk={topk}")
    sched, splits = get_mla_metadata(torch.zeros(B, dtype=torch.int32, device="cuda"), H, 1, parts, topk=topk, kv_cache=cache)
    out, lse = flash_mla_with_kvcache(q.cuda(), cache, None, None, 512, sched, splits, indices=idx.cuda().unsqueeze(1))
    torch.cuda.synchronize()
    assert_decode(out, lse, q, F4.dequantize_pages(codes, byte, rope), None, None, False, f"sparse H={H} topk={topk}", indices=idx)


@pytest.mark.parametrize("H", [33, 64, 128, 200])
@pytest.mark.parametrize("B", [3, 70, 200])
def test_one_page_a_sequence(gpu, H, B):
    """One column: no splits, whatever the schedule; with many sequences the forms for more rows again."""
    q, cache, table, lens, kv = problem(H + B, [(7 * b) % 65 for b in range(B)], H, 1)
    ld = lens.cuda()
    say(f"one page H={H} B={B}")
    sched, splits = get_mla_metadata(ld, H, 1, kv_cache=cache)
    o, lse = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), ld, 512, sched, splits)
    torch.cuda.synchronize()
    assert_decode(o, lse, q, kv, table, lens, False, f"one page H={H} B={B}")


@pytest.mark.parametrize("H", [33, 128, 200])
def test_schedule_for_few_pages(gpu, H):
    """A schedule made with the longest length a host knows has fewer parts, and decodes the same."""
    q, cache, table, lens, kv = problem(H, [0, 1, 700, 64], H, 1)
    ld = lens.cuda()
    say(f"few pages H={H}")
    out = []
    for longest in (None, 64 * table.shape[1]):
        sched, splits = get_mla_metadata(ld, H, 1, kv_cache=cache, max_seqlen=longest)
        o, lse = flash_mla_with_kvcache(q.cuda(), cache, table.cuda(), ld, 512, sched, splits)
        torch.cuda.synchronize()
        assert_decode(o, lse, q, kv, table, lens, False, f"few pages H={H} {longest}")
        out.append(sched.shape[0] * ((H + 15) // 16))
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert out[1] <= 2 * cus < out[0]
    with pytest.raises(ValueError, match="max_seqlen"):
        get_mla_metadata(ld, H, 1, kv_cache=cache, max_seqlen=-1)


def test_absorbed_and_noalloc_agree_with_the_decode(gpu):
    H = 64
    q, cache, table, lens, _ = problem(5, [400, 64, 1, 900], H, 1)
    g = torch.Generator().manual_seed(1)
    w = (torch.randn(H, 512, 128, generator=g) * 512 ** -0.5).to(torch.bfloat16)
    d = (q.cuda(), cache, table.cuda(), lens.cuda())
    say("absorbed, noalloc")
    sched, splits = get_mla_metadata(d[3], H, 1, forced_splits=3)
    out, lse = flash_mla_with_kvcache(*d, 512, sched, splits, causal=True)
    v, lse2 = mla_decode_absorbed(*d, sched, splits, prepare_w_uv(w.cuda()), causal=True)
    a, out3, lse3, keep = api.make_decode_args(*d, sched, splits, SCALE, True)
    a.workspace, a.workspace_bytes = None, 0
    import ctypes
    _lib.check("mla_decode_fwd_noalloc", _lib.load().mla_decode_fwd_noalloc(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, out3) and torch.equal(lse, lse3) and torch.equal(lse, lse2)
    o = out.double().cpu()
    want = torch.einsum("bshk,hkn->bshn", o, w.double())
    mag = torch.einsum("bshk,hkn->bshn", o.abs(), w.double().abs())
    # v's own rounding (2^-8) and fp32 sums of 512 products
    assert ((v.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * mag).all()


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("few", [False, True])
def test_two_graphs_of_one_decode(gpu, H, few):
    """Schedule and decode captured twice on one stream (they share a workspace), replayed in turn with lengths that change in
    place and eager decodes between: each replay is the eager call's result bit for bit."""
    q, cache, table, lens, _ = problem(8, [1000, 300, 64, 5], H, 1, poison=False)
    table = table_for(table, H, few).cuda()
    qd, ld = [q.cuda(), q.flip(0).cuda()], lens.cuda()
    say(f"two graphs H={H} few={few}")
    eager = lambda i: mla_decode_with_kvcache(qd[i], cache, table, ld)  # noqa: E731
    eager(0)
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            held.append(eager(i))
    for new in ([1000, 300, 64, 5], [0, 1, 63, 64], [512, 299, 1, 0], [1000, 300, 64, 5]):
        ld.copy_(torch.tensor(new, dtype=torch.int32))
        for i in (0, 1):
            graphs[i].replay()
            out, lse = (t.clone() for t in held[i])
            want = eager(i)
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), f"graph {i} lens {new}"


@pytest.mark.parametrize("few", [False, True])
def test_same_result_on_another_stream_and_twice(gpu, few):
    H = 128
    q, cache, table, lens, _ = problem(6, [1000, 300, 64, 5], H, 1)
    table = table_for(table, H, few)
    d = (q.cuda(), cache, table.cuda(), lens.cuda())
    say("two streams")
    out, lse = mla_decode_with_kvcache(*d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out2, lse2 = mla_decode_with_kvcache(*d)
    out3, lse3 = mla_decode_with_kvcache(*d)
    torch.cuda.synchronize()
    for o, l in ((out2, lse2), (out3, lse3)):
        assert torch.equal(out, o) and torch.equal(lse, l)


def test_empty_cache_decodes_zero_tokens(gpu):
    cache = fp4_kv_cache(3)
    q = torch.randn(2, 1, 16, 576, device="cuda").to(torch.bfloat16)
    lens = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 0], [1, 2]], dtype=torch.int32, device="cuda")
    out, lse = mla_decode_with_kvcache(q, cache, table, lens)
    torch.cuda.synchronize()
    assert (out == 0).all() and torch.isinf(lse[0]).all()
    assert torch.allclose(lse[1], torch.full_like(lse[1], math.log(70)), atol=1e-5)
