"""GPU tests of the operators on drafted tokens: whole numbers against the oracle exactly, the tree decode against the
64-bit attention of the dequantised cache within a bound derived from its roundings."""
import random
import sys

import pytest
import torch

import mlc_decode_amd as M
from mlc_decode_amd import api
from oracle import mla_tree_ref as T

pytestmark = pytest.mark.gpu

SCALE = 576 ** -0.5
INF, NAN = float("inf"), float("nan")


def say(msg):
    print(f"[gpu-drafts] {msg}", flush=True)
    sys.stdout.flush()


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def random_parents(rng, s, drop=0.15):
    return [-1 if i == 0 or rng.random() < 0.05 else rng.choice((-2, i, i + 3, 99)) if rng.random() < drop else rng.randrange(i) for i in range(s)]


# ---------------------------------------------------------------------------------------
# plan, accept, keep
# ---------------------------------------------------------------------------------------
def check_plan(parents, lens, table, tree_lens=None, width=None):
    t = ints(table)
    if width is not None:  # a view of a wider table
        t = t[:, :width]
    got = M.tree_plan(ints(parents), ints(lens), t, ints(tree_lens) if tree_lens is not None else None)
    torch.cuda.synchronize()
    mask, pos, slots, prefix = T.plan(parents, lens, [r[:width] for r in table], tree_lens)
    assert got.mask.tolist() == [[T.bits(line) for line in row] for row in mask]
    assert got.positions.tolist() == pos and got.slots.tolist() == slots and got.prefix_lens.tolist() == prefix
    return got, mask


@pytest.mark.parametrize("s", [1, 2, 3, 7, 16, 33, 63, 64])
def test_plan(gpu, s):
    rng = random.Random(s)
    B = 37
    say(f"plan s={s}")
    parents = [random_parents(rng, s) for _ in range(B)]
    parents[0] = [i - 1 for i in range(s)]                       # a chain
    parents[1] = [-1] * s                                        # roots alone
    parents[2] = [-1] + [0] * (s - 1)                            # a star
    parents[3] = [-2] * s                                        # nothing
    lens = [rng.choice((0, s - 1, s, s + 1, 64, 127, 190, rng.randrange(400))) for _ in range(B)]
    lens[4], lens[5] = -3, 0
    table = [[rng.randrange(1000) for _ in range(7)] for _ in range(B)]
    table[6][1], table[7][2] = -1, 2 ** 31 // 64
    check_plan(parents, lens, table)
    check_plan(parents, lens, table, [rng.choice((-1, 0, 1, s, s + 5, rng.randrange(s + 1))) for _ in range(B)])
    check_plan(parents, lens, table, width=2)


def test_plan_of_nothing_and_refusals(gpu):
    say("plan refusals")
    e = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert M.tree_plan(e, e[:, 0], e).mask.shape == (0, 4)
    p, n, t = ints([[-1, 0]] * 3), ints([5] * 3), ints([[0]] * 3)
    for args in [(p.long(), n, t), (p, n.long(), t), (p, n[:2], t), (p, n, t.long()), (p, n, t[:2]), (p, n, t[:, 0]), (p[:, :0], n, t),
                 (ints([[-1] * 65] * 3), n, t), (p[:, ::2], n, t), (p, n, t, n[:2]), (p, n, t, n.cpu()), (p, n, ints([[0, 1]] * 3).T[:3].T[:, ::2].T[:1])]:
        with pytest.raises(ValueError):
            M.tree_plan(*args)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("s", [1, 2, 5, 16, 40, 64])
def test_accept(gpu, s, dtype):
    rng = random.Random(10 * s)
    B = 61
    say(f"accept s={s} {dtype}")
    parents = [random_parents(rng, s, 0.1) for _ in range(B)]
    parents[0] = [i - 1 for i in range(s)]
    parents[1] = [-2] + [-1] * (s - 1)  # node 0 is none
    tree_lens = [s] * (B - 3) + [0, max(s - 2, 0), s]
    table = [list(range(b, b + 4)) for b in range(B)]
    plan, mask = check_plan(parents, [rng.randrange(s, 200) for _ in range(B)], table, tree_lens)
    big = 2 ** 40 if dtype is torch.int64 else 0
    tokens = [[big + rng.randrange(2) for _ in range(s)] for _ in range(B)]  # many agree, siblings often alike
    targets = [[big + rng.randrange(2) for _ in range(s)] for _ in range(B)]
    tokens[0] = targets[0] = [big] * s  # the whole chain
    got = M.tree_accept(plan, ints(tokens, dtype), ints(targets, dtype))
    torch.cuda.synchronize()
    path, counts, after, keep = T.accept(mask, plan.prefix_lens.tolist(), tokens, targets)
    assert got.path.tolist() == path and got.counts.tolist() == counts and got.keep_lens.tolist() == keep
    assert got.next_tokens.dtype == dtype and got.next_tokens.tolist() == after
    assert counts[0] == s and counts[1] == 0


def test_accept_refusals(gpu):
    say("accept refusals")
    plan = M.tree_plan(ints([[-1, 0]] * 3), ints([5] * 3), ints([[0]] * 3))
    t = ints([[0, 1]] * 3)
    for args in [(plan, t, t.long()), (plan, t.float(), t.float()), (plan, t[:2], t[:2]), (plan, t, t[:, :1]), (plan, t[0], t[0]),
                 (plan._replace(mask=plan.mask.int()), t, t), (plan._replace(prefix_lens=plan.prefix_lens[:2]), t, t)]:
        with pytest.raises(ValueError):
            M.tree_accept(*args)


FORMATS = ["bf16", "f16", "fp8", "fp4", "pair"]


def make_cache(fmt, pages, seed, spread=True):
    """(cache, rows [pages, 64, 576] in 64 bits), random with blocks of many scales where the format is coded."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(pages, 64, 1, 576, generator=g)
    if fmt in ("fp8", "fp4") and spread:
        mag = torch.exp2(torch.randint(-3, 2, (pages, 64, 1, 16), generator=g).float())
        kv[..., :512] = (kv[..., :512].reshape(pages, 64, 1, 16, 32) * mag[..., None]).reshape(pages, 64, 1, 512)
    kv = kv.to(torch.float16 if fmt == "f16" else torch.bfloat16).cuda()
    cache = M.quantize_kv_cache(kv, bits=4 if fmt == "fp4" else 8) if fmt in ("fp8", "fp4") else kv
    if fmt == "pair":  # two tensors, rows further apart than they are long
        wide = torch.zeros(pages, 64, 1, 640, dtype=torch.bfloat16, device="cuda")
        wide[..., :512] = kv[..., :512]
        cache = (wide[..., :512], kv[..., 512:].contiguous())
    rows = M.kv_gather(cache, torch.arange(pages * 64, dtype=torch.int32, device="cuda"))
    return cache, rows.double().cpu().view(pages, 64, 576)


def parts_of(cache):
    return [cache] if isinstance(cache, torch.Tensor) else list(cache)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("s", [1, 5, 8, 9, 17, 64])
def test_keep_path(gpu, fmt, s):
    rng = random.Random(s)
    B, pages = 9, 24
    cache, rows = make_cache(fmt, pages, s)
    say(f"keep {fmt} s={s}")
    order = list(range(pages * 64))
    rng.shuffle(order)
    slots = [order[b * s:(b + 1) * s] for b in range(B)]
    path = []
    for b in range(B):
        keep = sorted(rng.sample(range(1, s), rng.randrange(s))) if s > 1 else []
        path.append([0] + keep + [-1] * (s - 1 - len(keep)))
    path[0] = list(range(s))                                   # nothing moves
    path[1] = [-1] * s
    path[2] = list(range(1, s)) + [-1]                         # everything by one
    path[3] = [s - 1] * s                                      # the same row to all
    path[4] = [0, 0, 1, s, 2 ** 30][:s] + [-1] * max(s - 5, 0)   # below their place, past the tree
    slots[5] = [-1 if i % 3 == 1 else v for i, v in enumerate(slots[5])]
    slots[6][0] = pages * 64 + 5
    want = [t.clone() for t in parts_of(cache)]
    flat = [t for t in want]
    for b in range(B):
        moves = [(slots[b][k], slots[b][j]) for k, j in enumerate(path[b]) if k < j < s and 0 <= slots[b][k] < pages * 64 and 0 <= slots[b][j] < pages * 64]
        for t, old in zip(flat, parts_of(cache)):
            for dst, src in moves:
                if t.dtype == torch.float32:  # the fp8 cache's scales: [page, block, row]
                    t[dst // 64, :, dst % 64] = old[src // 64, :, src % 64]
                else:
                    t[dst // 64, dst % 64] = old[src // 64, src % 64]
    M.kv_keep_path(cache, ints(slots), ints(path))
    torch.cuda.synchronize()
    for t, w in zip(parts_of(cache), want):
        assert torch.equal(t.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def test_keep_refusals(gpu):
    say("keep refusals")
    cache, _ = make_cache("bf16", 2, 0)
    t = ints([[0, 1]] * 3)
    for args in [(cache, t.long(), t), (cache, t, t.long()), (cache, t[:2], t), (cache, t[0], t[0]), (cache, ints([[0] * 65]), ints([[0] * 65])), (cache, t.cpu(), t)]:
        with pytest.raises(ValueError):
            M.kv_keep_path(*args)
    M.kv_keep_path(cache, t[:0], t[:0])


# ---------------------------------------------------------------------------------------
# the decode
# ---------------------------------------------------------------------------------------
def bounds(q, o, lse, size, reach, keys, dtype, fmt, rows):
    """Of each output and lse.  eps is half a step of the 16-bit type.  A score is a sum of 576 fp32 products, below
    2^-14 of sum |q k| off; a 4-bit cache above 32 rows loses another 2^-13 of that sum taken with the largest |q| of
    each block of 32 in all its places (`reach` is made so).  Weights: rounded to 16 bits in numerator and denominator, 2
    eps; a score's error d makes e^2d - 1.  The output's rounding is eps, a partial's 2^-11 (its chunk's largest takes
    the place of its own value, which covers those that are subnormal next to it).  lse: d, its sum of `keys` terms in
    fp32, and the fast exponential and logarithm, 2^-20 of 1 + |lse|."""
    eps = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    d = reach * (2.0 ** -14 if fmt != "fp4" or rows <= 32 else 2.0 ** -13 + 2.0 ** -14) + 2.0 ** -20 * (1 + lse.abs().nan_to_num(0, 0, 0))
    dd = torch.expm1(2 * d).transpose(1, 2)[..., None]
    chunk = size.unflatten(-1, (4, 128)).amax(-1, keepdim=True).expand(*size.shape[:-1], 4, 128).flatten(-2)
    return (3 * eps + 8 * eps * eps + dd) * size + 2.0 ** -11 * chunk + 2.0 ** -24, d + keys * 2.0 ** -24


def check_decode(q, cache, rows, table, plan, mask, fmt, got, what, skip=()):
    out, lse = got
    ro, rl, size, reach = T.attend(q.double().cpu(), rows, table.cpu(), plan.prefix_lens.tolist(), mask, SCALE)
    if fmt == "fp4":  # the bound of the split queries takes each block's largest in every place of it
        a = q.double().cpu()[..., :512].unflatten(-1, (16, 32)).abs().amax(-1, keepdim=True).expand(*q.shape[:-1], 16, 32).flatten(-2)
        reach = T.attend(torch.cat([a, q.double().cpu()[..., 512:].abs()], -1), rows.abs(), table.cpu(), plan.prefix_lens.tolist(), mask, SCALE)[3]
    keys = max(plan.prefix_lens.tolist() + [0]) + q.shape[1]
    to, tl = bounds(q, ro, rl, size, reach, keys, q.dtype, fmt, q.shape[1] * q.shape[2])
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(lse == -INF, rl == -INF), f"{what}: empty rows differ"
    fine = rl != -INF
    assert torch.isfinite(out).all(), what
    eo = ((out - ro).abs() / to).max().item()
    el = ((lse - rl).abs()[fine] / tl[fine]).max().item() if fine.any() else 0.0
    say(f"{what}: out {eo:.3f} of its bound, lse {el:.3f}")
    assert (out[~fine.transpose(1, 2)] == 0).all(), f"{what}: a row without a key is not zero"
    assert eo <= 1 and el <= 1, what


def problem(fmt, H, s, prefixes, seed, tree_lens=None, drop=0.15, extra=1, max_pages=None):
    rng = random.Random(seed)
    B = len(prefixes)
    n = tree_lens or [s] * B
    lens = [p + t for p, t in zip(prefixes, n)]
    width = max_pages or max(-(-v // 64) for v in lens + [1]) + extra
    pages = B * width
    order = list(range(pages))
    rng.shuffle(order)
    table = ints([order[b * width:(b + 1) * width] for b in range(B)])
    cache, rows = make_cache(fmt, pages, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(B, s, H, 576, generator=g).to(torch.float16 if fmt == "f16" else torch.bfloat16).cuda()
    parents = [random_parents(rng, s, drop) for _ in range(B)]
    plan = M.tree_plan(ints(parents), ints(lens), table, ints(n))
    mask = T.plan(parents, lens, table.tolist(), n)[0]
    return q, cache, rows, table, plan, mask


def decode(q, cache, table, plan, **kw):
    sched = M.get_mla_metadata(plan.prefix_lens, q.shape[1] * q.shape[2], 1, kv_cache=cache, **kw)
    return M.flash_mla_with_kvcache(q, cache, table, None, 512, *sched, tree=plan)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,s", [(1, 1), (2, 3), (16, 1), (5, 7), (16, 2), (16, 5), (24, 3), (128, 2), (16, 17), (3, 33), (8, 64), (130, 1)])
def test_decode(gpu, fmt, H, s):
    prefixes = [0, 1, 63, 64, 65, 200, 130]
    q, cache, rows, table, plan, mask = problem(fmt, H, s, prefixes, 1000 + 10 * H + s)
    say(f"decode {fmt} H={H} s={s}")
    got = decode(q, cache, table, plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, fmt, got, f"{fmt} H={H} s={s}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,s", [(1, 1), (2, 3), (16, 5), (3, 33), (8, 64), (128, 8), (100, 8), (40, 33), (16, 64)])
def test_decode_behind_a_wide_table(gpu, fmt, H, s):
    """A table too wide for the decode of pages by themselves: the split-KV pass over the schedule, then the drafted
    tokens, by 16 rows and by 64."""
    prefixes = [0, 1, 63, 64, 65, 200, 130]
    q, cache, rows, table, plan, mask = problem(fmt, H, s, prefixes, 2000 + 10 * H + s)
    wide = table.repeat(1, -(-600 // table.shape[1]))[:, :600]
    code = {"fp8": 1, "fp4": 4}.get(fmt, 0)
    sched = M.get_mla_metadata(plan.prefix_lens, H * s, 1, kv_cache=cache)
    lib = M._lib.load()
    assert not lib.mla_tree_takes_pages(7, s, H, sched[0].shape[0], code, 600) and api._tree_without_schedule(7, s, H, code, 600) is None
    say(f"wide table {fmt} H={H} s={s}")
    got = decode(q, cache, wide, plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, fmt, got, f"wide {fmt} H={H} s={s}")
    auto = M.mla_decode_with_kvcache(q, cache, wide, None, tree=plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, fmt, auto, f"wide auto {fmt} H={H} s={s}")


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_decode_ragged_trees(gpu, fmt):
    prefixes, n = [0, 0, 40, 60, 300, 5, 128], [0, 3, 12, 1, 7, 0, 12]
    q, cache, rows, table, plan, mask = problem(fmt, 16, 12, prefixes, 7, tree_lens=n)
    say(f"ragged {fmt}")
    got = decode(q, cache, table, plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, fmt, got, f"ragged {fmt}")
    assert (got[1][0] == -INF).all() and (got[0][0] == 0).all()  # neither a prefix nor a tree


@pytest.mark.parametrize("splits", [1, 2, 7])
def test_decode_forced_splits_and_auto(gpu, splits):
    q, cache, rows, table, plan, mask = problem("bf16", 16, 6, [700, 64, 0, 129], 11)
    say(f"forced {splits}")
    got = M.mla_decode_with_kvcache(q, cache, table, None, num_splits=splits, tree=plan)
    auto = M.mla_decode_with_kvcache(q, cache, table, None, tree=plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, "bf16", got, f"splits {splits}")
    check_decode(q, cache, rows, table, plan, mask, "bf16", auto, "auto")


@pytest.mark.parametrize("parts", [255, 256, 300])
def test_decode_many_splits(gpu, parts):
    """One long sequence in as many splits as there are parts, and the drafted tokens' one more."""
    q, cache, rows, table, plan, mask = problem("bf16", 2, 4, [64 * 320 + 9], 13)
    say(f"one sequence in {parts} parts")
    got = decode(q, cache, table, plan, num_parts=parts, fixed_overhead=0)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, "bf16", got, f"{parts} parts")


def test_chain_is_the_causal_decode(gpu):
    """A tree without branches sees what the causal decode sees."""
    q, cache, rows, table, _, _ = problem("bf16", 16, 5, [200, 64, 3], 17)
    lens = ints([205, 69, 8])
    plan = M.tree_plan(ints([[-1, 0, 1, 2, 3]] * 3), lens, table)
    say("chain")
    a = decode(q, cache, table, plan)
    b = M.mla_decode_with_kvcache(q, cache, table, lens)
    torch.cuda.synchronize()
    mask = [[set(range(i + 1)) for i in range(5)]] * 3
    check_decode(q, cache, rows, table, plan, mask, "bf16", a, "chain")
    # both are within the bounds of one exact result: twice them apart at most
    ro, rl, size, reach = T.attend(q.double().cpu(), rows, table.cpu(), plan.prefix_lens.tolist(), mask, SCALE)
    to, tl = bounds(q, ro, rl, size, reach, 210, q.dtype, "bf16", 80)
    assert ((a[0] - b[0]).double().cpu().abs() <= 2 * to).all() and ((a[1] - b[1]).double().cpu().abs() <= 2 * tl).all()


def test_masks_of_ones_own(gpu):
    """Any bits: a row that does not see itself, rows that see none, later tokens; bits past s_q name nothing."""
    q, cache, rows, table, plan, _ = problem("bf16", 8, 6, [70, 0, 0], 19)
    sets = [[{0}, {5}, set(), {1, 3}, {0, 1, 2, 3, 4, 5}, {2}], [set(), {0}, {3}, set(), {5, 0}, {4}], [set()] * 6]
    words = [[T.bits(v | {6, 9, 63}) for v in row] for row in sets]
    plan = plan._replace(mask=ints(words, torch.int64))
    say("own masks")
    got = decode(q, cache, table, plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, sets, "bf16", got, "own masks")


def test_tokens_past_the_table(gpu):
    """Drafted tokens behind the table's last column are no keys, and raise the status; so does a prefix longer than it."""
    q, cache, rows, table, plan, mask = problem("bf16", 8, 6, [60, 120], 23, extra=0)
    assert table.shape[1] == 2
    for prefix, raised in (([60, 120], 0), ([60, 125], 1), ([60, 128], 1), ([60, 200], 1), ([-5, 2 ** 31 - 10], 1)):
        for t in (table, torch.cat([table, torch.full_like(table, 10 ** 6)], 1)[:, :2]):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            p = plan._replace(prefix_lens=ints(prefix))
            say(f"past the table {prefix}")
            sched = M.get_mla_metadata(p.prefix_lens.clamp(max=128), 48, 1)
            got = M.flash_mla_with_kvcache(q, cache, t, None, 512, *sched, tree=p, status=status)
            torch.cuda.synchronize()
            seen = [[{j for j in line if max(n, 0) + j < 128} for line in row] for n, row in zip(prefix, mask)]
            cut = p._replace(prefix_lens=ints([min(max(n, 0), 128) for n in prefix]))
            check_decode(q, cache, rows, table, cut, seen, "bf16", got, f"past the table {prefix}")
            assert status.item() == raised


def test_bad_page_ids_stay_in_the_cache(gpu):
    """Ids outside the cache are read as its nearest page, as the decode reads them."""
    q, cache, rows, table, plan, mask = problem("bf16", 4, 9, [60, 61], 27, extra=0)
    bad = table.clone()
    bad[0, 1], bad[1, 1] = -7, 2 ** 31 - 1
    near = table.clone()
    near[0, 1], near[1, 1] = 0, cache.shape[0] - 1
    say("bad page ids")
    got = decode(q, cache, bad, plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, near, plan, mask, "bf16", got, "bad page ids")


@pytest.mark.parametrize("fmt", ["bf16", "f16", "fp8", "fp4"])
def test_hidden_tokens_may_hold_anything(gpu, fmt):
    """Infinities and NaNs in a drafted token's row reach the rows that see it, and no bit of the others."""
    s = 9
    q, cache, rows, table, plan, mask = problem(fmt, 16, s, [60, 10], 29, drop=0.0)
    say(f"hidden {fmt}")
    clean = decode(q, cache, table, plan)
    slots = plan.slots.cpu()
    spoilt = [(0, 3), (0, 7), (1, s - 1)]
    for n, (b, j) in enumerate(spoilt):
        page, row = divmod(int(slots[b, j]), 64)
        if fmt == "fp4":
            cache.scale[page, row, 2 + n] = 255
        elif fmt == "fp8":
            cache.latent[page, row, 100 * n + 5] = 0x7F
        else:
            cache[page, row, 0, 100 * n + 5] = (INF, NAN, -INF)[n]
    got = decode(q, cache, table, plan)
    torch.cuda.synchronize()
    for b in range(2):
        for i in range(s):
            if any(x == b and j in mask[b][i] for x, j in spoilt):
                assert torch.isnan(got[0][b, i]).all() and (got[1][b, :, i] == -INF).all(), (b, i)
            else:
                assert torch.equal(got[0][b, i], clean[0][b, i]) and torch.equal(got[1][b, :, i], clean[1][b, :, i]), (b, i)
    # the rope part: a NaN score
    if fmt == "bf16":
        page, row = divmod(int(slots[0, 5]), 64)
        cache[page, row, 0, 512] = NAN
        again = decode(q, cache, table, plan)
        torch.cuda.synchronize()
        for i in range(s):
            if 5 in mask[0][i]:
                assert torch.isnan(again[0][0, i]).all()
            else:
                assert torch.equal(again[0][0, i].isnan(), got[0][0, i].isnan())


def test_extreme_values(gpu):
    """Large queries (one key takes all the weight) and zero ones, tiny and large latents."""
    for scale_q, scale_k in ((1000.0, 1.0), (0.0, 1.0), (1.0, 2.0 ** -100), (2.0 ** -60, 2.0 ** 60)):
        q, cache, rows, table, plan, mask = problem("bf16", 8, 6, [70, 3], 31)
        q, cache, rows = q * scale_q, cache * scale_k, rows * scale_k
        say(f"extreme {scale_q} {scale_k}")
        got = decode(q, cache, table, plan)
        torch.cuda.synchronize()
        ro, rl, size, reach = T.attend(q.double().cpu(), rows, table.cpu(), plan.prefix_lens.tolist(), mask, SCALE)
        to, tl = bounds(q, ro, rl, size, reach, 80, q.dtype, "bf16", 48)
        assert ((got[0].double().cpu() - ro).abs() <= to).all() and ((got[1].double().cpu() - rl).abs() <= tl).all()


def test_strided_queries_and_outputs(gpu):
    q, cache, rows, table, plan, mask = problem("fp8", 16, 5, [100, 7], 37)
    wide = torch.zeros(5, 2, 20, 640, dtype=q.dtype, device="cuda")
    view = wide.permute(1, 0, 2, 3)[:, :, 2:18, 8:584]
    view.copy_(q)
    out = torch.full((2, 16, 5, 520), 7.0, dtype=q.dtype, device="cuda")
    say("strided")
    sched = M.get_mla_metadata(plan.prefix_lens, 80, 1)
    o = out[..., :512].transpose(1, 2)
    got = M.flash_mla_with_kvcache(view, cache, torch.cat([table, table], 1)[:, :table.shape[1]], None, 512, *sched, tree=plan, out=o)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, "fp8", got, "strided")
    assert (out[..., 512:] == 7.0).all()


@pytest.mark.parametrize("fmt,H,s", [("bf16", 16, 4), ("fp4", 16, 4), ("fp8", 128, 2), ("bf16", 2, 3)])
def test_absorbed(gpu, fmt, H, s):
    """The value projection of the merged rows, rounded to 16 bits, as of the decode's own output."""
    q, cache, rows, table, plan, mask = problem(fmt, H, s, [300, 64, 0], 41)
    g = torch.Generator().manual_seed(5)
    w = (torch.randn(H, 512, 128, generator=g) * 512 ** -0.5).to(q.dtype).cuda()
    say(f"absorbed {fmt} H={H} s={s}")
    sched = M.get_mla_metadata(plan.prefix_lens, s * H, 1, kv_cache=cache)
    out, lse = M.flash_mla_with_kvcache(q, cache, table, None, 512, *sched, tree=plan)
    v, lse2 = M.mla_decode_absorbed(q, cache, table, None, *sched, M.prepare_w_uv(w), tree=plan)
    torch.cuda.synchronize()
    want = (out.double().transpose(1, 2).transpose(0, 1).reshape(H, -1, 512) @ w.double()).view(H, 3, s, 128).permute(1, 2, 0, 3)
    size = (out.double().abs().transpose(1, 2).transpose(0, 1).reshape(H, -1, 512) @ w.double().abs()).view(H, 3, s, 128).permute(1, 2, 0, 3)
    # the merged row may be summed in another order (half a step of 16 bits where it rounds apart: 2^-8 of each product
    # at most), the fp32 products 512 of them, v's own rounding
    assert ((v.double() - want).abs() <= (2.0 ** -7 + 2.0 ** -14) * size + 2.0 ** -8 * want.abs()).all()
    assert torch.equal(lse, lse2)


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_many_pages_by_themselves(gpu, fmt):
    """Pages in one launch, more of them than the merge holds at once (a schedule of more parts makes the room)."""
    q, cache, rows, table, plan, mask = problem(fmt, 8, 2, [64 * 700 + 3], 53)
    sched = M.get_mla_metadata(plan.prefix_lens, 16, 1, num_parts=1000, fixed_overhead=0)
    code = 1 if fmt == "fp8" else 0
    assert M._lib.load().mla_tree_takes_pages(1, 2, 8, 1000, code, table.shape[1])
    say(f"many pages {fmt}")
    got = M.flash_mla_with_kvcache(q, cache, table, None, 512, *sched, tree=plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, fmt, got, f"many pages {fmt}")


@pytest.mark.parametrize("width", [0, 900])
def test_absorbed_of_many_splits(gpu, width):
    """Merges past 64 splits, from pages by themselves and from the schedule's: whole rows first, then the projection."""
    H, s = 2, 4
    q, cache, rows, table, plan, mask = problem("bf16", H, s, [64 * 200 + 9], 59)
    if width:
        table = table.repeat(1, -(-width // table.shape[1]))[:, :width]
    g = torch.Generator().manual_seed(7)
    w = (torch.randn(H, 512, 128, generator=g) * 512 ** -0.5).to(q.dtype).cuda()
    sched = M.get_mla_metadata(plan.prefix_lens, s * H, 1, num_parts=256, fixed_overhead=0)
    assert bool(M._lib.load().mla_tree_takes_pages(1, s, H, 256, 0, table.shape[1])) == (not width)
    say(f"absorbed of many splits, width {width}")
    out, lse = M.flash_mla_with_kvcache(q, cache, table, None, 512, *sched, tree=plan)
    v, lse2 = M.mla_decode_absorbed(q, cache, table, None, *sched, M.prepare_w_uv(w), tree=plan)
    torch.cuda.synchronize()
    check_decode(q, cache, rows, table, plan, mask, "bf16", (out, lse), f"absorbed, width {width}")
    rows_ = out.double().transpose(1, 2).transpose(0, 1).reshape(H, -1, 512)
    want = (rows_ @ w.double()).view(H, 1, s, 128).permute(1, 2, 0, 3)
    size = (rows_.abs() @ w.double().abs()).view(H, 1, s, 128).permute(1, 2, 0, 3)
    # as in test_absorbed
    assert ((v.double() - want).abs() <= (2.0 ** -7 + 2.0 ** -14) * size + 2.0 ** -8 * want.abs()).all()
    assert torch.equal(lse, lse2)


def test_tiny_latents(gpu):
    """One key in sight and latents near the smallest normal number: the output is the key's latent, rounded twice (the
    partial to 2^-11 of its chunk's largest, at worst as subnormals of 16 bits)."""
    q, cache, rows, table, plan, _ = problem("bf16", 4, 3, [0, 0], 61)
    plan = plan._replace(mask=ints([[1, 2, 4]] * 2, torch.int64))
    for e in (-100, -113, -118):
        tiny = (cache.float().clamp(-4, 4) * 2.0 ** e).bfloat16()
        say(f"tiny 2^{e}")
        out, _ = decode(q, tiny, table, plan)
        torch.cuda.synchronize()
        for b in range(2):
            for i in range(3):
                page, row = divmod(int(plan.slots[b, i]) if int(plan.slots[b, i]) >= 0 else int(table[b, 0]) * 64 + i, 64)
                want = tiny[page, row, 0, :512].double()
                got = out[b, i].double()
                assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * want.abs().max()).all()


def test_decode_refusals(gpu):
    q, cache, rows, table, plan, mask = problem("bf16", 4, 5, [10, 20], 43)
    say("decode refusals")
    sched = M.get_mla_metadata(plan.prefix_lens, 20, 1)
    idx = torch.zeros(2, 1, 4, dtype=torch.int32, device="cuda")
    for t, kw in [(plan._replace(mask=plan.mask[:, :4]), {}), (plan._replace(mask=plan.mask.int()), {}), (plan._replace(mask=plan.mask.cpu()), {}),
                  (plan._replace(prefix_lens=plan.prefix_lens.long()), {}), (plan._replace(prefix_lens=plan.prefix_lens[:1]), {}), (plan, dict(indices=idx))]:
        with pytest.raises(ValueError):
            M.flash_mla_with_kvcache(q, cache, table, None, 512, *sched, tree=t, **kw)
    with pytest.raises(ValueError):
        M.flash_mla_with_kvcache(q, cache, None, None, 512, *sched, tree=plan)
    big = torch.zeros(1, 65, 1, 576, dtype=q.dtype, device="cuda")
    with pytest.raises(ValueError):
        M.flash_mla_with_kvcache(big, cache, table[:1], None, 512, *sched, tree=plan)


def test_other_streams_and_graphs(gpu):
    """Two captured steps that share the stream's workspace, replayed in turns with eager work between them."""
    q, cache, rows, table, plan, mask = problem("bf16", 16, 6, [200, 5, 77], 47)
    q2 = q.flip(0).contiguous()
    lens = plan.prefix_lens + 6
    parents = ints([[-1, 0, 0, 1, 2, 2]] * 3)
    tok = ints([[1, 2, 3, 4, 5, 6]] * 3)
    side = torch.cuda.Stream()
    say("graphs")

    def step(x):
        p = M.tree_plan(parents, lens, table)
        out, lse = M.mla_decode_with_kvcache(x, cache, table, None, tree=p)
        a = M.tree_accept(p, tok, tok.roll(-1, 1))
        return [out, lse, *p, *a]

    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        want = [[t.clone() for t in step(x)] for x in (q, q2)]
        side.synchronize()
        graphs = []
        for x in (q, q2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                res = step(x)
            graphs.append((gr, res))
        for _ in range(3):
            for (gr, res), w in zip(graphs, want):
                for t in res:
                    t.fill_(3)
                gr.replay()
                side.synchronize()
                for t, u in zip(res, w):
                    assert torch.equal(t, u)
            again = step(q)
            side.synchronize()
            assert all(torch.equal(t, u) for t, u in zip(again, want[0]))


@pytest.mark.parametrize("width", [0, 600])
def test_two_streams_at_once(gpu, width):
    """Decodes of different problems queued on two streams without a wait between them: each its own workspace, whether
    pages go by themselves or the schedule is followed."""
    jobs = []
    for seed, (H, s) in ((67, (16, 6)), (71, (32, 9))):
        q, cache, rows, table, plan, mask = problem("bf16", H, s, [300, 64, 5, 0], seed)
        if width:
            table = table.repeat(1, -(-width // table.shape[1]))[:, :width]
        jobs.append((q, cache, table, plan))
    want = [[t.clone() for t in M.mla_decode_with_kvcache(q, c, t, None, tree=p)] for q, c, t, p in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    say(f"two streams, width {width}")
    for _ in range(20):
        for st, (q, c, t, p), res in zip(streams, jobs, got):
            with torch.cuda.stream(st):
                res.append(M.mla_decode_with_kvcache(q, c, t, None, tree=p))
    torch.cuda.synchronize()
    for res, w in zip(got, want):
        assert all(torch.equal(x, y) for r in res for x, y in zip(r, w))


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_whole_step(gpu, fmt):
    """Reserve, plan, append, decode, accept, keep, release: afterwards the cache holds the prefix and the kept tokens, in
    order, and their decode as a chain gives what the tree gave."""
    B, H, s = 3, 16, 7
    nb = 12
    start = [130, 61, 0]
    g = torch.Generator().manual_seed(53)
    pool, table = M.page_pool(nb), torch.zeros(B, 4, dtype=torch.int32, device="cuda")
    lens = ints([0] * B)
    cache = {"fp4": M.fp4_kv_cache, "fp8": M.fp8_kv_cache}[fmt](nb) if fmt != "bf16" else torch.zeros(nb, 64, 1, 576, dtype=torch.bfloat16, device="cuda")
    rope = M.rope_plan(64, scaling="yarn", factor=40.0)
    say(f"whole step {fmt}")
    r = M.reserve_pages(pool, table, lens, ints(start), sum(start))
    M.kv_append_slots(torch.randn(sum(start), 576, generator=g).to(torch.bfloat16).cuda(), cache, r.slots, r.positions, rope)
    parents = ints([[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 1, 2, 3, 4, 5], [-1, 0, 0, 0, 3, 3, 5]])
    tokens = ints([[9, 1, 2, 3, 4, 5, 6]] * B)
    targets = ints([[2, 0, 5, 0, 0, 6, 8], [1, 2, 7, 0, 0, 0, 0], [3, 0, 0, 5, 0, 0, 0]])
    kept = [[0, 2, 5, 6], [0, 1, 2], [0, 3, 5]]
    M.reserve_pages(pool, table, lens, ints([s] * B), B * s)
    plan = M.tree_plan(parents, lens, table)
    new = torch.randn(B * s, 576, generator=g).to(torch.bfloat16).cuda()
    q_pe, q = torch.randn(B * s, H, 64, generator=g).to(torch.bfloat16).cuda(), torch.randn(B * s, H, 576, generator=g).to(torch.bfloat16).cuda()
    M.kv_append_slots(new, cache, plan.slots.view(-1), plan.positions.view(-1), rope, q_pe, q)
    out, lse = M.mla_decode_with_kvcache(q.view(B, s, H, 576), cache, table, None, tree=plan)
    a = M.tree_accept(plan, tokens, targets)
    M.kv_keep_path(cache, plan.slots, a.path)
    free = pool.count.clone()
    M.release_pages(pool, table, lens, a.keep_lens)
    torch.cuda.synchronize()
    assert a.counts.tolist() == [4, 3, 3] and [[i for i in p if i >= 0] for p in a.path.tolist()] == kept
    assert a.next_tokens.tolist() == [8, 7, 0] and lens.tolist() == [134, 64, 3]
    assert (pool.count - free).tolist() == [0 + 1 + 0]  # sequence 1 gives back the page that tokens 64 .. 67 took
    rows = M.kv_gather(cache, torch.arange(nb * 64, dtype=torch.int32, device="cuda")).double().cpu().view(nb, 64, 576)
    for b, path in enumerate(kept):
        n = len(path)
        qc = q.view(B, s, H, 576)[b:b + 1, path].contiguous()
        o2, l2 = M.mla_decode_with_kvcache(qc, cache, table[b:b + 1], lens[b:b + 1])
        chain = [[set(range(i + 1)) for i in range(n)]]
        ro, rl, size, reach = T.attend(qc.double().cpu(), rows, table[b:b + 1].cpu(), [start[b]], chain, SCALE)
        if fmt == "fp4":
            mag = qc.double().cpu()[..., :512].unflatten(-1, (16, 32)).abs().amax(-1, keepdim=True).expand(1, n, H, 16, 32).flatten(-2)
            reach = T.attend(torch.cat([mag, qc.double().cpu()[..., 512:].abs()], -1), rows.abs(), table[b:b + 1].cpu(), [start[b]], chain, SCALE)[3]
        to, tl = bounds(qc, ro, rl, size, reach, 140, q.dtype, fmt, s * H)
        for o, l in ((o2, l2), (out[b:b + 1, path], lse[b:b + 1, :, path])):
            assert ((o.double().cpu() - ro).abs() <= to).all() and ((l.double().cpu() - rl).abs() <= tl).all(), (fmt, b)
