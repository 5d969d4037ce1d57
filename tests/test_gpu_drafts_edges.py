"""GPU tests of the tree decode in every one of its forms: what cache rows hold that a query row does not see reaches no bit of
it, whether the rows are drafted tokens or lie behind the last one; weights keep more bits than the cache's type has; and the
documented step."""
import os
import re

import pytest
import torch

import mlc_decode_amd as M
from oracle import mla_tree_ref as T
from test_gpu_drafts import INF, NAN, SCALE, ints, problem, say

pytestmark = pytest.mark.gpu

# (heads, drafted tokens, columns of the table, 64 rows a workgroup): pages by themselves, and the schedule's pass before
# the drafted tokens, which are one tile of 32 or 64 keys there
FORMS = [(16, 9, 0, False), (64, 9, 0, True), (16, 9, 600, False), (128, 14, 600, True), (16, 40, 600, False), (48, 40, 600, True)]


def spoil(cache, fmt, slot, n):
    """An infinity or a NaN in a cached token, of the n-th kind of its format."""
    page, row = divmod(slot, 64)
    if fmt == "fp4":
        cache.scale[page, row, (5 * n) % 16] = 255
    elif fmt == "fp8" and n % 2:
        cache.scale[page, n % 4, row] = (INF, NAN)[n // 2 % 2]
        cache.latent[page, row, 128 * (n % 4):128 * (n % 4) + 128] = 0x38  # 1.0: a NaN times a zero would do as well
    elif fmt == "fp8":
        cache.latent[page, row, (97 * n) % 512] = 0x7F
    else:
        cache[page, row, 0, (97 * n + 5) % 512] = (INF, NAN, -INF)[n % 3]
        if n % 4 == 1:
            cache[page, row, 0, 512:] = NAN


@pytest.mark.parametrize("fmt", ["bf16", "f16", "fp8", "fp4"])
@pytest.mark.parametrize("H,s,width,rows64", FORMS)
def test_hidden_tokens_in_every_form(gpu, fmt, H, s, width, rows64):
    """Of prefixes that end inside a page, with it, and of none; the tokens behind the last one are spoilt too."""
    prefixes = [60, 0, 64]
    q, cache, rows, table, plan, mask = problem(fmt, H, s, prefixes, 100 + H + s, drop=0.1)
    B = len(prefixes)
    slot = lambda b, t: int(pages[b][t // 64]) * 64 + t % 64  # noqa: E731
    pages = table.tolist()
    wide = table.repeat(1, -(-width // table.shape[1]))[:, :width] if width else table
    sched = M.get_mla_metadata(plan.prefix_lens, H * s, 1, kv_cache=cache)
    code = {"fp8": 1, "fp4": 4}.get(fmt, 0)
    lone = M._lib.load().mla_tree_takes_pages(B, s, H, sched[0].shape[0], code, wide.shape[1])
    assert bool(lone) == (not width)
    tiles = -(-H * s // 16) * B * (1 + wide.shape[1] if lone else 1)
    assert (4 * tiles > 5 * 256) == rows64
    say(f"hidden {fmt} H={H} s={s} columns {wide.shape[1]}")
    run = lambda: M.flash_mla_with_kvcache(q, cache, wide, None, 512, *sched, tree=plan)  # noqa: E731
    clean = [t.clone() for t in run()]
    for b, p in enumerate(prefixes):  # what is behind the trees
        for t in range(p + s, 64 * table.shape[1]):
            spoil(cache, fmt, slot(b, t), t)
    got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, clean)), "rows behind the trees"
    spoilt = [(0, 3), (0, s - 1), (1, 1), (1, s // 2), (2, s - 2), (0, 33 % s), (2, 2)]
    for n, (b, j) in enumerate(spoilt):
        spoil(cache, fmt, slot(b, prefixes[b] + j), n)
    got = run()
    torch.cuda.synchronize()
    seen = torch.tensor([[any(x == b and j in mask[b][i] for x, j in spoilt) for i in range(s)] for b in range(B)], device="cuda")
    assert seen.any() and not seen.all()
    assert torch.isnan(got[0][seen]).all() and (got[1].transpose(1, 2)[seen] == -INF).all()
    assert torch.equal(got[0][~seen], clean[0][~seen]) and torch.equal(got[1].transpose(1, 2)[~seen], clean[1].transpose(1, 2)[~seen])


@pytest.mark.parametrize("width", [0, 600])
def test_dropped_nodes_still_see_the_prefix(gpu, width):
    """A node that is none has no drafted token in sight, itself neither: its row is the prefix's attention, and empty only
    where there is no prefix."""
    q, cache, rows, table, plan, _ = problem("bf16", 16, 5, [70, 0], 5)
    plan = M.tree_plan(ints([[-1, 0, -2, 2, 9]] * 2), ints([75, 5]), table)
    wide = table.repeat(1, -(-width // table.shape[1]))[:, :width] if width else table
    say(f"dropped nodes, columns {wide.shape[1]}")
    out, lse = M.mla_decode_with_kvcache(q, cache, wide, None, tree=plan)
    alone, alse = M.mla_decode_with_kvcache(q, cache, wide, None, tree=plan._replace(mask=torch.zeros_like(plan.mask)))
    torch.cuda.synchronize()
    none = plan.mask == 0
    assert none.tolist() == [[False, False, True, True, True]] * 2 and torch.equal(none, plan.positions == -1)
    assert torch.equal(out[none], alone[none]) and torch.equal(lse.transpose(1, 2)[none], alse.transpose(1, 2)[none])
    assert torch.isfinite(lse[0]).all() and (out[0].abs().amax(-1) > 0).all()
    assert (out[1, 2:] == 0).all() and (lse[1, :, 2:] == -INF).all() and torch.isfinite(lse[1, :, :2]).all()


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
def test_documented_step_when_pages_run_out(gpu, fmt):
    """The step that the README shows, as it stands there: requests that got no pages (one longer than its tree, one empty)
    and one with nothing to verify keep every cached row, their length and their pages; the others, trees of their own
    sizes, go on."""
    readme = open(os.path.join(os.path.dirname(__file__), "..", "README.md")).read()
    code, = [c for c in re.findall(r"```python\n(.*?)```", readme, re.S) if "tree_plan" in c]
    B, s, H, D, nb = 5, 6, 16, 64, 7
    start, each = [62, 200, 0, 40, 64], [6, 6, 6, 3, 0]  # pages 1, 4, 0, 1, 1: all; sequences 0 and 2 want one that is not there
    g = torch.Generator().manual_seed(3)
    rand = lambda *shape: torch.randn(*shape, generator=g).bfloat16().cuda()  # noqa: E731
    cache = {"fp4": M.fp4_kv_cache, "fp8": M.fp8_kv_cache}[fmt](nb) if fmt != "bf16" else torch.zeros(nb, 64, 1, 576, dtype=torch.bfloat16, device="cuda")
    pool, table, lens = M.page_pool(nb), torch.zeros(B, 6, dtype=torch.int32, device="cuda"), ints([0] * B)
    rope = M.rope_plan(64)
    r = M.reserve_pages(pool, table, lens, ints(start), sum(start))
    assert r.granted.tolist() == [1] * B and pool.count.item() == 0
    M.kv_append_slots(rand(sum(start), 576), cache, r.slots, r.positions, rope)
    every = torch.arange(nb * 64, dtype=torch.int32, device="cuda")
    before = M.kv_gather(cache, every).clone()
    names = dict(M=M, torch=torch, pool=pool, table=table, lens=lens, cache=cache, rope=rope, B=B, s=s, H=H, s_each=ints(each),
                 parents=ints([[-1, 0, 0, 1, 2, 2]] * B), tokens=ints([[9, 1, 2, 3, 4, 5]] * B), targets=ints([[2, 0, 5, 0, 0, 7]] * B),
                 w_o_matrix=rand(D, H * 128), w_norm=rand(D), x=rand(B * s, D), h=rand(B * s, D), kv_new=rand(B * s, 576), q_pe=rand(B * s, H, 64),
                 q=rand(B * s, H, 576), w_uv=M.prepare_w_uv(rand(H, 512, 128)))
    say(f"documented step {fmt}")
    exec(code, names)
    torch.cuda.synchronize()
    a = names["a"]
    counts = [0, 3, 0, 2, 0]
    assert a.counts.tolist() == counts and a.next_tokens.tolist() == [-1, 7, -1, 5, -1]
    assert lens.tolist() == [p + c for p, c in zip(start, counts)] and pool.count.item() == 0
    after = M.kv_gather(cache, every)
    rows = table.tolist()
    for b in range(B):
        at = [rows[b][t // 64] * 64 + t % 64 for t in range(start[b])]
        assert torch.equal(after[at].view(torch.int16), before[at].view(torch.int16)), f"sequence {b}"


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("H,s,width,rows64", FORMS)
def test_weights_keep_their_bits(gpu, fmt, H, s, width, rows64):
    """Softmax weights are held past 16 bits.  Queries have one dim that is not zero, a power of two, so that scores have one
    product each: off by their scaling, the fast exponential and its argument, 2^-20 (1 + |score|) together, as is the sum of
    the weights.  Two 16-bit halves hold a weight to 2^-16.  Then the partials' rounding, 2^-11 of each, and the output's,
    2^-8.  (Of the schedule's form the drafted tokens alone are looked at, without a prefix.)"""
    prefixes = [0, 0, 0] if width else [10, 60, 70]
    q, cache, rows, table, plan, mask = problem(fmt, H, s, prefixes, 300 + H + s, drop=0.1)
    q = torch.zeros_like(q)
    q[..., 512] = 64.0
    wide = table.repeat(1, -(-width // table.shape[1]))[:, :width] if width else table
    sched = M.get_mla_metadata(plan.prefix_lens, H * s, 1, kv_cache=cache)
    code = {"fp8": 1, "fp4": 4}.get(fmt, 0)
    lone = M._lib.load().mla_tree_takes_pages(3, s, H, sched[0].shape[0], code, wide.shape[1])
    assert bool(lone) == (not width)
    say(f"weights {fmt} H={H} s={s} columns {wide.shape[1]}")
    out, _ = M.flash_mla_with_kvcache(q, cache, wide, None, 512, *sched, tree=plan)
    torch.cuda.synchronize()
    ro, rl, size, reach = T.attend(q.double().cpu(), rows, table.cpu(), plan.prefix_lens.tolist(), mask, SCALE)
    d = 2.0 ** -20 * (1 + reach + rl.abs().nan_to_num(0, 0, 0)).transpose(1, 2)[..., None]
    tol = (2.0 ** -16 + torch.expm1(2 * d) + 2.0 ** -11) * size * (1 + 2.0 ** -8) + 2.0 ** -8 * ro.abs() + 2.0 ** -24
    off = ((out.double().cpu() - ro).abs() / tol).max().item()
    say(f"  {off:.3f} of the bound")
    assert off <= 1
