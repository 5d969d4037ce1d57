"""GPU tests of the serving step at its edges: rows without a position, bit for bit; appends by slot at both ends of bf16; pools
and tables that hold ids of no page."""
import pytest
import torch

import mlc_decode_amd as M
from oracle import mla_fp4_ref as F4
from oracle import mla_fp8_ref as F8
from test_gpu_fp4 import varied_cache
from test_gpu_serving import Model, assert_state, device_state, make_cache, say, state

pytestmark = pytest.mark.gpu

BITS = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}


def any_bits(shape, dtype, seed):
    """Every kind of value: random bit patterns, among them infinities, NaNs with payloads, zeros of both signs."""
    g = torch.Generator().manual_seed(seed)
    lo, hi = (-2 ** 15, 2 ** 15) if dtype != torch.float32 else (-2 ** 31, 2 ** 31)
    x = torch.randint(lo, hi, shape, generator=g, dtype=torch.int64).to(BITS[dtype]).view(dtype)
    flat = x.view(-1)
    flat[::7], flat[1::11], flat[3::13] = -0.0, float("inf"), float("nan")
    return x


def bits(x):
    return x.contiguous().view(BITS[x.dtype])


# 16-byte chunks and single values, with and without dims beside the rotated ones
@pytest.mark.parametrize("D,rot,first", [(64, 64, 0), (128, 64, 32), (71, 8, 1), (96, 64, 16)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_without_a_position_stay_as_they_were(gpu, D, rot, first, layout, dtype):
    T, H = 1100, 3
    x = any_bits((T, H, D), dtype, D + rot)
    pos = torch.arange(T, dtype=torch.int32) * 3
    pos[::2] = -1 - pos[::2]
    rope = M.rope_plan(rot, layout=layout, scaling="yarn", factor=8.0)
    say(f"no position D={D} rot={rot} first={first} {layout} {dtype}")
    xd, pd = x.cuda(), pos.cuda()
    out = M.apply_rope(xd, pd, rope, first=first)
    assert torch.equal(bits(out[::2]).cpu(), bits(x[::2]))
    finite = torch.where(torch.isfinite(x.float()) & (x.float().abs() < 1e4), x, torch.ones_like(x)).cuda()
    alone = M.apply_rope(finite[1::2].contiguous(), pd[1::2].contiguous(), rope, first=first)
    beside = M.apply_rope(finite, pd, rope, first=first)
    assert torch.equal(bits(beside[1::2]), bits(alone))  # the rows beside them are rotated as ever
    M.apply_rope(xd, pd, rope, first=first, out=xd)
    torch.cuda.synchronize()
    assert torch.equal(bits(xd), bits(out))


@pytest.mark.parametrize("kind", ["bf16", "f16", "pair", "fp8", "fp4"])
@pytest.mark.parametrize("layout", ["interleaved", "half", None])
def test_append_without_a_position_stores_what_it_got(gpu, kind, layout):
    """A negative position, and no rope at all: the rope dims of tokens and queries bit for bit."""
    T, H, nb = 300, 2, 6
    dt = torch.float16 if kind == "f16" else torch.bfloat16
    g = torch.Generator().manual_seed(4)
    cache, _ = make_cache(kind, nb, 1)
    new = torch.randn(T, 576, generator=g).to(dt)
    new[:, 512:] = any_bits((T, 64), dt, 9)
    slots = torch.randperm(nb * 64, generator=g)[:T].to(torch.int32)
    pos = torch.full((T,), -1, dtype=torch.int32)
    say(f"append without a position {kind} {layout}")
    if layout is None:
        M.kv_append_slots(new.cuda(), cache, slots.cuda())
    else:
        pe = any_bits((T, H, 64), dt, 10)
        q = torch.zeros(T, H, 576, dtype=dt, device="cuda")
        M.kv_append_slots(new.cuda(), cache, slots.cuda(), pos.cuda(), M.rope_plan(layout=layout, scaling="yarn", factor=8.0), pe.cuda(), q)
        assert torch.equal(bits(q[..., 512:]).cpu(), bits(pe)) and not q[..., :512].any()
    rows = M.kv_gather(cache, slots.cuda())
    torch.cuda.synchronize()
    assert torch.equal(bits(rows[:, 512:]).cpu(), bits(new[:, 512:]))


@pytest.mark.parametrize("kind", ["fp8", "fp4"])
@pytest.mark.parametrize("n", [1, 7, 64])
def test_append_by_slot_at_the_ends_of_bf16(gpu, kind, n):
    """Zeros, subnormals, the largest values, infinities and NaNs: as kv_append and the format's oracle have them."""
    B = 5
    new = varied_cache(B, 3).reshape(B, 64, 576)[:, :n].contiguous()
    if n > 8:
        new[1, :, :128] *= 2.0 ** -120
        new[1, 0, :512], new[1, 1, :512], new[1, 2, :512] = 0.0, -0.0, 2.0 ** -133
        new[2, 0, 128:256], new[2, 1, :128], new[2, 2, 256:384] = 3.3895313892515355e38, -2.5e38, 2.0 ** 127
        new[3, 5, 300], new[3, 6, 10] = float("-inf"), float("nan")
        new[3, 7, :512] = float("nan")
    make = {"fp8": M.fp8_kv_cache, "fp4": M.fp4_kv_cache}[kind]
    a, b = make(B), make(B)
    table = torch.arange(B, dtype=torch.int32, device="cuda").reshape(B, 1)
    slots = (table * 64 + torch.arange(n, dtype=torch.int32, device="cuda")).reshape(-1)
    say(f"append by slot, ends {kind} n={n}")
    M.kv_append(new.cuda(), a, table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    M.kv_append_slots(new.reshape(-1, 576).cuda(), b, slots)
    torch.cuda.synchronize()
    for x, y, what in zip(a, b, ("codes", "scales", "rope")):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), what
    if kind == "fp4":
        codes, byte = F4.quantize_latent(new.reshape(-1, 576)[:, :512])
        assert torch.equal(b.latent[:, :n].cpu().reshape(-1, 256), torch.from_numpy(codes)) and torch.equal(b.scale[:, :n].cpu().reshape(-1, 16), torch.from_numpy(byte))
    else:
        fin = torch.isfinite(new.float()).all(-1)
        codes, scale = F8.quantize_latent(new[fin][:, :512])
        got = b.scale[:, :, :n].transpose(1, 2)[fin.cuda()].cpu()
        assert torch.equal(b.latent[:, :n][fin.cuda()].cpu(), torch.from_numpy(codes)) and torch.equal(got, torch.from_numpy(scale))


# ---------------------------------------------------------------------------------------
# ids that name no page
# ---------------------------------------------------------------------------------------
class Pool(Model):
    """The model with what a release may put back: pages of the pool."""

    def release(self, keep):
        count = min(max(self.count, 0), self.nb)
        back = []
        for b, k in enumerate(keep):
            k, L = max(k, 0), self.lens[b]
            if L > k:
                back += [p for p in self.table[b][-(-k // 64):min(-(-L // 64), len(self.table[b]))] if 0 <= p < self.nb]
                self.lens[b] = k
        for i, p in enumerate(reversed(back)):
            self.free[count + i] = p
        self.count = count + len(back)


def foreign(m, rows, seed):
    """Ids of no page into the tables of some sequences; the pages they stood for are nobody's now."""
    g = torch.Generator().manual_seed(seed)
    ids = [-1, m.nb, 2 ** 31 - 1, -2 ** 31, m.nb + 7]
    for b in rows:
        held = -(-max(m.lens[b], 0) // 64)
        for c in range(held):
            if torch.rand(1, generator=g).item() < 0.4:
                m.table[b][c] = ids[(b + c) % len(ids)]
    return m


@pytest.mark.parametrize("B,hi,P", [(1, 300, 6), (7, 700, 12), (64, 500, 9), (1000, 500, 9), (1030, 200, 5), (2500, 100, 3), (40, 64 * 40, 41)])
def test_release_gives_back_pages_of_the_pool_only(gpu, B, hi, P):
    m, g = state(B, B, P, hi, 10)
    m = foreign(Pool(m.free, m.count, m.table, m.lens, m.nb), range(0, B, 3), B)
    if B > 5:
        m.lens[2] = 64 * P + 1000  # longer than its row: what the row holds comes back
        m.table[2] = [-1] * P
    pool, table, lens = device_state(m)
    say(f"release foreign B={B}")
    for keep in ([max(0, n // 2) for n in m.lens], [0] * B):
        M.release_pages(pool, table, lens, torch.tensor(keep, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        m.release(keep)
        assert_state(pool, table, lens, m, f"release foreign B={B}")
    assert all(0 <= p < m.nb for p in m.free[:m.count])


@pytest.mark.parametrize("count", [-5, 0])
def test_release_into_an_empty_pool(gpu, count):
    """A count below zero holds no page, for a release as for a reservation."""
    m, _ = state(3, 6, 8, 400, 0)
    m = Pool(m.free, count, m.table, m.lens, m.nb)
    pool, table, lens = device_state(m)
    say(f"release count={count}")
    M.release_pages(pool, table, lens, torch.zeros_like(lens))
    torch.cuda.synchronize()
    m.release([0] * 6)
    assert_state(pool, table, lens, m, f"count={count}")
    assert m.count == m.nb and sorted(m.free) == list(range(m.nb))


@pytest.mark.parametrize("new", [1, 300])
def test_a_popped_id_of_no_page_names_no_row(gpu, new):
    """A stack that its user filled with such ids: the rows on them have slot -1, never another page's slot."""
    B, nb = 40, 500
    free = torch.arange(nb, dtype=torch.int32)
    bad = torch.tensor([-1, nb, 2 ** 26 + 3, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)  # 2^26 pages are 2^32 rows
    free[1::2] = bad[torch.arange(nb // 2) % 5]
    pool = M.PagePool(free.cuda(), torch.tensor([nb], dtype=torch.int32, device="cuda"))
    table, lens = torch.zeros(B, 8, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    say(f"bad stack new={new}")
    r = M.reserve_pages(pool, table, lens, torch.full_like(lens, new), B * new)
    torch.cuda.synchronize()
    assert r.granted.all()
    page = table.cpu().long().repeat_interleave(new, 0).gather(1, (r.positions.cpu().long() // 64)[:, None])[:, 0]
    ok = (page >= 0) & (page < nb)
    want = torch.where(ok, page * 64 + r.positions.cpu().long() % 64, torch.full_like(page, -1))
    assert not ok.all() and torch.equal(r.slots.cpu().long(), want)


def test_the_longest_slot_map(gpu):
    """2^31 - 1 rows: the last workgroup's row numbers pass 2^31."""
    T = 2 ** 31 - 1
    pool, table = M.page_pool(9), torch.zeros(3, 3, dtype=torch.int32, device="cuda")
    lens, new = torch.tensor([0, 70, 5], dtype=torch.int32, device="cuda"), torch.tensor([100, 0, 3], dtype=torch.int32, device="cuda")
    say("longest map")
    r = M.reserve_pages(pool, table, lens, new, T)
    torch.cuda.synchronize()
    assert r.cu_new.tolist() == [0, 100, 100, 103] and r.granted.tolist() == [1, 1, 1] and lens.tolist() == [100, 70, 8]
    assert r.positions[:104].tolist() == [*range(100), 5, 6, 7, -1] and r.slots[:101].tolist() == [*range(100), 5]
    for m in (r.slots, r.positions):
        assert m.shape == (T,) and (m[-(1 << 20):] == -1).all() and (m[1 << 30:(1 << 30) + 1000] == -1).all()


def test_outputs_whose_rows_share_memory_are_refused(gpu):
    """Strides that are wide enough each, but not together."""
    x, pos, rope = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), M.rope_plan()
    buf = torch.zeros(8192, dtype=torch.bfloat16, device="cuda")
    for strides in ((64, 64, 1), (64, 128, 1), (128, 64 + 32, 1)):
        with pytest.raises(ValueError, match="rows overlap"):
            M.apply_rope(x, pos, rope, out=buf.as_strided((3, 2, 64), strides))
    M.apply_rope(x, pos, rope, out=buf.as_strided((3, 2, 64), (64, 256, 1)))  # heads apart, tokens close
    new, cache = torch.zeros(3, 576, dtype=torch.bfloat16, device="cuda"), M.fp4_kv_cache(1)
    with pytest.raises(ValueError, match="q's rows overlap"):
        M.kv_append_slots(new, cache, pos, pos, rope, x, buf.as_strided((3, 2, 576), (576, 576, 1)))
