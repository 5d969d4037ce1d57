"""GPU tests of the serving step around the decode: rotary positions against complex arithmetic in 64 bits, appends and
gathers by slot against the formats' oracles, page bookkeeping against a plain integer model, and a run of all
of them together, eager and captured."""
import math
import sys

import numpy as np
import pytest
import torch

import mlc_decode_amd as M
from oracle import mla_fp4_ref as F4
from oracle import mla_fp8_ref as F8

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def say(msg):
    print(f"[gpu-serving] {msg}", flush=True)
    sys.stdout.flush()


def rotated(x, positions, rope, first):
    """x [T, H, D] in 64 bits rotated, and the bound of the kernel's error without the final rounding: sine and cosine
    are off by 2^-21 at most (the reduced turn's rounding to fp32, 2^-25 turns, times 2 pi, and two steps of
    the functions), each product and sum by 2^-24 of its size."""
    y = x.double().clone()
    freqs, n = rope.freqs.cpu(), rope.freqs.numel()
    turns = positions.double()[:, None] * freqs
    z = torch.polar(torch.ones_like(turns), (turns - turns.round()) * 2 * math.pi)[:, None] * rope.amp
    v = y[..., first:first + 2 * n]
    a, b = (v[..., 0::2], v[..., 1::2]) if rope.layout == "interleaved" else (v[..., :n], v[..., n:])
    w = torch.complex(a.clone(), b.clone()) * z
    tol = torch.zeros_like(y)
    size = (a.abs() + b.abs()) * abs(rope.amp) * (2.0 ** -21 + 3 * 2.0 ** -24)
    on = (positions >= 0)[:, None, None]
    for dst, val in ((y, (w.real, w.imag)), (tol, (size, size))):
        d = dst[..., first:first + 2 * n]
        old = d.clone()
        if rope.layout == "interleaved":
            d[..., 0::2], d[..., 1::2] = val
        else:
            d[..., :n], d[..., n:] = val
        d.copy_(torch.where(on, d, old))
    return y, tol


def assert_rotated(got, x, positions, rope, first, what):
    y, tol = rotated(x, positions, rope, first)
    half = HALF_STEP[x.dtype]
    tol = tol * (1 + half) + torch.where(tol > 0, half * y.abs(), torch.zeros_like(y))
    if x.dtype == torch.float16:
        tol = torch.where(tol > 0, tol + 2.0 ** -25, tol)  # half a step of the subnormals
    err = (got.double().cpu() - y).abs()
    assert (err <= tol).all(), f"{what}: off by {err.max():.3e} at {np.unravel_index(int((err - tol).argmax()), err.shape)}"


# T, H, D, rotated dims, first, layout, dtype, scaling
ROPE_CASES = [
    (1, 1, 64, 64, 0, "interleaved", torch.bfloat16, None),
    (128, 16, 64, 64, 0, "interleaved", torch.bfloat16, "yarn"),
    (5, 128, 576, 64, 512, "interleaved", torch.bfloat16, "yarn"),
    (33, 3, 128, 64, 0, "half", torch.float16, "linear"),
    (33, 3, 128, 128, 0, "half", torch.float32, "ntk"),
    (7, 5, 96, 64, 16, "half", torch.bfloat16, None),
    (7, 5, 71, 8, 1, "interleaved", torch.bfloat16, None),      # nothing falls on 16 bytes
    (9, 2, 67, 6, 61, "half", torch.float16, None),
    (3, 2, 20, 4, 4, "half", torch.float32, "linear"),
    (2, 2, 2, 2, 0, "interleaved", torch.float32, None),
    (3, 1, 1024, 1024, 0, "half", torch.bfloat16, None),
    (2, 1, 1030, 1022, 8, "interleaved", torch.bfloat16, None),
    (4097, 2, 64, 64, 0, "half", torch.bfloat16, "yarn"),
    (8195, 3, 96, 64, 16, "half", torch.bfloat16, None),        # eight tokens a workgroup, chunks beside the rotated ones
    (8195, 3, 96, 64, 16, "interleaved", torch.float32, "ntk"),
    (8195, 2, 71, 8, 1, "half", torch.float16, None),           # and one value at a time
]


@pytest.mark.parametrize("T,H,D,rot,first,layout,dtype,scaling", ROPE_CASES)
def test_rope(gpu, T, H, D, rot, first, layout, dtype, scaling):
    g = torch.Generator().manual_seed(T * 7 + D)
    x = torch.randn(T, H, D, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, dtype=torch.int32)
    pos[0] = 0 if T > 1 else 163839
    if T > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -1
    rope = M.rope_plan(rot, layout=layout, scaling=scaling, factor=8.0 if scaling else 1.0, base=10000.0)
    say(f"rope T={T} H={H} D={D} rot={rot} first={first} {layout} {dtype}")
    xd, pd = x.cuda(), pos.cuda()
    got = M.apply_rope(xd, pd, rope, first=first)
    torch.cuda.synchronize()
    assert_rotated(got, x, pos, rope, first, "rope")
    rest = torch.ones(D, dtype=torch.bool)
    rest[first:first + rot] = False
    assert torch.equal(got[..., rest].cpu(), x[..., rest])
    same = M.apply_rope(xd, pd, rope, first=first, out=xd)  # in place: the same values
    torch.cuda.synchronize()
    assert same is xd and torch.equal(xd, got)


def test_rope_views_batches_and_default_place(gpu):
    """A projection's part into the decode's query buffer; leading dims; both parts of one row."""
    g = torch.Generator().manual_seed(3)
    B, s, H = 3, 2, 10
    w = torch.randn(B, s, H, 192, generator=g).to(torch.bfloat16)
    q = torch.full((B, s, H, 576), 5.0, dtype=torch.bfloat16, device="cuda")
    pos = torch.randint(0, 100000, (B, s), generator=g, dtype=torch.int32)
    rope = M.rope_plan(scaling="yarn", factor=40.0, mscale_all_dim=1.0)
    wd = w.cuda()
    say("rope views")
    out = M.apply_rope(wd[..., 128:], pos.cuda(), rope, out=q[..., 512:])
    last = M.apply_rope(wd, pos.cuda(), rope)  # the last 64 dims by default
    torch.cuda.synchronize()
    assert out.data_ptr() == q[..., 512:].data_ptr() and (q[..., :512] == 5.0).all()
    x = w[..., 128:].reshape(B * s, H, 64)
    assert_rotated(q[..., 512:].reshape(B * s, H, 64), x, pos.reshape(-1), rope, 0, "into q")
    assert torch.equal(last[..., :128], wd[..., :128]) and torch.equal(last[..., 128:], q[..., 512:])
    wide = torch.randn(4, 5, 160, device="cuda").to(torch.bfloat16)
    before = wide.clone()
    p4 = torch.arange(4, dtype=torch.int32, device="cuda")
    M.apply_rope(wide[..., :64], p4, rope, out=wide[..., 64:128])
    torch.cuda.synchronize()
    assert torch.equal(wide[..., :64], before[..., :64]) and torch.equal(wide[..., 128:], before[..., 128:])
    assert torch.equal(wide[..., 64:128], M.apply_rope(before[..., :64], p4, rope))
    assert M.apply_rope(wide[:0], p4[:0], rope).shape == (0, 5, 160)


def test_rope_python_refusals(gpu):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    rope = M.rope_plan()
    bad = [
        (lambda: M.apply_rope(x.double(), pos, rope), "bfloat16"),
        (lambda: M.apply_rope(x[0], pos[0], rope), "H, D"),
        (lambda: M.apply_rope(x, pos[:3], rope), "shape"),
        (lambda: M.apply_rope(x, pos.long(), rope), "int32"),
        (lambda: M.apply_rope(x, torch.zeros(8, dtype=torch.int32, device="cuda")[::2], rope), "contiguous"),
        (lambda: M.apply_rope(x, pos.cpu(), rope), "GPU"),
        (lambda: M.apply_rope(x[..., ::2], pos, M.rope_plan(32)), "unit stride"),
        (lambda: M.apply_rope(x, pos, rope, first=1), "rotated dims"),
        (lambda: M.apply_rope(x, pos, M.rope_plan(128)), "rotated dims"),
        (lambda: M.apply_rope(x, pos, rope, out=x.float()), "dtype"),
        (lambda: M.apply_rope(x, pos, rope, out=torch.zeros(1, 2, 64, dtype=x.dtype, device="cuda").expand(4, 2, 64)), "overlap"),
        (lambda: M.apply_rope(x, pos, rope._replace(layout="odd")), "layout"),
        (lambda: M.apply_rope(x, pos, rope._replace(amp=math.nan)), "amp"),
        (lambda: M.apply_rope(x, pos, rope._replace(freqs=rope.freqs.float())), "float64"),
    ]
    buf = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device="cuda")
    bad.append((lambda: M.apply_rope(buf[:4], pos, rope, out=buf[1:]), "overlaps"))
    for call, needle in bad:
        with pytest.raises(ValueError, match=needle):
            call()


# ---------------------------------------------------------------------------------------
# append and gather by slot
# ---------------------------------------------------------------------------------------
def make_cache(kind, nb, seed):
    """A filled cache of a kind, and its values in 64 bits [nb * 64, 576]."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn(nb, 64, 1, 576, generator=g)
    if kind in ("bf16", "f16", "pair"):
        kv = kv.to(torch.float16 if kind == "f16" else torch.bfloat16)
        d = kv.cuda()
        return ((d[..., :512].contiguous(), d[..., 512:].contiguous()) if kind == "pair" else d), kv.double().reshape(-1, 576)
    kv = kv.to(torch.bfloat16)
    if kind == "fp8":
        lat, sc, rope = F8.quantize_pages(kv)
        return M.Fp8KVCache(torch.from_numpy(lat).cuda(), torch.from_numpy(sc).cuda(), rope.cuda()), F8.dequantize_pages(lat, sc, rope).double().reshape(-1, 576)
    c, b, rope = F4.quantize_pages(kv)
    return M.Fp4KVCache(torch.from_numpy(c).cuda(), torch.from_numpy(b).cuda(), rope.cuda()), F4.dequantize_pages(c, b, rope).reshape(-1, 576)


def stored_latent(kind, lat):
    """What the cache holds of latents [n, 512], in 64 bits."""
    if kind == "fp4":
        return torch.from_numpy(F4.dequantize_latent(*F4.quantize_latent(lat)))
    if kind == "fp8":
        return torch.from_numpy(F8.dequantize_latent(*F8.quantize_latent(lat))).double()
    return lat.double()


def every_slot(nb):
    return torch.arange(nb * 64, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["bf16", "f16", "pair", "fp8", "fp4"])
@pytest.mark.parametrize("T,H,layout", [(1, 1, "interleaved"), (128, 16, "interleaved"), (131, 3, "half"), (2100, 8, "half"), (9000, 2, "interleaved")])
def test_append_slots(gpu, kind, T, H, layout):
    g = torch.Generator().manual_seed(T + H)
    nb = -(-T // 64) + 3
    cache, want = make_cache(kind, nb, T)
    dt = torch.float16 if kind == "f16" else torch.bfloat16
    new = (torch.randn(T, 576, generator=g) * torch.exp2(torch.randint(-8, 8, (T, 1), generator=g).float())).to(dt)
    slots = torch.randperm(nb * 64, generator=g)[:T].to(torch.int32)
    pos = torch.randint(0, 200000, (T,), generator=g, dtype=torch.int32)
    if T > 4:
        slots[2], slots[3] = -1, nb * 64
        pos[4] = -1  # written, unrotated
    w = torch.randn(T, H, 192, generator=g).to(dt).cuda()
    q = torch.full((T, H, 576), 7.0, dtype=dt, device="cuda")
    rope = M.rope_plan(layout=layout, scaling="yarn", factor=8.0)
    say(f"append slots {kind} T={T} H={H} {layout}")
    M.kv_append_slots(new.cuda(), cache, slots.cuda(), pos.cuda(), rope, w[..., 128:], q)
    rows = M.kv_gather(cache, every_slot(nb))
    torch.cuda.synchronize()
    on = (slots >= 0) & (slots < nb * 64)
    got, hit = rows.double().cpu(), torch.zeros(nb * 64, dtype=torch.bool)
    hit[slots[on].long()] = True
    assert torch.equal(got[~hit], want[~hit])
    assert torch.equal(got[slots[on].long()][:, :512], stored_latent(kind, new[on][:, :512]))
    assert_rotated(rows[slots[on].long().cuda()][:, None, 512:], new[on][:, None, 512:], pos[on], rope, 0, "k rope")
    assert (q[..., :512] == 7.0).all() and (q[~on.cuda()] == 7.0).all()
    assert_rotated(q[on.cuda()][..., 512:], w[on.cuda()][..., 128:].cpu(), pos[on], rope, 0, "q rope")


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
def test_append_slots_without_rope_is_the_append(gpu, kind):
    """As kv_append writes them, bit for bit, for strided rows too."""
    g = torch.Generator().manual_seed(9)
    a, _ = make_cache(kind, 6, 1)
    b, _ = make_cache(kind, 6, 1)
    wide = torch.randn(2, 40, 600, generator=g).to(torch.bfloat16).cuda()
    new = wide[..., 8:584]
    table = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([60, 100], dtype=torch.int32, device="cuda")
    pos = lens.long()[:, None] + torch.arange(40, device="cuda")
    slots = (torch.gather(table.long(), 1, pos // 64) * 64 + pos % 64).to(torch.int32).reshape(-1)
    say(f"append slots without rope {kind}")
    M.kv_append(new, a, table, lens)
    for i in range(2):
        M.kv_append_slots(new[i], b, slots[40 * i:40 * i + 40])
    torch.cuda.synchronize()
    for x, y in zip(*((c,) if isinstance(c, torch.Tensor) else c for c in (a, b))):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_append_slots_rotates_queries_in_place(gpu):
    g = torch.Generator().manual_seed(2)
    cache, _ = make_cache("fp4", 2, 0)
    q = torch.randn(5, 4, 576, generator=g).to(torch.bfloat16).cuda()
    before = q.clone()
    rope, pos = M.rope_plan(), torch.tensor([5, 6, 7, 8, 9], dtype=torch.int32, device="cuda")
    M.kv_append_slots(torch.zeros(5, 576, dtype=torch.bfloat16, device="cuda"), cache, torch.tensor([0, 1, -1, 3, 4], dtype=torch.int32, device="cuda"),
                      pos, rope, q[..., 512:], q)
    torch.cuda.synchronize()
    want = M.apply_rope(before, pos, rope)
    want[2] = before[2]
    assert torch.equal(q, want)


@pytest.mark.parametrize("kind", ["bf16", "f16", "pair", "fp8", "fp4"])
@pytest.mark.parametrize("T", [0, 1, 3, 1000])
def test_gather(gpu, kind, T):
    g = torch.Generator().manual_seed(T)
    nb = 7
    cache, want = make_cache(kind, nb, 5)
    slots = torch.randint(-3, nb * 64 + 3, (T,), generator=g, dtype=torch.int32)
    say(f"gather {kind} T={T}")
    wide = torch.full((max(T, 1), 600), 3.0, dtype=torch.float16 if kind == "f16" else torch.bfloat16, device="cuda")
    out = M.kv_gather(cache, slots.cuda(), out=wide[:T, 8:584])
    torch.cuda.synchronize()
    ok = (slots >= 0) & (slots < nb * 64)
    assert torch.equal(out.double().cpu(), torch.where(ok[:, None], want[slots.clamp(0, nb * 64 - 1).long()], torch.zeros(1, dtype=torch.float64)))
    assert (wide[:, :8] == 3.0).all() and (wide[:, 584:] == 3.0).all()


def test_gather_keeps_nan_blocks(gpu):
    cache = M.fp4_kv_cache(1)
    cache.scale[0, 5, 3] = 255
    rows = M.kv_gather(cache, torch.tensor([5, 6], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.isnan(rows[0, 96:128]).all() and int(torch.isnan(rows).sum()) == 32


def test_slot_python_refusals(gpu):
    cache, _ = make_cache("bf16", 2, 0)
    f4 = M.fp4_kv_cache(2)
    new = torch.zeros(4, 576, dtype=torch.bfloat16, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    rope, q = M.rope_plan(), torch.zeros(4, 2, 576, dtype=torch.bfloat16, device="cuda")
    pe = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call, needle in [
        (lambda: M.kv_append_slots(new.half(), cache, i), "dtype"), (lambda: M.kv_append_slots(new.half(), f4, i), "dtype"),
        (lambda: M.kv_append_slots(new[:, :575], cache, i), "576"), (lambda: M.kv_append_slots(new, cache, i[:3]), "slots"),
        (lambda: M.kv_append_slots(new, cache, i.long()), "slots"), (lambda: M.kv_append_slots(new, cache, i, None, rope), "positions"),
        (lambda: M.kv_append_slots(new, cache, i, i, M.rope_plan(32)), "64 dims"), (lambda: M.kv_append_slots(new, cache, i, i, rope, pe), "together"),
        (lambda: M.kv_append_slots(new, cache, i, i, None, pe, q), "rope"), (lambda: M.kv_append_slots(new, cache, i, i, rope, pe[:, :, :32], q), "q_pe"),
        (lambda: M.kv_append_slots(new, cache, i, i, rope, pe, q[..., :512]), "q must"), (lambda: M.kv_append_slots(new, cache, i, i, rope, pe, q[:1].expand(4, 2, 576)), "overlap"),
        (lambda: M.kv_append_slots(new, cache, i, i, rope, q[..., 508:572], q), "overlap"),
        (lambda: M.kv_append_slots(new, cache[..., :512], i), "576"), (lambda: M.kv_gather(cache.float(), i), "bfloat16"),
        (lambda: M.kv_gather(f4._replace(scale=f4.scale[:, :, :8]), i), "fp4 scale"), (lambda: M.kv_gather(f4._replace(latent=f4.latent.int()), i), "fp4 latent"),
        (lambda: M.kv_gather(f4, i, out=new[:3]), "out must"), (lambda: M.kv_gather(f4, i.reshape(2, 2)), "1-D"),
        (lambda: M.mla_decode_with_kvcache(torch.zeros(1, 1, 4, 576, dtype=torch.float16, device="cuda"), f4, i.reshape(1, 4), i[:1]), "bf16"),
    ]:
        with pytest.raises(ValueError, match=needle):
            call()


# ---------------------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------------------
class Model:
    """The pool, tables and lengths in plain integers."""

    def __init__(self, free, count, table, lens, nb):
        self.free, self.count, self.table, self.lens, self.nb = list(free), count, [list(r) for r in table], list(lens), nb

    def reserve(self, new, T):
        slots, positions, granted, cu, at = [-1] * T, [-1] * T, [], [0], self.count
        asked, used, count, P = 0, 0, self.count, len(self.table[0])
        for b, n in enumerate(new):
            n, L, start = max(n, 0), self.lens[b], cu[-1]
            cu.append(start + n)
            ok = L >= 0 and L + n <= 64 * P and start + n <= T
            if ok and n and L % 64 and not 0 <= self.table[b][L // 64] < self.nb:
                ok = False
            need = -(-(L + n) // 64) - -(-L // 64) if ok else 0
            asked += need
            ok = ok and (need == 0 or asked <= count)
            granted.append(int(ok))
            if not ok:
                continue
            for i in range(need):
                self.table[b][-(-L // 64) + i] = self.free[count - 1 - (asked - need + i)]
            used += need
            for t in range(n):
                p = L + t
                slots[start + t], positions[start + t] = self.table[b][p // 64] * 64 + p % 64, p
            self.lens[b] = L + n
        self.count = count - used
        return slots, positions, cu, granted

    def release(self, keep):
        back = []
        for b, k in enumerate(keep):
            k, L = max(k, 0), self.lens[b]
            if L > k:
                back += self.table[b][-(-k // 64):min(-(-L // 64), len(self.table[b]))]
                self.lens[b] = k
        for i, p in enumerate(reversed(back)):
            self.free[self.count + i] = p
        self.count += len(back)


def state(seed, B, P, hi, spare):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, hi + 1, (B,), generator=g)
    held = [-(-int(n) // 64) for n in lens]
    nb = sum(held) + spare
    order = torch.randperm(nb, generator=g).tolist()
    table = torch.full((B, P), -5, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    free = order[at:] + [-9] * at
    return Model(free, spare, table.tolist(), lens.tolist(), nb), g


def device_state(m):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return M.PagePool(i32(m.free), i32([m.count])), i32(m.table), i32(m.lens)


def assert_state(pool, table, lens, m, what):
    assert lens.tolist() == m.lens, f"{what}: lengths"
    assert pool.count.item() == m.count, f"{what}: count"
    assert table.tolist() == m.table, f"{what}: table"
    assert pool.free_pages.tolist() == m.free, f"{what}: stack"


@pytest.mark.parametrize("B,hi,new,spare,pad", [
    (1, 0, 1, 4, 0), (1, 200, 300, 3, 5), (3, 130, 70, 8, 0), (64, 500, 1, 64, 0), (64, 500, 1, 5, 0), (64, 64, 64, 40, 9),
    (1023, 300, 2, 500, 3), (1024, 300, 2, 5000, 0), (1025, 300, 3, 5000, 0), (2500, 100, 9, 900, 77), (40, 3000, 2500, 2000, 11),
])
def test_reserve_and_release(gpu, B, hi, new, spare, pad):
    """Both launch forms (few rows: one launch), requests that do not fit, and the way back."""
    P = -(-(hi + new) // 64)
    m, g = state(B + new, B, P, hi, spare)
    ask = torch.randint(-1 if B > 3 else new, new + 1, (B,), generator=g)
    if B > 8:
        m.lens[5] = -3              # no sequence
        m.lens[6] = 64 * P          # full
    pool, table, lens = device_state(m)
    old_lens, old_free, old_count = list(m.lens), list(m.free), m.count
    T = int(ask.clamp(min=0).sum()) + pad
    say(f"reserve B={B} T={T} spare={spare}")
    r = M.reserve_pages(pool, table, lens, ask.to(torch.int32).cuda(), T)
    torch.cuda.synchronize()
    slots, positions, cu, granted = m.reserve(ask.tolist(), T)
    assert r.cu_new.tolist() == cu and r.granted.tolist() == granted
    assert r.slots.tolist() == slots and r.positions.tolist() == positions
    assert_state(pool, table, lens, m, "reserve")
    live = [s for s in slots if s >= 0]
    assert len(set(live)) == len(live)
    # a too small row buffer: whole requests are refused
    short = T // 2
    r = M.reserve_pages(pool, table, lens, ask.to(torch.int32).cuda(), short)
    slots, positions, cu, granted = m.reserve(ask.tolist(), short)
    assert r.slots.tolist() == slots and r.positions.tolist() == positions and r.granted.tolist() == granted and r.cu_new.tolist() == cu
    assert_state(pool, table, lens, m, "second reserve")
    half = [max(0, (n + a) // 2) for n, a in zip(m.lens, old_lens)]
    for keep in (half, old_lens):
        M.release_pages(pool, table, lens, torch.tensor(keep, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        m.release(keep)
        assert_state(pool, table, lens, m, "release")
    assert m.count == old_count and sorted(m.free[:m.count]) == sorted(old_free[:old_count])


def test_release_restores_the_stack(gpu):
    m, g = state(8, 100, 12, 500, 300)
    pool, table, lens = device_state(m)
    keep, free, count = lens.clone(), pool.free_pages.clone(), pool.count.clone()
    ask = torch.randint(0, 200, (100,), generator=g, dtype=torch.int32).cuda()
    say("release restores")
    for _ in range(3):
        M.reserve_pages(pool, table, lens, ask, int(ask.sum()))
        M.release_pages(pool, table, lens, keep)
    torch.cuda.synchronize()
    assert torch.equal(pool.free_pages, free) and torch.equal(pool.count, count) and torch.equal(lens, keep)
    M.release_pages(pool, table, lens, torch.zeros_like(lens))  # every request done: all pages are free again
    torch.cuda.synchronize()
    assert pool.count.item() == m.nb and sorted(pool.free_pages.tolist()) == list(range(m.nb)) and not lens.any()


def test_reserve_bad_tail_page_and_strided_table(gpu):
    m, _ = state(4, 4, 4, 0, 10)
    m.lens = [10, 10, 0, 64]
    m.table[0][0], m.table[1][0], m.table[3][0] = 3, m.nb, 2
    pool, _, lens = device_state(m)
    wide = torch.full((4, 9), 77, dtype=torch.int32, device="cuda")
    table = wide[:, 2:6]
    table.copy_(torch.tensor(m.table, dtype=torch.int32))
    ask = torch.tensor([5, 5, 100, 1], dtype=torch.int32, device="cuda")
    say("reserve bad tail page")
    r = M.reserve_pages(pool, table, lens, ask, 120)
    torch.cuda.synchronize()
    slots, positions, cu, granted = m.reserve(ask.tolist(), 120)
    assert granted == [1, 0, 1, 1]
    assert r.slots.tolist() == slots and r.positions.tolist() == positions and r.granted.tolist() == granted
    assert_state(pool, table, lens, m, "bad tail")
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()


def test_pool_python_refusals(gpu):
    pool = M.page_pool(4)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for call, needle in [
        (lambda: M.reserve_pages(pool, i(2, 3).long(), i(2), i(2), 4), "block_table"), (lambda: M.reserve_pages(pool, i(2, 6)[:, ::2], i(2), i(2), 4), "block_table"),
        (lambda: M.reserve_pages(pool, i(2, 3), i(3), i(2), 4), "cache_seqlens"), (lambda: M.reserve_pages(pool, i(2, 3), i(2), i(3), 4), "new_lens"),
        (lambda: M.reserve_pages(pool, i(2, 3), i(2), i(2), -1), "num_tokens"), (lambda: M.reserve_pages(pool._replace(count=i(2)), i(2, 3), i(2), i(2), 4), "count"),
        (lambda: M.release_pages(pool, i(2, 3), i(2), i(4)[::2]), "keep_lens"), (lambda: M.reserve_pages(pool, i(1, 3).expand(2, 3), i(2), i(2), 4), "overlap"),
    ]:
        with pytest.raises(ValueError, match=needle):
            call()


# ---------------------------------------------------------------------------------------
# all together
# ---------------------------------------------------------------------------------------
def attend(q, k, n):
    s = q.double() @ k[:n].double().T * 576 ** -0.5
    return torch.softmax(s, -1) @ k[:n, :512].double(), torch.logsumexp(s, -1)


def serve(kind, steps=3, capture=False):
    """A ragged prefill, then decode steps of one token; returns per step (out, lse), and what they should be."""
    B, H, P, nb = 5, 16, 6, 24
    g = torch.Generator().manual_seed(17)
    cache = {"bf16": lambda: torch.zeros(nb, 64, 1, 576, dtype=torch.bfloat16, device="cuda"), "fp8": lambda: M.fp8_kv_cache(nb), "fp4": lambda: M.fp4_kv_cache(nb)}[kind]()
    pool, table, lens = M.page_pool(nb), torch.zeros(B, P, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    rope = M.rope_plan(scaling="yarn", factor=8.0)
    ask = torch.tensor([1, 64, 130, 0, 200], dtype=torch.int32)
    T = int(ask.sum()) + 5
    new = torch.randn(T, 576, generator=g).to(torch.bfloat16)
    r = M.reserve_pages(pool, table, lens, ask.cuda(), T)
    M.kv_append_slots(new.cuda(), cache, r.slots, r.positions, rope)
    torch.cuda.synchronize()
    seqs = [new[a:a + n] for a, n in zip(r.cu_new.tolist(), ask.tolist())]
    got, want = [], []
    kv = torch.empty(B, 576, dtype=torch.bfloat16, device="cuda")
    pe, q = torch.empty(B, H, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, H, 576, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(B, dtype=torch.int32, device="cuda")

    def step():
        s = M.reserve_pages(pool, table, lens, one, B)
        M.kv_append_slots(kv, cache, s.slots, s.positions, rope, pe, q)
        sched = M.get_mla_metadata(lens, H, 1, kv_cache=cache)
        return M.flash_mla_with_kvcache(q.unsqueeze(1), cache, table, lens, 512, *sched)

    graph, held = None, None
    if capture:
        keep = lens.clone()
        step()  # eager once: workspace; then its token is taken back
        M.release_pages(pool, table, lens, keep)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        torch.cuda.synchronize()
    for _ in range(steps):
        n, p, l = torch.randn(B, 576, generator=g).to(torch.bfloat16), torch.randn(B, H, 64, generator=g).to(torch.bfloat16), torch.randn(B, H, 512, generator=g).to(torch.bfloat16)
        kv.copy_(n), pe.copy_(p), q[..., :512].copy_(l)
        if graph is None:
            out, lse = step()
        else:
            graph.replay()
            out, lse = held
            torch.zeros(1000, device="cuda").add_(1)  # other work between the replays
        torch.cuda.synchronize()
        got.append((out[:, 0].double().cpu(), lse[..., 0].double().cpu()))
        res = []
        for b in range(B):
            seqs[b] = torch.cat([seqs[b], n[b:b + 1]])
            L = seqs[b].shape[0]
            pos = torch.arange(L, dtype=torch.int32)
            kr, _ = rotated(seqs[b][:, None, 512:], pos, rope, 0)
            keys = torch.cat([stored_latent(kind, seqs[b][:, :512]), kr[:, 0].to(torch.bfloat16).double()], -1)
            qr, _ = rotated(p[b][None], pos[-1:], rope, 0)
            res.append(attend(torch.cat([l[b].double(), qr[0].to(torch.bfloat16).double()], -1), keys, L))
        want.append(res)
    return got, want


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
def test_serving_step_makes_its_device_current(gpu, kind, monkeypatch):
    """Every launch of a step happens with the tensors' device current, where another one was."""
    from mlc_decode_amd import api
    inside, streams, stream_of = [], [], api._stream_ptr

    class Guard(torch.cuda.device):
        def __enter__(self):
            inside.append(self.idx)
            super().__enter__()

        def __exit__(self, *exc):
            inside.pop()
            return super().__exit__(*exc)

    def stream_ptr(device):  # a launch asks for its stream inside the guard, the workspace outside
        streams.append(list(inside))
        return stream_of(device)

    say(f"device {kind}")
    want, _ = serve(kind, steps=1)
    monkeypatch.setattr(api, "_current_device", lambda: 1)  # another than the tensors'
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(api, "_stream_ptr", stream_ptr)
    got, _ = serve(kind, steps=1)
    assert streams.count([0]) == 6  # two reservations, two appends, schedule, decode
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1], want[0][1])


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("capture", [False, True])
def test_serving_steps(gpu, kind, capture):
    """Reserve, rotate and append, schedule, decode.  The decode's bar (1e-2, lse 1e-3); a rope value that the kernel
    rounds to the other neighbour adds at most 2^-7 |k| |q| / 24 of one product to a logit, far below it."""
    say(f"serving steps {kind} capture={capture}")
    got, want = serve(kind, capture=capture)
    for i, ((out, lse), res) in enumerate(zip(got, want)):
        for b, (o, l) in enumerate(res):
            assert (out[b] - o).abs().max() <= 1e-2 * max(1.0, o.abs().max().item()), f"step {i} seq {b}"
            assert (lse[b] - l).abs().max() <= 1e-3 + 2e-3, f"step {i} seq {b}: lse"
