"""GPU tests of the operators around the attention, against plain implementations in 64 bits."""
import sys

import pytest
import torch

import mlc_decode_amd as M

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def say(msg):
    print(f"[gpu-layer] {msg}", flush=True)
    sys.stdout.flush()


def values8(rows):
    """The values of 8-bit rows, in 64 bits."""
    v = rows.codes.view(torch.float8_e4m3fn).double()
    return v * torch.exp2(rows.scale.double() - 127).repeat_interleave(32, -1)


# ---------------------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------------------
def exact_norm(x, w, eps, residual=None):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()


def norm_slack(dim):
    """Relative error of y in fp32 ahead of its rounding: h (half a step), its square's sum (at most dim + 2 roundings, all
    terms positive; the root halves them), the mean, the root and the quotient (a step each), two products."""
    return (dim / 2 + 10) * 2.0 ** -24


def check_norm(x, w, eps=1e-6, residual=None, got=None, what=""):
    h, y = exact_norm(x, w, eps, residual)
    gy, gh = got if residual is not None else (got, None)
    e = EPS[x.dtype]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -134  # half of the type's smallest step
    assert gy.dtype == x.dtype and gy.shape == x.shape
    off = (gy.double() - y).abs() - (e * (1 + 2 * norm_slack(x.shape[-1])) + norm_slack(x.shape[-1])) * y.abs() - tiny
    assert (off <= 0).all(), f"{what}: {off.max().item()}"
    if gh is not None:
        check_sum(h, gh, what)


def check_sum(h, gh, what):
    """h: added in fp32, rounded once."""
    e, tiny = EPS[gh.dtype], 2.0 ** -25 if gh.dtype == torch.float16 else 2.0 ** -134
    off = (gh.double() - h).abs() - (e + 2.0 ** -23) * h.abs() - tiny
    assert (off <= 0).all(), f"{what}: h {off.max().item()}"


def tensors(T, D, dtype, pitch, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, pitch, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-6, 7, (T, 1), generator=g).float())
    return x.to(dtype).cuda()[:, pitch - D:], (torch.randn(T, D, generator=g) * 3).to(dtype).cuda(), (1 + 0.2 * torch.randn(D, generator=g))


DIMS = [1, 2, 7, 8, 31, 32, 64, 96, 500, 512, 513, 576, 1000, 1024, 1536, 2048, 2056, 4096, 4104, 7168, 8192, 8200, 9001, 16384, 16392, 20000, 32768, 40000]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", DIMS)
def test_norm(gpu, D, dt):
    dtype = DT[dt]
    for T, pitch in ((1, D), (5, D), (3, D + 5), (2, D + 64)):
        x, r, w = tensors(T, D, dtype, pitch, D + T)
        for wt in {dtype, torch.float32}:
            say(f"norm D={D} {dt} T={T} pitch={pitch} weight {wt}")
            ww = w.to(wt).cuda()
            a = M.rms_norm(x, ww)
            b = M.rms_norm(x, ww, 1e-3, residual=r)
            torch.cuda.synchronize()
            check_norm(x, ww, 1e-6, None, a, "plain")
            check_norm(x, ww, 1e-3, r, b, "residual")


@pytest.mark.parametrize("T", [64, 511, 513, 2000, 5000])
def test_norm_many_rows(gpu, T):
    """Above and below the rows where workgroups of one size and the other are taken; the latent part of wider rows."""
    for D, pitch in ((7168, 7168), (512, 576), (1536, 1536)):
        x, r, w = tensors(T, D, torch.bfloat16, pitch, T)
        say(f"norm T={T} D={D}")
        ww = w.to(torch.bfloat16).cuda()
        got = M.rms_norm(x, ww, residual=r)
        torch.cuda.synchronize()
        check_norm(x, ww, 1e-6, r, got, f"T={T}")


def check_norm8(x, w, eps, residual, got, what):
    """y in 8 bits: within half a step of e4m3 (2^-4, and of its smallest step) at its own scale, and that scale the
    smallest that holds the block: of y's largest, up to the error that y has in fp32."""
    _, y = exact_norm(x, w, eps, residual)
    rows = got if residual is None else got[0]
    D = x.shape[-1]
    assert rows.codes.dtype == torch.uint8 and rows.codes.shape == x.shape and rows.scale.shape == (*x.shape[:-1], D // 32)
    two = torch.exp2(rows.scale.double() - 127).repeat_interleave(32, -1)
    v = values8(rows)
    s = norm_slack(D)
    off = (v - y).abs() - (2.0 ** -4 + 2 * s) * y.abs() - 2.0 ** -10 * two
    assert (off <= 0).all(), f"{what}: {off.max().item()}"
    amax = y.unflatten(-1, (-1, 32)).abs().amax(-1)
    two = two[..., ::32]
    assert (amax <= 448 * two * (1 + 2 * s)).all() and ((amax >= 224 * two * (1 - 2 * s)) | (rows.scale == 1) | (amax == 0)).all(), what
    assert (rows.scale[amax == 0] == 127).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [3, 16, 25, 36, 64, 65, 72, 128, 130, 160, 256, 264])
def test_norm_of_short_rows(gpu, D, dt):
    """Several rows a wave, the last wave with fewer; heads of a token, rows out of wider ones; a row of NaN beside others."""
    for T, pitch in ((7, D), (33, D), (129, D + 5), (1000, D + 64)):
        x, r, w = tensors(T, D, DT[dt], pitch, D + T)
        ww = w.to(DT[dt]).cuda()
        say(f"norm of short rows D={D} {dt} T={T} pitch={pitch}")
        a, b = M.rms_norm(x, ww), M.rms_norm(x, ww, 1e-3, residual=r)
        torch.cuda.synchronize()
        check_norm(x, ww, 1e-6, None, a, "plain")
        check_norm(x, ww, 1e-3, r, b, "residual")
        if D % 32 == 0:
            c, d = M.rms_norm(x, ww, quantize=True), M.rms_norm(x, ww, residual=r, quantize=True)
            torch.cuda.synchronize()
            check_norm8(x, ww, 1e-6, None, c, "plain")
            check_norm8(x, ww, 1e-6, r, d, "residual")
            check_sum(exact_norm(x, ww, 1e-6, r)[0], d[1], "residual")
        spoilt = x.clone()
        spoilt[5, D // 2] = float("nan")
        e, f = M.rms_norm(spoilt, ww), M.rms_norm(x.clone(), ww)  # in one layout: the order of a row's sum is the layout's
        torch.cuda.synchronize()
        assert e[5].isnan().all() and torch.equal(e[:5], f[:5]) and torch.equal(e[6:], f[6:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [32, 64, 96, 512, 544, 1536, 2048, 2080, 4096, 7168, 8192, 8224, 16384, 20000 // 32 * 32, 40000])
def test_norm_8bit(gpu, D, dt):
    for T, pitch in ((1, D), (6, D), (3, D + 5)):
        x, r, w = tensors(T, D, DT[dt], pitch, D + T)
        g = torch.Generator().manual_seed(1)
        w = w * torch.exp2(torch.randint(-20, 20, (D // 32,), generator=g).float()).repeat_interleave(32)
        w[:32] = 0
        ww = w.cuda()
        say(f"norm 8 bit D={D} {dt} T={T}")
        a, b = M.rms_norm(x, ww, quantize=True), M.rms_norm(x, ww, residual=r, quantize=True)
        torch.cuda.synchronize()
        check_norm8(x, ww, 1e-6, None, a, "plain")
        check_norm8(x, ww, 1e-6, r, b, "residual")
        check_sum(exact_norm(x, ww, 1e-6, r)[0], b[1], "residual")


def test_norm_8bit_rounds_to_nearest_even(gpu):
    """Every midpoint between two codes: rows whose norm is exactly 1 (8 and values whose squares are lost next to 64)."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mids = (v[:-1] + v[1:]) / 2
    x = torch.zeros(2 * len(mids), 64)
    x[:, 0], x[:, 32] = 8.0, 448 * 2.0 ** -23
    x[:len(mids), 40], x[len(mids):, 40] = (mids * 2.0 ** -23).float(), (-mids * 2.0 ** -23).float()
    got = M.rms_norm(x.cuda(), torch.ones(64, device="cuda"), 0.0, quantize=True)
    torch.cuda.synchronize()
    assert (got.scale[:, 1] == 127 - 23).all()
    i = torch.arange(len(mids))
    even = i + i % 2
    assert got.codes[:, 40].tolist() == even.tolist() + (even + 128).tolist()


def test_norm_extremes(gpu):
    say("norm extremes")
    w = torch.ones(96, device="cuda")
    z = torch.zeros(3, 96, device="cuda", dtype=torch.bfloat16)
    assert (M.rms_norm(z, w) == 0).all()  # zeros stay zeros
    q = M.rms_norm(z, w, quantize=True)
    assert (q.codes == 0).all() and (q.scale == 127).all()
    x = torch.randn(4, 96, device="cuda").bfloat16()
    x[1, 5], x[2, 40], x[3, 95] = float("nan"), float("inf"), -float("inf")
    y, q = M.rms_norm(x, w), M.rms_norm(x, w, quantize=True)
    torch.cuda.synchronize()
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all()
    for i, j in ((2, 40), (3, 95)):  # an infinite row: 0 where it is finite, NaN where it is not
        assert torch.isnan(y[i, j]) and (y[i].nan_to_num(0) == 0).all()
        assert q.scale[i, j // 32] == 255 and (q.codes[i, j // 32 * 32:j // 32 * 32 + 32] == 0x7F).all()
        assert (q.scale[i, :j // 32] == 127).all()
    assert (q.scale[1] == 255).all() and (q.scale[0] != 255).all()
    for m in (2.0 ** -55, 2.0 ** 55):  # squares far out in fp32
        x = (torch.randn(4, 96) * m).bfloat16().cuda()
        check_norm(x, w, 0.0, None, M.rms_norm(x, w.bfloat16(), 0.0), f"{m}")


def test_norm_in_place_and_shapes(gpu):
    say("norm in place")
    g = torch.Generator().manual_seed(3)
    w = (1 + 0.1 * torch.randn(512, generator=g)).bfloat16().cuda()
    kv = torch.randn(7, 576, generator=g).bfloat16().cuda()
    old = kv.clone()
    assert M.rms_norm(kv[:, :512], w, out=kv[:, :512]).data_ptr() == kv.data_ptr()  # the latent, where it lies
    check_norm(old[:, :512], w, got=kv[:, :512], what="latent")
    assert torch.equal(kv[:, 512:], old[:, 512:])
    x, r = (torch.randn(2, 3, 512, generator=g).bfloat16().cuda() for _ in range(2))
    want = M.rms_norm(x, w, residual=r)
    for out, hout in ((0, 1), (1, 0), (None, 1), (0, None)):  # out and residual_out: x or residual themselves
        a, b = x.clone(), r.clone()
        pick = (a, b)
        y, h = M.rms_norm(a, w, residual=b, out=None if out is None else pick[out], residual_out=None if hout is None else pick[hout])
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
        assert out is None or y is pick[out]
    wide = torch.full((6, 1024), 5.0, dtype=torch.bfloat16, device="cuda")
    y = M.rms_norm(x.view(6, 512), w, out=wide[:, 256:768])
    assert torch.equal(y, M.rms_norm(x, w).view(6, 512)) and (wide[:, :256] == 5).all() and (wide[:, 768:] == 5).all()
    one = torch.randn(1, 512, generator=g).bfloat16().cuda()
    assert torch.equal(M.rms_norm(one.expand(4, 512), w), M.rms_norm(one, w).expand(4, 512))  # a broadcast row
    long = torch.randn(2, 20000, generator=g).cuda()
    lw = torch.ones(20000, device="cuda")
    want = M.rms_norm(long, lw, residual=long * 0.5)
    res = long * 0.5
    y, h = M.rms_norm(long, lw, residual=res, out=long, residual_out=res)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    assert M.rms_norm(torch.empty(0, 512, device="cuda"), torch.ones(512, device="cuda")).shape == (0, 512)
    assert M.rms_norm(torch.empty(0, 512, device="cuda"), torch.ones(512, device="cuda"), quantize=True).scale.shape == (0, 16)


def test_norm_refusals(gpu):
    say("norm refusals")
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    buf = torch.zeros(8 * 64, dtype=torch.bfloat16, device="cuda")
    v = lambda off, st=64: buf[off:].as_strided((4, 64), (st, 1))  # noqa: E731
    for args, kw in [((x.double(), w), {}), ((x[0], w), {}), ((x, w.half()), {}), ((x, w[:32]), {}), ((x, w.cpu()), {}), ((x.t(), w[:4]), {}), ((x, w, -1.0), {}),
                     ((x, w, float("nan")), {}), ((x, w), dict(residual=x[:2])), ((x, w), dict(residual=x.half())), ((x, w), dict(out=x.half())),
                     ((x, w), dict(residual_out=x)), ((x, w), dict(out=x, quantize=True)), ((x[:, :48], w[:48]), dict(quantize=True)),
                     ((v(0), w), dict(out=v(8))), ((v(0), w), dict(out=v(0, 32))), ((v(0), w), dict(residual=v(256), residual_out=v(128))),
                     ((v(0), w), dict(residual=x, out=v(256), residual_out=v(256))), ((x.expand(2, 4, 64).transpose(0, 1), w), {})]:
        with pytest.raises(ValueError):
            M.rms_norm(*args, **kw)


def test_norm_of_millions_of_rows(gpu):
    """More rows than a launch holds threads for at 1024 a row; inputs whose token dim has stride 0, and memory past 2^32
    elements in the output."""
    T, D = 2 ** 22 + 5, 1026
    say("norm millions of rows")
    g = torch.Generator().manual_seed(3)
    pair = torch.randn(2, D, generator=g).bfloat16().cuda()
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    few = M.rms_norm(pair, w)
    y = M.rms_norm(pair[:1].expand(T, D), w)
    torch.cuda.synchronize()
    for part in y.split(2 ** 20):
        assert (part == few[0]).all()
    rows = pair[None].expand(2 ** 11, 2, D).reshape(-1, D)  # [2^12, D], the two in turns
    assert torch.equal(M.rms_norm(rows, w), few.repeat(2 ** 11, 1))
    x = torch.empty(2 ** 24, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        M.rms_norm(x, w[:1])
    assert (M.rms_norm(x.fill_(-3)[1:], w[:1]) == -1).all()


def test_empty_batches(gpu):
    say("empty batches")
    w, packed = torch.ones(64, dtype=torch.bfloat16, device="cuda"), M.quantize_w_fp4(torch.ones(17, 64, device="cuda"))
    for shape in ((0, 64), (3, 0, 64), (0, 3, 64), (2, 3, 0, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        y, h = M.rms_norm(x, w, residual=x)
        assert y.shape == h.shape == shape
        q = M.rms_norm(x, w, quantize=True)
        assert q.codes.shape == shape and q.scale.shape == (*shape[:-1], 2)
        for rows in (x, q):
            assert M.linear_fp4(rows, packed).shape == (*shape[:-1], 17)


def test_outputs_apart_from_the_other_inputs(gpu):
    say("overlaps")
    buf = torch.zeros(64 * 40, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        M.rms_norm(x, buf[:64], out=buf[32:].as_strided((4, 64), (64, 1)))
    with pytest.raises(ValueError):
        M.rms_norm(x, buf[200:264], residual=x, residual_out=buf.as_strided((4, 64), (64, 1)))
    w = M.quantize_w_fp4(torch.zeros(16, 64, device="cuda"))
    raw = buf.view(torch.uint8)
    rows = M.Fp8Rows(raw[:256].view(4, 64), raw[256:264].view(4, 2))
    with pytest.raises(ValueError):
        M.linear_fp4(rows, w, out=buf[131:131 + 64].view(4, 16))
    M.linear_fp4(rows, w, out=buf[132:132 + 64].view(4, 16))
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        M.linear_fp4(x[:1, :32].expand(2 ** 20 + 1, 32), M.quantize_w_fp4(torch.zeros(16, 32, device="cuda")))


def test_norm_in_a_graph(gpu):
    say("norm graph")
    x, r, w = tensors(9, 7168, torch.bfloat16, 7168, 5)
    ww = w.bfloat16().cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        f = lambda: [t for a in (M.rms_norm(x, ww, residual=r), M.rms_norm(x, ww, residual=r, quantize=True)[0]) for t in a]  # noqa: E731
        want = [t.clone() for t in f()]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            res = f()
        for _ in range(3):
            for t in res:
                t.zero_()
            gr.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want))
            f()


# ---------------------------------------------------------------------------------------
# projections by 4-bit weights
# ---------------------------------------------------------------------------------------
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def weights(n, k, seed, spread=8, bias=-4):
    """(codes, scale, values in 64 bits): random codes, scales 2^(bias - spread .. bias + spread)."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 16, (n, k), generator=g)
    s = torch.randint(127 + bias - spread, 128 + bias + spread, (n, k // 32), generator=g)
    v = E2M1[c] * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    return (c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8), s.to(torch.uint8), v


def rows_of(kind, T, k, seed):
    """(what linear_fp4 takes, its values in 64 bits)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, k, generator=g) * torch.exp2(torch.randint(-3, 4, (T, 1), generator=g).float())
    if kind != "fp8":
        x = x.to(DT[kind])
        return x.cuda(), x.double()
    s = torch.randint(120, 130, (T, k // 32), generator=g)
    codes = x.clamp(-448, 448).to(torch.float8_e4m3fn)
    return M.Fp8Rows(codes.view(torch.uint8).cuda(), s.to(torch.uint8).cuda()), codes.double() * torch.exp2(s.double() - 127).repeat_interleave(32, 1)


def check_linear(got, x, w, kind, what):
    """Products are exact; their sum is of k terms in fp32, whatever the order, below k 2^-24 of the sum of their sizes.  The
    block-scaled MFMA (8-bit rows) may drop what lies 13 bits below the largest product of each group of eight: 8 times
    2^-13 of that largest at most, 2^-10 of the sum of sizes.  fp16 rows: weights below 2^-35 of their output's largest
    vanish, those near it round, each by 2^-36 of it.  Then one rounding, and half a smallest step of fp16."""
    y, size = x @ w.T, x.abs() @ w.abs().T
    slack = x.shape[1] * 2.0 ** -24 + (2.0 ** -10 if kind == "fp8" else 0.0)
    tol = EPS[got.dtype] * (1 + slack) * y.abs() + slack * size
    if kind == "f16":
        tol = tol + 2.0 ** -36 * x.abs().sum(1, keepdim=True) * 2 * w.abs().amax(1)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = ((got.double().cpu() - y).abs() / tol.clamp(min=1e-300)).max().item()
    say(f"{what}: {off:.3f} of the bound, {((got.double().cpu() - y).norm() / y.norm()).item():.2e} off")
    assert off <= 1, what


@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("n,k", [(1, 32), (5, 64), (16, 96), (17, 128), (100, 160), (40, 544), (576, 1536), (130, 4128), (1000, 2048)])
def test_linear(gpu, n, k, kind):
    codes, scale, w = weights(n, k, n + k, spread=3 if kind == "f16" else 8)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    for T in (1, 2, 7, 15, 16, 17, 32, 33, 64, 65, 130):
        x, xv = rows_of(kind, T, k, T)
        say(f"linear {kind} T={T} n={n} k={k}")
        got = M.linear_fp4(x, p)
        torch.cuda.synchronize()
        assert got.shape == (T, n) and got.dtype == (torch.float16 if kind == "f16" else torch.bfloat16)
        check_linear(got, xv, w, kind, f"{kind} T={T} n={n} k={k}")


@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8"])
def test_linear_large(gpu, kind):
    """Many chunks a wave, every number of splits, more rows than a workgroup takes."""
    for T, n, k in ((3, 2064, 16384), (64, 528, 16384), (40, 2048, 7168), (300, 1040, 1024), (64, 7168, 512)):
        codes, scale, w = weights(n, k, 3, spread=2)
        x, xv = rows_of(kind, T, k, 5)
        say(f"linear large {kind} {T} {n} {k}")
        got = M.linear_fp4(x, M.pack_w_fp4(codes.cuda(), scale.cuda()))
        torch.cuda.synchronize()
        check_linear(got, xv, w, kind, f"large {kind} {T} {n} {k}")


@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("T,n,k,splits", [(17, 8200, 32, 1), (33, 6000, 160, 1), (40, 5500, 96, 1), (64, 7175, 288, 1), (100, 4112, 1696, 1), (32, 9000, 3200, 2),
                                          (20, 3000, 16384, 10), (64, 2200, 16384, 10), (130, 1500, 16384, 7), (64, 1040, 32768, 16)])
def test_linear_rows_together(gpu, T, n, k, splits, kind):
    """More rows and outputs than go by themselves: both halves of a workgroup, one of them without a chunk, splits that end
    inside a step, outputs past the last tile."""
    ws = M._lib.load().mla_linear_workspace_bytes(T, n, k)
    assert ws == (splits * T * -(-n // 16) * 64 if splits > 1 else 0)
    codes, scale, w = weights(n, k, T + n + k, spread=2)
    x, xv = rows_of(kind, T, k, T)
    say(f"linear together {kind} T={T} n={n} k={k}")
    got = M.linear_fp4(x, M.pack_w_fp4(codes.cuda(), scale.cuda()))
    torch.cuda.synchronize()
    check_linear(got, xv, w, kind, f"together {kind} T={T} n={n} k={k}")


def test_linear_one_hot(gpu):
    """Every weight in its place: rows that pick one input each give the weights back exactly."""
    n, k = 50, 416
    codes, scale, w = weights(n, k, 9, spread=2)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    eye = torch.eye(k, device="cuda")
    say("one hot")
    for x in (eye.bfloat16(), eye.half(), M.Fp8Rows(eye.to(torch.float8_e4m3fn).view(torch.uint8), torch.full((k, k // 32), 127, dtype=torch.uint8, device="cuda"))):
        for a in range(0, k, 16):
            part = M.Fp8Rows(x.codes[a:a + 16], x.scale[a:a + 16]) if isinstance(x, M.Fp8Rows) else x[a:a + 16]
            assert torch.equal(M.linear_fp4(part, p).double().cpu(), w.T[a:a + 16])
        assert torch.equal(M.linear_fp4(x, p).double().cpu(), w.T)


def test_linear_scales_and_special_values(gpu):
    """Scales over the type's whole range (bf16 and 8-bit rows), outputs of very different size (fp16 rows), NaN blocks,
    infinities in the rows, zeros."""
    n, k = 32, 256
    codes, _, _ = weights(n, k, 11)
    scale = torch.arange(n * 8, dtype=torch.int32).view(n, 8) % 200 + 20
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()
    w = E2M1[c] * torch.exp2(scale.double() - 127).repeat_interleave(32, 1)
    p = M.pack_w_fp4(codes.cuda(), scale.to(torch.uint8).cuda())
    for kind in ("bf16", "fp8"):
        x, xv = rows_of(kind, 5, k, 1)
        got = M.linear_fp4(x, p)
        torch.cuda.synchronize()
        check_linear(got, xv, w, kind, f"scales {kind}")
    rows = torch.arange(n, dtype=torch.int32)[:, None].expand(n, 8) % 30 + 100  # each output at a size of its own
    w = E2M1[c] * torch.exp2(rows.double() - 127).repeat_interleave(32, 1)
    x, xv = rows_of("f16", 4, k, 2)
    got = M.linear_fp4(x * 2.0 ** -6, M.pack_w_fp4(codes.cuda(), rows.to(torch.uint8).cuda()), dtype=torch.bfloat16)
    check_linear(got, xv * 2.0 ** -6, w, "f16", "sizes f16")
    scale = torch.full((n, 8), 120, dtype=torch.uint8)
    scale[7, 3] = 255
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    for kind in ("bf16", "f16", "fp8"):
        for T in (2, 20):
            x, _ = rows_of(kind, T, k, 3)
            got = M.linear_fp4(x, p)
            torch.cuda.synchronize()
            assert torch.isnan(got[:, 7]).all() and torch.isfinite(got[:, :7]).all() and torch.isfinite(got[:, 8:]).all(), kind
    x = torch.zeros(3, k, dtype=torch.bfloat16, device="cuda")
    x[1, 40], x[2, 41] = float("nan"), float("inf")
    scale[7, 3] = 120
    got = M.linear_fp4(x, M.pack_w_fp4(codes.cuda(), scale.cuda()))
    torch.cuda.synchronize()
    assert (got[0] == 0).all() and torch.isnan(got[1]).all() and not torch.isfinite(got[2]).any()  # inf * 0 is a NaN
    nan8 = M.Fp8Rows(torch.zeros(2, k, dtype=torch.uint8, device="cuda"), torch.full((2, k // 32), 127, dtype=torch.uint8, device="cuda"))
    nan8.scale[1, 2], nan8.codes[1, 64:96] = 255, 0x7F
    got = M.linear_fp4(nan8, p)
    torch.cuda.synchronize()
    assert torch.isnan(got[1]).all() and (got[0, torch.arange(n, device="cuda") != 7] == 0).all()


@pytest.mark.parametrize("T", [3, 40])
def test_linear_strides_and_shapes(gpu, T):
    n, k = 100, 512
    codes, scale, w = weights(n, k, 13)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    x, xv = rows_of("bf16", T, k, 1)
    want = M.linear_fp4(x, p)
    say(f"strides T={T}")
    wide = torch.zeros(T, 600, dtype=torch.bfloat16, device="cuda")
    for at in (8, 3):  # rows on 16 bytes, and not
        wide[:, at:at + k] = x
        assert torch.equal(M.linear_fp4(wide[:, at:at + k], p), want)
    odd = torch.zeros(T, 601, dtype=torch.bfloat16, device="cuda")[:, :k]
    odd.copy_(x)
    assert torch.equal(M.linear_fp4(odd, p), want)
    assert torch.equal(M.linear_fp4(x.view(1, T, 1, k), p), want.view(1, T, 1, n))
    buf = torch.full((T, 131), 3.0, dtype=torch.bfloat16, device="cuda")
    for at in (4, 1):
        buf.fill_(3.0)
        out = buf[:, at:at + n]
        assert M.linear_fp4(x, p, out=out) is out and torch.equal(out, want)
        assert (buf[:, :at] == 3).all() and (buf[:, at + n:] == 3).all()
    h = M.linear_fp4(x, p, dtype=torch.float16)
    check_linear(h, xv, w, "bf16", "to f16")
    assert M.linear_fp4(x[:0], p).shape == (0, n)
    r, rv = rows_of("fp8", T, k, 2)
    side = M.Fp8Rows(torch.zeros(T, 1024, dtype=torch.uint8, device="cuda")[:, 16:16 + k], torch.zeros(T, 40, dtype=torch.uint8, device="cuda")[:, 3:3 + k // 32])
    side.codes.copy_(r.codes), side.scale.copy_(r.scale)
    assert torch.equal(M.linear_fp4(side, p), M.linear_fp4(r, p))
    off = M.Fp8Rows(torch.zeros(T, k + 8, dtype=torch.uint8, device="cuda")[:, 8:], r.scale)
    off.codes.copy_(r.codes)
    assert torch.equal(M.linear_fp4(off, p), M.linear_fp4(r, p))
    one = x[:1].expand(T, k)
    assert torch.equal(M.linear_fp4(one, p)[0], M.linear_fp4(one, p)[-1])


def test_linear_refusals(gpu):
    say("linear refusals")
    codes, scale, _ = weights(20, 128, 1)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    r = M.Fp8Rows(torch.zeros(4, 128, dtype=torch.uint8, device="cuda"), torch.zeros(4, 4, dtype=torch.uint8, device="cuda"))
    buf = torch.zeros(4 * 128 + 200, dtype=torch.bfloat16, device="cuda")
    for args, kw in [((x.float(), p), {}), ((x[:, :96], p), {}), ((x[0], p), {}), ((x.t(), p), {}), ((x, p._replace(codes=p.codes[:1])), {}), ((x, p._replace(top=p.top.cpu())), {}),
                     ((x, p._replace(n=40)), {}), ((x, p), dict(dtype=torch.float32)), ((x, p), dict(out=torch.zeros(4, 21, dtype=x.dtype, device="cuda"))),
                     ((x, p), dict(out=torch.zeros(4, 20, dtype=torch.float16, device="cuda"), dtype=torch.bfloat16)), ((r._replace(scale=r.scale[:, :3]), p), {}),
                     ((r._replace(scale=r.scale.int()), p), {}), ((r._replace(codes=r.codes.int()), p), {}), ((x, p), dict(out=buf[:80].view(4, 20).expand(4, 20)[:1].expand(4, 20))),
                     ((buf[:512].view(4, 128), p), dict(out=buf[480:560].view(4, 20))), ((x.expand(2, 4, 128).transpose(0, 1), p), {})]:
        with pytest.raises(ValueError):
            M.linear_fp4(*args, **kw)


def test_linear_streams_and_graphs(gpu):
    """Two captured calls that share a stream's workspace, replayed in turns, and two streams at once."""
    k, n, T = 16384, 4096, 64
    codes, scale, _ = weights(n, k, 21)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    xs = [rows_of("bf16", T, k, i)[0] for i in range(3)]
    want = [M.linear_fp4(x, p) for x in xs]
    torch.cuda.synchronize()
    say("linear graphs")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(M.linear_fp4(xs[0], p), want[0])
        graphs = []
        for x in xs[:2]:
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                y = M.linear_fp4(x, p)
            graphs.append((gr, y))
        for _ in range(3):
            for (gr, y), wt in zip(graphs, want):
                y.zero_()
                gr.replay()
                assert torch.equal(M.linear_fp4(xs[2], p), want[2])
                side.synchronize()
                assert torch.equal(y, wt)
    other = torch.cuda.Stream()
    got = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else other):
            got.append(M.linear_fp4(xs[i % 3], p))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))


def test_norm_then_linear(gpu):
    """The norm's 8-bit rows through a projection, against the same in 64 bits of what the rows hold; and the absorbed
    decode's output projection by such weights."""
    T, D, n = 9, 7168, 576
    x, r, w = tensors(T, D, torch.bfloat16, D, 3)
    codes, scale, wv = weights(n, D, 5, spread=2)
    p = M.pack_w_fp4(codes.cuda(), scale.cuda())
    say("norm then linear")
    rows, _ = M.rms_norm(x, w.cuda(), residual=r, quantize=True)
    y = M.linear_fp4(rows, p)
    torch.cuda.synchronize()
    check_linear(y, values8(rows).cpu(), wv, "fp8", "norm then linear")


def test_absorbed_with_4bit_output_projection(gpu):
    B, H, D = 3, 16, 320
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(6, 64, 1, 576, generator=g).bfloat16().cuda()
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(B, 2)
    lens = torch.tensor([100, 64, 7], dtype=torch.int32, device="cuda")
    q = torch.randn(B, 1, H, 576, generator=g).bfloat16().cuda()
    w_uv = M.prepare_w_uv((torch.randn(H, 512, 128, generator=g) * 512 ** -0.5).bfloat16().cuda())
    w_o = M.quantize_w_fp4(torch.randn(D, H * 128, generator=g).cuda() * (H * 128) ** -0.5)
    say("absorbed with w_o")
    sched = M.get_mla_metadata(lens, H, 1)
    v, _ = M.mla_decode_absorbed(q, kv, table, lens, *sched, w_uv)
    y, _ = M.mla_decode_absorbed(q, kv, table, lens, *sched, w_uv, w_o)
    assert y.shape == (B, 1, D) and torch.equal(y, M.linear_fp4(v.view(B, 1, H * 128), w_o))
