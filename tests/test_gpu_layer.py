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
