"""GPU tests of the operators around the attention where every sum is exact: no tolerance hides a term that is lost, taken
twice or in another's place."""
import sys

import pytest
import torch

import mlc_decode_amd as M

pytestmark = pytest.mark.gpu

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def say(msg):
    print(f"[gpu-layer-edges] {msg}", flush=True)
    sys.stdout.flush()


def packed(codes, scale):
    """Weights from codes 0 .. 15 [n, k] and scale bytes [n, k / 32], and their values in 64 bits."""
    w = E2M1[codes] * torch.exp2(scale.double() - 127).repeat_interleave(32, 1)
    return M.pack_w_fp4((codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).cuda(), scale.to(torch.uint8).cuda()), w


def given(x, kind):
    """Rows of 64-bit values as linear_fp4 takes them; 8-bit ones with scales 2^-1 .. 2^1 in turns."""
    if kind != "fp8":
        assert torch.equal(x.to(DT[kind]).double(), x)
        return x.to(DT[kind]).cuda()
    s = 126 + torch.arange(x.shape[0] * x.shape[1] // 32).view(x.shape[0], -1) % 3
    v = x * torch.exp2(127 - s.double()).repeat_interleave(32, 1)
    codes = v.to(torch.float8_e4m3fn)
    assert torch.equal(codes.double(), v)
    return M.Fp8Rows(codes.view(torch.uint8).cuda(), s.to(torch.uint8).cuda())


def exactly(T, n, k, kind, seed):
    """(rows, weights, y in 64 bits).  Values of the rows are multiples of 1/2 up to 3 and pairs of +-224 eight inputs apart or
    fewer, those of the weights multiples of 1/4 up to 12 of one size in a pair's places, so that what is left of 224 * 12 less
    itself is the small products'.  All products are multiples of 2^-3 and their sizes add up to less than 2^21: every sum of some of them, in any order, is exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-6, 7, (T, k), generator=g).double() / 2
    codes = torch.randint(0, 16, (n, k), generator=g)
    for a in range(0, k - 8, max(32, k // 24 // 8 * 8)):  # a pair in each of some groups of eight
        i, j = a + int(torch.randint(0, 4, (1,), generator=g)), a + int(torch.randint(4, 8, (1,), generator=g))
        x[:, i], x[:, j] = 224.0, -224.0
        codes[:, i] = codes[:, j]
    scale = torch.randint(126, 129, (n, k // 32), generator=g)
    p, w = packed(codes, scale)
    assert (x.abs() @ w.abs().T).max() < 2 ** 21
    return given(x, kind), p, x @ w.T


SHAPES = [(1, 576, 7168), (3, 2064, 16384), (16, 100, 7168), (8, 25600, 160), (17, 576, 7168),     # by themselves, 4, 8 and 16 waves
          (32, 12288, 512), (17, 8200, 32), (33, 6000, 160), (40, 5500, 96), (64, 7175, 288),        # together, one split
          (32, 9000, 3200), (20, 3000, 16384), (64, 2200, 16384), (130, 1500, 16384), (64, 1040, 32768), (200, 2100, 7168 + 96)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("T,n,k", SHAPES)
def test_linear_exact(gpu, T, n, k, kind):
    """Outputs are the exact sums, rounded once: every product in its place, none lost beside larger ones."""
    rows, p, y = exactly(T, n, k, kind, T + n + k)
    for dtype in (torch.bfloat16, torch.float16):
        say(f"exact {kind} T={T} n={n} k={k} to {dtype}")
        got = M.linear_fp4(rows, p, dtype=dtype)
        torch.cuda.synchronize()
        want = y.to(dtype)
        assert torch.equal(got.cpu(), want), f"{(got.cpu() != want).sum().item()} of {want.numel()} differ"


@pytest.mark.parametrize("T", [1, 5, 9, 16, 40])
def test_linear_8bit_small_products_beside_large_ones(gpu, T):
    """An outlier's products cancel and leave those of its neighbours, 2^19 times smaller, whole: 448 * 6 and 2^-8."""
    k, n = 64, 16 if T <= 16 else 16 * 1100
    x = torch.zeros(T, k, dtype=torch.float64)
    codes = torch.zeros(n, k, dtype=torch.long)
    for j in range(0, k, 8):
        x[:, j], x[:, j + 3], x[:, j + 1:j + 3], x[:, j + 4:j + 8] = 448.0, -448.0, 2.0 ** -7, 2.0 ** -7
        codes[:, [j, j + 3]], codes[:, j + 1:j + 3], codes[:, j + 4:j + 8] = 7, 1, 1  # 6, and 0.5
    p, w = packed(codes, torch.full((n, k // 32), 127))
    rows = M.Fp8Rows(x.to(torch.float8_e4m3fn).view(torch.uint8).cuda(), torch.full((T, k // 32), 127, dtype=torch.uint8, device="cuda"))
    y = x @ w.T
    assert (y == 48 * 2.0 ** -8).all()
    say(f"outliers T={T}")
    got = M.linear_fp4(rows, p)
    torch.cuda.synchronize()
    assert (got.double().cpu() == y).all(), got[0, :4]


@pytest.mark.parametrize("T", [4, 40])
def test_linear_8bit_scales_one_hot(gpu, T):
    """A code of each size at scales over bf16's range, in every block of a row: rows that pick one input each; a scale byte
    of 255 is a NaN whatever its codes, and of its own row alone."""
    k, n = 160, 64 if T <= 16 else 16 * 1100
    p, w = packed(torch.full((n, k), 2), torch.full((n, k // 32), 127))
    x = torch.zeros(T, k, dtype=torch.uint8)
    s = torch.full((T, k // 32), 127, dtype=torch.uint8)
    g = torch.Generator().manual_seed(T)
    codes = torch.randint(1, 127, (T,), generator=g)
    at = torch.randint(0, k, (T,), generator=g)
    for t in range(T):
        x[t, at[t]] = codes[t]
        s[t, at[t] // 32] = 12 + (t * 37) % 230  # 2^-115 .. 2^114: with codes of 2^-9 .. 448 inside bf16's normal numbers
    want = x.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    want = want.sum(1, keepdim=True).expand(T, n)
    rows = M.Fp8Rows(x.cuda(), s.cuda())
    say(f"scales T={T}")
    got = M.linear_fp4(rows, p)
    torch.cuda.synchronize()
    assert torch.equal(got.double().cpu(), want)
    rows.scale[1, 4] = 255  # its codes are zeros, or one
    bad = M.linear_fp4(rows, p)
    torch.cuda.synchronize()
    assert bad[1].isnan().all() and torch.equal(bad[0], got[0]) and torch.equal(bad[2:], got[2:])


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("k", [96, 128, 416])
@pytest.mark.parametrize("top", [3, 10, 80, 140, 250])
def test_linear_f16_rows_by_weights_of_any_size(gpu, T, k, top):
    """fp16 rows take weights relative to their output's largest, whether or not the last chunk has inputs past the end: exact
    sums of eight products a row, rounded once to bf16."""
    n = 50 if T <= 16 else 16 * 1100
    g = torch.Generator().manual_seed(k + top)
    p, w = packed(torch.randint(0, 16, (n, k), generator=g), torch.randint(top - 2, top + 1, (n, k // 32), generator=g))
    assert (p.top[:n].cpu() == p.scale.cpu().view(-1, p.scale.shape[1], 4, 16).permute(0, 3, 1, 2).reshape(-1, 4 * p.scale.shape[1])[:n, :k // 32].amax(1)).all()
    x = torch.zeros(T, k, dtype=torch.float64)
    x[:, k - 32:] = torch.randint(1, 5, (T, 32), generator=g).double()
    x[:, k - 24:] = 0
    x[:, 0] = 4
    say(f"f16 rows T={T} k={k} top={top}")
    got = M.linear_fp4(x.half().cuda(), p, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    want = (x @ w.T).to(torch.bfloat16)  # top 250: of up to 2^130, some past bf16's range
    assert want.abs().max() > 0
    assert (got.cpu() == want).all()


def test_norm_refuses_an_eps_that_fp32_does_not_hold(gpu):
    say("extreme eps")
    x, w = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for eps in (1e39, 3.4028235677973366e38):
        with pytest.raises(ValueError):
            M.rms_norm(x, w, eps)
    assert (M.rms_norm(x, w, 3.4028234e38) == 2.0 ** -64).all()


def test_linear_refuses_outputs_in_the_weights(gpu):
    """Projections that would write over the weights that they read: codes, scales, largest scales."""
    say("outputs in the weights")
    x = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda")
    buf = torch.zeros(2048, dtype=torch.uint8, device="cuda")
    p = M.quantize_w_fp4(torch.zeros(16, 64, device="cuda"))
    for name, at in (("codes", 0), ("scale", 1024), ("top", 1024 + 64)):
        buf[at:at + getattr(p, name).numel()].copy_(getattr(p, name).flatten())
    p = p._replace(codes=buf[:1024].view(p.codes.shape), scale=buf[1024:1088].view(p.scale.shape), top=buf[1088:1104])
    half = buf.view(torch.bfloat16)
    for at in (0, 449, 511, 540, 551):
        with pytest.raises(ValueError):
            M.linear_fp4(x, p, out=half[at:at + 64].view(4, 16))
    assert M.linear_fp4(x, p, out=half[552:616].view(4, 16)).data_ptr() == half[552:].data_ptr()
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["f16", "fp8"])
@pytest.mark.parametrize("T,n,k", [(5, 576, 7168), (64, 2200, 16384)])
def test_linear_of_every_kind_in_a_graph(gpu, T, n, k, kind):
    """Captured once and replayed beside eager calls of the same stream, with rows that change in place, and on two streams at
    once."""
    rows, p, y = exactly(T, n, k, kind, 7)
    other, _, _ = exactly(T, n, k, kind, 7)
    parts = lambda r: list(r) if isinstance(r, M.Fp8Rows) else [r]  # noqa: E731
    for t in parts(other):
        t.copy_(t.flip(0))
    want, flipped = y.to(torch.bfloat16), M.linear_fp4(other, p, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    say(f"graph {kind} T={T}")
    side, third = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(M.linear_fp4(rows, p, dtype=torch.bfloat16).cpu(), want)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            got = M.linear_fp4(rows, p, dtype=torch.bfloat16)
        first = [t.clone() for t in parts(rows)]
        for i in range(4):
            for t, a, b in zip(parts(rows), first, parts(other)):
                t.copy_(b if i % 2 else a)
            got.zero_()
            gr.replay()
            eager = M.linear_fp4(other, p, dtype=torch.bfloat16)
            side.synchronize()
            assert torch.equal(got.cpu(), flipped.cpu() if i % 2 else want) and torch.equal(eager, flipped)
    results = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else third):
            results.append(M.linear_fp4(other, p, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    assert all(torch.equal(r, flipped) for r in results)
