"""Operators of a serving step around the paged MLA decode, and the cases they are measured on.

  decode   attention over the latent cache held in 4 bits: e2m1 codes, one power-of-two scale per token and 32
           dims, the 64 rope dims in bf16.  ``flash_mla_with_kvcache`` with the step's schedule in hand,
           ``mla_decode_with_kvcache`` where it schedules too, and the sparse form with an index list
  rope     ``apply_rope``: rotary positions on the rotated part of each head
  append   ``kv_append_slots``: a step's new tokens, their key part rotated, written to the cache rows that a slot
           map names, and the queries' rope part rotated into the query buffer; caches of 4 and 8 bits come
           back as values, through ``kv_gather``
  gather   ``kv_gather``: cached tokens, named by slot, as bf16 rows (what a chunked prefill attends to)
  pages    ``reserve_pages`` and ``release_pages``: pages, block tables and slot maps of a step's new tokens,
           and their return when the tokens are rejected again

The lengths of a case are fixed by its values, so that its work is known; page order, contents, queries and index
lists come from the seed.  Latents are N(0, 1) (they come from a normalisation), as in the repository's other inputs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE, D_QK, D_V, D_ROPE = 64, 576, 512, 64
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, kind, **kw):
    base = {
        # s_q query tokens of `heads` heads for each of `batch` sequences of lo .. hi cached tokens; topk keys of each
        "decode": dict(batch=1, heads=16, s_q=1, lo=1024, hi=1024, topk=0, auto=False),
        # tokens x heads x dim, `rot` of the dims from `first` on rotated; heads are `pitch` elements apart
        "rope": dict(tokens=1, heads=16, dim=64, pitch=64, rot=64, first=0, layout="interleaved", scaling="none", base=10000.0, far=4096, dtype="bf16"),
        # lo .. hi cached and new_lo .. new_hi new tokens per sequence, `pad` rows behind the last one
        "append": dict(batch=1, heads=16, lo=1, hi=4096, new_lo=1, new_hi=1, pad=0, cache="bf16", layout="interleaved", scaling="yarn", far=163840),
        "gather": dict(tokens=64, pages=64, holes=False, cache="fp4"),
        # a pool of the cached and new tokens' pages; `short` of them are missing, so the last requests are refused
        "pages": dict(batch=1, lo=0, hi=8192, new_lo=1, new_hi=1, pad=0, short=0),
    }[kind]
    return dict(base, kind=kind, name=name, **kw)


def listed():
    return [
        # one short conversation on one tensor-parallel rank: schedule and decode, launches and latency count
        _case("decode_auto_b1_h16_l1024", "decode", auto=True),
        # one of eight tensor-parallel ranks, a ragged batch: bound by the cache's bytes
        _case("decode_b128_h16_ragged", "decode", batch=128, lo=256, hi=8192),
        # all 128 heads of a token on one GPU, 64 sequences of 4096 tokens
        _case("decode_b64_h128_l4096", "decode", batch=64, heads=128, lo=4096, hi=4096),
        # long contexts, two query tokens (multi-token prediction), all heads: the largest case
        _case("decode_b32_s2_h128_l16384", "decode", batch=32, s_q=2, heads=128, lo=16384, hi=16384),
        # sparse attention: the top 2048 tokens of 8192-token contexts, all heads
        _case("sparse_b64_h128_top2048", "decode", batch=64, heads=128, lo=8192, hi=8192, topk=2048),
        # the queries of one decode step: the rope part of a [tokens, heads, 192] projection, far positions
        _case("rope_t128_h128_step", "rope", tokens=128, heads=128, pitch=192, first=0, scaling="yarn", far=163840),
        # a prefill chunk in the other layout: half of 128-dim heads, fp16, positions divided by 8
        _case("rope_t8191_h32_half", "rope", tokens=8191, heads=32, dim=128, pitch=128, rot=64, layout="half", scaling="linear", far=32768, dtype="f16"),
        # one decode step's append on a tensor-parallel rank: a token per sequence into the bf16 cache, and its queries
        _case("append_b128_n1_bf16", "append", batch=128, lo=64, hi=64, far=163840),
        # a ragged prefill chunk into the 4-bit cache, padded to the captured size, and the pool read back
        _case("append_b32_ragged_fp4", "append", batch=32, lo=0, hi=512, new_lo=1, new_hi=1024, pad=100, cache="fp4"),
        # the context of a chunked prefill: 65,536 cached tokens of the fp8 cache as bf16 rows
        _case("gather_t65536_fp8", "gather", tokens=65536, pages=2048, cache="fp8"),
        # the bookkeeping of a decode step: one token per sequence, some need a page
        _case("pages_b128_n1", "pages", batch=128),
        # of a large ragged prefill: up to 512 new tokens each, the pool runs out before the last requests
        _case("pages_b512_ragged", "pages", batch=512, hi=32768, new_lo=0, new_hi=512, pad=1000, short=100),
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the ranges above: sizes log-uniform, odd and ragged ones among them."""
    most = {k: max(w[k] for w in map(work, listed())) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(("decode", "decode", "decode", "rope", "append", "gather", "pages"))
        c = _case("", kind)
        del c["name"]
        if kind == "decode":
            hi = _log_int(rng, 1, 32768)
            c.update(batch=_log_int(rng, 1, 256), heads=rng.choice((1, 8, 16, 16, 24, 32, 40, 64, 96, 128, 128)), s_q=rng.choice((1, 1, 1, 2, 3, 4)), hi=hi)
            c["lo"] = hi if rng.random() < 0.3 else hi // rng.choice((2, 8, 32))
            if rng.random() < 0.2:
                c.update(s_q=1, lo=max(hi, 64), hi=max(hi, 64))
                c["topk"] = _log_int(rng, 1, min(2048, c["hi"]))
            c["auto"] = not c["topk"] and rng.random() < 0.3
            if c["batch"] * c["hi"] > 1 << 20 or c["batch"] * c["s_q"] * c["heads"] * c["hi"] > 1 << 28:
                continue  # the plain form pads every sequence to the longest
        elif kind == "rope":
            rot = 2 * _log_int(rng, 4, 64)
            c.update(tokens=_log_int(rng, 1, 16384), heads=_log_int(rng, 1, 128), rot=rot, first=rng.choice((0, 0, 1, 8, 64)), far=_log_int(rng, 1024, 1 << 20))
            c["dim"] = c["first"] + rot + rng.choice((0, 0, 3, 64))
            c["pitch"] = c["dim"] + rng.choice((0, 0, 5, 128))
            c.update(layout=rng.choice(("interleaved", "half")), scaling=rng.choice(("none", "linear", "ntk", "yarn")), dtype=rng.choice(("bf16", "bf16", "f16", "f32")), base=rng.choice((10000.0, 500000.0)))
        elif kind == "append":
            new = _log_int(rng, 1, 2048)
            c.update(batch=_log_int(rng, 1, 256), heads=rng.choice((0, 8, 16, 24, 128)), lo=0, hi=_log_int(rng, 1, 1024), new_hi=new, new_lo=rng.choice((0, 1, new)), pad=rng.choice((0, 0, 7, 64)))
            c.update(cache=rng.choice(("bf16", "f16", "fp8", "fp4", "fp4")), layout=rng.choice(("interleaved", "half")), scaling=rng.choice(("none", "yarn")))
        elif kind == "gather":
            c.update(tokens=_log_int(rng, 1, 131072), pages=_log_int(rng, 1, 4096), holes=rng.random() < 0.3, cache=rng.choice(("bf16", "fp8", "fp4", "fp4")))
        else:
            new = _log_int(rng, 1, 2048)
            c.update(batch=_log_int(rng, 1, 2048), hi=_log_int(rng, 1, 32768), new_hi=new, new_lo=rng.choice((0, 1, new)), pad=rng.choice((0, 0, 100)), short=rng.choice((0, 0, 1, 50)))
        rows = sum(_new(c)) + c.get("pad", 0) if kind in ("append", "pages") else 1
        w = work(c)
        if 1 <= rows <= 131072 and w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


# ---------------------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------------------
def _cached(c):
    """Cached tokens of each sequence before the call."""
    r = random.Random("%d %d %d" % (c["batch"], c["lo"], c["hi"]))
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]


def _new(c):
    """New tokens of each sequence."""
    r = random.Random("new %d %d %d" % (c["batch"], c["new_lo"], c["new_hi"]))
    return [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


_TOKEN = {"bf16": 1152, "f16": 1152, "fp8": 512 + 16 + 128, "fp4": 256 + 16 + 128}  # bytes of a cached token


def work(c):
    """Each input read once, each output written once; the two products of every visible (row, key) pair."""
    if c["kind"] == "decode":
        lens = [c["topk"]] * c["batch"] if c["topk"] else _cached(c)
        rows = c["batch"] * c["s_q"] * c["heads"]
        seen = sum(max(0, n - i) for n in lens for i in range(c["s_q"])) * c["heads"]
        return {"bytes": sum(lens) * (_TOKEN["fp4"] + (4 if c["topk"] else 0)) + rows * (2 * D_QK + 2 * D_V + 4), "flops": 2 * seen * (D_QK + D_V)}
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * (4 if c["dtype"] == "f32" else 2) + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    if c["kind"] == "append":
        n = sum(_new(c))
        b = n * (2 * D_QK + _TOKEN[c["cache"]] + 8 + c["heads"] * 4 * D_ROPE)
        if c["cache"] in ("fp8", "fp4"):
            b += _pool_pages(c) * PAGE * (_TOKEN[c["cache"]] + 2 * D_QK)
        return {"bytes": b, "flops": 3 * n * D_ROPE * (1 + c["heads"])}
    if c["kind"] == "gather":
        return {"bytes": c["tokens"] * (_TOKEN[c["cache"]] + 2 * D_QK + 4), "flops": 0}
    n = sum(_new(c))
    return {"bytes": 8 * (n + c["pad"]) + 8 * _pages(n) + 8 * c["batch"] * 4, "flops": 0}


def _pool_pages(c):
    return sum(_pages(a + b) for a, b in zip(_cached(c), _new(c)))


def _freqs(c):
    """Turns per position of each rotated pair, and the factor on cosine and sine."""
    d = c.get("rot", D_ROPE)
    base, factor, orig = c.get("base", 10000.0), 8.0, 4096
    if c["scaling"] == "ntk":
        base *= factor ** (d / (d - 2))
    f = [base ** (-2 * i / d) for i in range(d // 2)]
    amp = 1.0
    if c["scaling"] == "linear":
        f = [v / factor for v in f]
    if c["scaling"] == "yarn":  # pairs that turn often keep their speed, slow ones are stretched, a ramp between
        edge = lambda turns: d * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(edge(32.0)), 0), min(math.ceil(edge(1.0)), d - 1)
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(d // 2)]
        f = [v / factor * r + v * (1 - r) for v, r in zip(f, ramp)]
        amp = 0.1 * math.log(factor) + 1.0
    return [v / (2 * math.pi) for v in f], amp


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _layout(c, lens, extra, g):
    """A block table over a shuffled pool for lens + extra tokens per sequence."""
    pages = [_pages(n) + e for n, e in zip(lens, extra)]
    ids = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(max(pages), 1), dtype=torch.int32, device="cuda")
    n = torch.tensor(pages, device="cuda")
    at = torch.arange(table.shape[1], device="cuda")[None] < n[:, None]
    table[at] = ids
    return table, max(sum(pages), 1)


def _pool(cache, pages, g):
    """A filled pool: bf16 / f16 rows, or codes and scales as random tokens of unit variance have them."""
    kv = torch.randn(pages, PAGE, D_QK, generator=g, dtype=torch.float32, device="cuda")
    if cache in ("bf16", "f16"):
        return {"kv": kv.to(_DT[cache]).unsqueeze(2)}
    rope = kv[..., D_V:].to(torch.bfloat16).contiguous()
    parts = [(_fp4 if cache == "fp4" else _fp8)(p.to(torch.bfloat16)[..., :D_V].float()) for p in kv.split(2048)]
    latent, scale = (torch.cat([p[i] for p in parts]) for i in range(2))
    return {"latent": latent, "scale": scale if cache == "fp4" else scale.transpose(1, 2).contiguous(), "rope": rope}


def prepare(c, seed):
    """The inputs, and what a program has ready before the call: of a decode, the step's schedule."""
    g = torch.Generator("cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x = {"case": c}
    if c["kind"] in ("rope", "append"):
        f, x["amp"] = _freqs(c)
        x["freqs"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if c["kind"] == "decode":
        lens = _cached(c)
        x["lens"] = ints(lens)
        x["table"], n = _layout(c, lens, [0] * len(lens), g)
        x.update(_pool("fp4", n, g))
        x["q"] = torch.randn(c["batch"], c["s_q"], c["heads"], D_QK, generator=g, dtype=torch.bfloat16, device="cuda")
        if c["topk"]:  # a random subset of each sequence's tokens, in no order, as pool token ids
            pos = torch.rand(c["batch"], c["hi"], generator=g, device="cuda").topk(c["topk"], dim=1).indices
            x["indices"] = (torch.gather(x["table"].long(), 1, pos // PAGE) * PAGE + pos % PAGE).to(torch.int32).unsqueeze(1)
        if own and not c["auto"]:
            import mlc_decode_amd as M
            cache = M.Fp4KVCache(x["latent"], x["scale"], x["rope"])
            x["sched"] = M.get_mla_metadata(x["lens"], c["s_q"] * c["heads"], 1, topk=c["topk"] or None, kv_cache=cache)
    elif c["kind"] == "rope":
        wide = torch.randn(c["tokens"], c["heads"], c["pitch"], generator=g, dtype=torch.float32, device="cuda").to(_DT[c["dtype"]])
        x["x"] = wide[..., c["pitch"] - c["dim"]:]
        x["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, dtype=torch.int32, device="cuda")
    elif c["kind"] == "append":
        dt = torch.float16 if c["cache"] == "f16" else torch.bfloat16
        lens, new = _cached(c), _new(c)
        table, n = _layout(c, [a + b for a, b in zip(lens, new)], [0] * len(lens), g)
        x.update(_pool(c["cache"], n, g))
        seq = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), torch.tensor(new, device="cuda"))
        before = torch.tensor([sum(new[:b]) for b in range(c["batch"])], device="cuda")
        pos = torch.arange(sum(new), device="cuda") - before[seq] + torch.tensor(lens, device="cuda")[seq]
        slots = table.long()[seq, pos // PAGE] * PAGE + pos % PAGE
        none = torch.full((c["pad"],), -1, device="cuda")
        x["slots"] = torch.cat([slots, none]).to(torch.int32)
        x["positions"] = torch.cat([pos + (c["far"] - 1 - 8192), none]).to(torch.int32)
        T = x["slots"].numel()
        x["kv_new"] = torch.randn(T, D_QK, generator=g, dtype=torch.float32, device="cuda").to(dt)
        if c["heads"]:
            x["q_pe"] = torch.randn(T, c["heads"], 192, generator=g, dtype=torch.float32, device="cuda").to(dt)[..., 128:]
            x["q"] = torch.randn(T, c["heads"], D_QK, generator=g, dtype=torch.float32, device="cuda").to(dt)
        x["all"] = torch.arange(n * PAGE, dtype=torch.int32, device="cuda")
    elif c["kind"] == "gather":
        x.update(_pool(c["cache"], c["pages"], g))
        x["slots"] = torch.randint(0, c["pages"] * PAGE, (c["tokens"],), generator=g, dtype=torch.int32, device="cuda")
        if c["holes"]:
            x["slots"][::5] = -1
    else:
        lens, new = _cached(c), _new(c)
        x["lens"], x["new"] = ints(lens), ints(new)
        x["keep"] = x["lens"].clone()
        need = [_pages(a + b) - _pages(a) for a, b in zip(lens, new)]
        x["table"], _ = _layout(c, lens, need, g)
        held = sum(map(_pages, lens))
        order = torch.randperm(max(held + sum(need), 1), generator=g, device="cuda").to(torch.int32)
        x["table"][torch.arange(x["table"].shape[1], device="cuda")[None] < _ceil(x["lens"])[:, None]] = order[:held]
        x["free"] = torch.cat([order[held:], order[:held]])  # a stack: the first `count` are free
        x["count"] = ints([max(0, sum(need) - c["short"])])
        x["tokens"] = sum(new) + c["pad"]
    return x


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------
def _ceil(t):
    return torch.div(t + (PAGE - 1), PAGE, rounding_mode="floor")


def _fp4(x):
    """Values [..., 512] -> codes [..., 256] (two a byte, the even dim low) and scale bytes [..., 16]: the scale of
    32 dims is the smallest 2^k with amax <= 6 * 2^k, stored as k + 127 (zeros: k = 0; k in -126 .. 127), values
    rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even code."""
    b = x.unflatten(-1, (16, 32))
    a = b.abs().amax(-1)
    m, e = torch.frexp(a)
    k = torch.where(a == 0, torch.zeros_like(e), torch.where(m <= 0.75, e - 3, e - 2).clamp(-126, 127))
    v = torch.ldexp(b, -k[..., None])
    a = v.abs()
    n = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    n = (n + 8 * torch.signbit(v)).to(torch.uint8).flatten(-2).unflatten(-1, (256, 2))
    return n[..., 0] | (n[..., 1] << 4), (k + 127).to(torch.uint8)


def _fp4_values(codes, scale):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return torch.ldexp(v.unflatten(-1, (16, 32)), scale[..., None].int() - 127).flatten(-2)


def _fp8(x):
    """Values [..., 512] -> e4m3 codes and the fp32 scales of 4 blocks of 128: the smallest 2^k with amax <= 448 * 2^k."""
    b = x.unflatten(-1, (4, 128))
    a = b.abs().amax(-1)
    m, e = torch.frexp(a)
    k = torch.where(a == 0, torch.zeros_like(e), torch.where(m <= 0.875, e - 9, e - 8).clamp(-126, 127))
    codes = torch.ldexp(b, -k[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    return codes, torch.ldexp(torch.ones_like(a), k)


def _rows(x, page, row):
    """Cached tokens (page, row) as fp32 [..., 576]."""
    if "kv" in x:
        return x["kv"][page, row, 0].float()
    if x["scale"].dtype == torch.uint8:
        v = _fp4_values(x["latent"][page, row], x["scale"][page, row])
    else:
        s = x["scale"].transpose(1, 2)[page, row]
        v = (x["latent"][page, row].view(torch.float8_e4m3fn).float().unflatten(-1, (4, 128)) * s[..., None]).flatten(-2)
    return torch.cat([v, x["rope"][page, row].float()], -1)


def _rotate(x, positions, freqs, amp, layout):
    """x [T, ..., rot] in fp32, rotated by positions [T]; rows of a negative position as they were."""
    turns = positions.double()[:, None] * freqs
    angle = (turns - torch.floor(turns)) * (2 * math.pi)
    shape = (positions.numel(),) + (1,) * (x.dim() - 2) + (freqs.numel(),)
    c, s = ((f(angle) * amp).float().reshape(shape) for f in (torch.cos, torch.sin))
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x.chunk(2, -1)
        y = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.where((positions >= 0).reshape(shape[:-1] + (1,)), y, x)


def _plain_decode(x):
    c, scale = x["case"], D_QK ** -0.5
    B, S, H = x["q"].shape[:3]
    if c["topk"]:
        at = x["indices"][:, 0].long()
        k, n = _rows(x, at // PAGE, at % PAGE), c["topk"]
        lens = torch.full((B,), n, device=x["q"].device)
    else:
        n, lens = c["hi"], x["lens"]
        t = torch.arange(n, device=lens.device)
        col = (t // PAGE).clamp(max=x["table"].shape[1] - 1)
        k = _rows(x, x["table"][:, col].long(), (t % PAGE)[None].expand(B, -1))
    s = torch.matmul(x["q"].reshape(B, S * H, D_QK).float(), k.transpose(1, 2).contiguous()).reshape(B, S, H, -1) * scale
    last = lens[:, None] - torch.arange(S - 1, -1, -1, device=lens.device)  # tokens query i sees
    s = s.masked_fill(torch.arange(s.shape[-1], device=lens.device) >= last[:, :, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, S * H, -1), k[..., :D_V].contiguous()).reshape(B, S, H, D_V)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.to(x["q"].dtype), (m + torch.log(total)).squeeze(-1).transpose(1, 2).contiguous()


def _plain_rope(x):
    c, y = x["case"], x["x"].float()
    a, b = c["first"], c["first"] + c["rot"]
    turned = _rotate(y[..., a:b], x["positions"], x["freqs"], x["amp"], c["layout"])
    return torch.cat([y[..., :a], turned, y[..., b:]], -1).to(x["x"].dtype)


def _plain_append(x):
    c, dt = x["case"], x["kv_new"].dtype
    on = x["slots"] >= 0
    slot, pos, new = x["slots"][on].long(), x["positions"][on], x["kv_new"][on]
    page, row = slot // PAGE, slot % PAGE
    pe = _rotate(new[:, D_V:].float(), pos, x["freqs"], x["amp"], c["layout"]).to(dt)
    if "kv" in x:
        x["kv"][page, row, 0] = torch.cat([new[:, :D_V], pe], -1)
    elif c["cache"] == "fp4":
        x["latent"][page, row], x["scale"][page, row] = _fp4(new[:, :D_V].float())
        x["rope"][page, row] = pe
    else:
        x["latent"][page, row], scale = _fp8(new[:, :D_V].float())
        x["scale"].transpose(1, 2)[page, row] = scale
        x["rope"][page, row] = pe
    out = {"cache": x["kv"] if "kv" in x else _rows(x, x["all"].long() // PAGE, x["all"].long() % PAGE).to(dt)}
    if c["heads"]:
        turned = _rotate(x["q_pe"][on].float(), pos, x["freqs"], x["amp"], c["layout"]).to(dt)
        x["q"][..., D_V:][on] = turned
        out["q"] = x["q"]
    return out


def _plain_gather(x):
    slot = x["slots"].long()
    rows = _rows(x, slot.clamp(min=0) // PAGE, slot.clamp(min=0) % PAGE)
    return torch.where((slot >= 0)[:, None], rows, torch.zeros_like(rows)).to(torch.bfloat16)


def _plain_pages(x):
    table, lens, free, count, T = x["table"], x["lens"], x["free"], x["count"], x["tokens"]
    B, P = table.shape
    col = torch.arange(P, device=table.device)[None]
    n = x["new"].clamp(min=0)
    ends = torch.cumsum(n, 0)
    # reserve: requests in order; one that does not fit the table, the pool or the token rows gets nothing
    fits = (lens + n <= P * PAGE) & (ends <= T)
    need = torch.where(fits, _ceil(lens + n) - _ceil(lens), torch.zeros_like(n))
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= count))
    first = _ceil(lens)[:, None]
    fresh = granted[:, None] & (col >= first) & (col < first + need[:, None])
    rank = (upto - need)[:, None] + col - first
    table.copy_(torch.where(fresh, free[(count - 1 - rank).clamp(0, free.numel() - 1)], table))
    t = torch.arange(T, device=table.device)
    seq = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    pos = lens[seq] + t - (ends - n)[seq]
    on = granted[seq] & (t < ends[-1])
    page = table[seq, (pos // PAGE).clamp(0, P - 1)]
    gone = torch.full_like(pos, -1)
    slots, positions = torch.where(on, page * PAGE + pos % PAGE, gone), torch.where(on, pos, gone)
    lens.add_(torch.where(granted, n, torch.zeros_like(n)))
    count.sub_(torch.where(granted, need, torch.zeros_like(need)).sum())
    # release: every sequence back to the tokens it keeps, its other pages back on the stack
    keep = torch.minimum(x["keep"], lens)
    drop = _ceil(lens) - _ceil(keep)
    before = torch.cumsum(drop, 0) - drop
    gives = (col >= _ceil(keep)[:, None]) & (col < _ceil(lens)[:, None])
    rank = (before[:, None] + col - _ceil(keep)[:, None])[gives]
    free[(count + drop.sum() - 1 - rank).long()] = table[gives]
    lens.copy_(keep)
    count.add_(drop.sum())
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    return {"slots": slots.int(), "positions": positions.int(), "cu_new": cu.int(), "granted": granted.int(), "table": table, "lens": lens, "free": free, "count": count}


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(x):
    c = x["case"]
    if own:
        return _own(x)
    return {"decode": _plain_decode, "rope": _plain_rope, "append": _plain_append, "gather": _plain_gather, "pages": _plain_pages}[c["kind"]](x)


def _own(x):
    import mlc_decode_amd as M
    c, kind = x["case"], x["case"]["kind"]
    cache = x.get("kv")
    if "latent" in x:
        cache = (M.Fp4KVCache if x["scale"].dtype == torch.uint8 else M.Fp8KVCache)(x["latent"], x["scale"], x["rope"])
    if kind == "decode":
        causal = c["s_q"] > 1
        if c["auto"]:
            return M.mla_decode_with_kvcache(x["q"], cache, x["table"], x["lens"], causal=causal)
        if c["topk"]:
            return M.flash_mla_with_kvcache(x["q"], cache, None, None, D_V, *x["sched"], indices=x["indices"])
        return M.flash_mla_with_kvcache(x["q"], cache, x["table"], x["lens"], D_V, *x["sched"], causal=causal)
    if kind == "rope":
        return M.apply_rope(x["x"], x["positions"], M.Rope(x["freqs"], c["layout"], x["amp"]), first=c["first"])
    if kind == "append":
        M.kv_append_slots(x["kv_new"], cache, x["slots"], x["positions"], M.Rope(x["freqs"], c["layout"], x["amp"]), x.get("q_pe"), x.get("q"))
        out = {"cache": cache if "kv" in x else M.kv_gather(cache, x["all"])}
        if c["heads"]:
            out["q"] = x["q"]
        return out
    if kind == "gather":
        return M.kv_gather(cache, x["slots"])
    pool = M.PagePool(x["free"], x["count"])
    r = M.reserve_pages(pool, x["table"], x["lens"], x["new"], x["tokens"])
    M.release_pages(pool, x["table"], x["lens"], x["keep"])
    return {"slots": r.slots, "positions": r.positions, "cu_new": r.cu_new, "granted": r.granted, "table": x["table"], "lens": x["lens"], "free": x["free"], "count": x["count"]}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------
def exact(c, seed):
    """What run() returns, from the definitions in 64 bits; None where whole numbers come back."""
    if c["kind"] == "pages":
        return None
    x = prepare(c, seed)
    dev = "cuda"
    byte = torch.arange(256, device=dev)
    mag = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=dev) / 2
    nibble = torch.cat([mag, -mag])
    pairs = torch.stack([nibble[byte % 16], nibble[byte // 16]], -1)  # a byte's two values

    def token(page, row):  # pool rows in 64 bits
        if "kv" in x:
            return x["kv"][page, row, 0].double()
        codes, rope = x["latent"][page, row], x["rope"][page, row].double()
        if x["scale"].dtype == torch.uint8:
            size = torch.exp2(x["scale"][page, row].double() - 127).repeat_interleave(32, -1)
            latent = pairs[codes.long()].reshape(*codes.shape[:-1], D_V)
        else:
            size = x["scale"][page, :, row].double().repeat_interleave(128, -1)
            latent = codes.view(torch.float8_e4m3fn).double()
        return torch.cat([latent * size, rope], -1)

    def turn(v, positions):  # a complex product with amp * exp(2 pi i pos f)
        w = torch.remainder(positions.double()[:, None] * x["freqs"], 1.0) * (2 * math.pi)
        z = torch.polar(torch.full_like(w, x["amp"]), w)
        while z.dim() < v.dim():
            z = z.unsqueeze(1)
        h = v.shape[-1] // 2
        a, b = (v[..., ::2], v[..., 1::2]) if c["layout"] == "interleaved" else (v[..., :h], v[..., h:])
        y = torch.complex(a.double(), b.double()) * z
        y = torch.stack([y.real, y.imag], -1)
        y = y.flatten(-2) if c["layout"] == "interleaved" else y.transpose(-1, -2).flatten(-2)
        hold = positions < 0
        y[hold] = v[hold].double()
        return y

    def snap(v, bits):  # rows rounded to what the 4- or 8-bit cache holds of them
        if bits == 4:
            v = v.double().reshape(-1, 16, 32)
            top, grid, odd = 6.0, mag, torch.arange(8, device=dev) % 2
        else:
            v = v.double().reshape(-1, 4, 128)
            grid = byte[:127].to(torch.uint8).view(torch.float8_e4m3fn).double()
            top, odd = 448.0, byte[:127] % 2
        peak = v.abs().amax(-1, keepdim=True)
        k = torch.ceil(torch.log2(peak.clamp(min=1e-300) / top)) + 1
        for _ in range(3):  # log2 is off by less than that
            k = torch.where(peak <= top * torch.exp2(k - 1), k - 1, k)
        size = torch.where(peak == 0, torch.ones_like(k), torch.exp2(k.clamp(-126, 127)))
        u = v.abs() / size
        hi = torch.searchsorted(grid, u.contiguous()).clamp(1, grid.numel() - 1)
        lo = hi - 1
        up = (grid[hi] - u < u - grid[lo]) | ((grid[hi] - u == u - grid[lo]) & (odd[hi] == 0))
        return (torch.copysign(torch.where(up, grid[hi], grid[lo]), v) * size).reshape(-1, D_V)

    if c["kind"] == "rope":
        y = x["x"].double()
        a, b = c["first"], c["first"] + c["rot"]
        y[..., a:b] = turn(x["x"][..., a:b], x["positions"])
        return y
    if c["kind"] == "gather":
        slot = x["slots"].long()
        y = token(slot.clamp(min=0) // PAGE, slot.clamp(min=0) % PAGE)
        y[slot < 0] = 0
        return y
    if c["kind"] == "append":
        on = x["slots"] >= 0
        every = x["all"].long()
        rows = torch.cat([token(e // PAGE, e % PAGE) for e in every.split(65536)])
        new = x["kv_new"][on]
        latent = new[:, :D_V].double() if "kv" in x else snap(new[:, :D_V], 4 if c["cache"] == "fp4" else 8)
        rows[x["slots"][on].long()] = torch.cat([latent, turn(new[:, D_V:], x["positions"][on])], -1)
        out = {"cache": rows.reshape(x["kv"].shape) if "kv" in x else rows}
        if c["heads"]:
            q = x["q"].double()
            q[on, :, D_V:] = turn(x["q_pe"][on], x["positions"][on])
            out["q"] = q
        return out
    outs, lses = [], []
    for b in range(c["batch"]):
        if c["topk"]:
            at, n = x["indices"][b, 0].long(), c["topk"]
        else:
            n = int(x["lens"][b])
            t = torch.arange(n, device=dev)
            at = x["table"][b].long()[t // PAGE] * PAGE + t % PAGE
        k = token(at // PAGE, at % PAGE)
        o = torch.zeros(c["s_q"], c["heads"], D_V, dtype=torch.float64, device=dev)
        lse = torch.full((c["heads"], c["s_q"]), -math.inf, dtype=torch.float64, device=dev)
        for i in range(c["s_q"]):
            see = n - (c["s_q"] - 1 - i)
            if see > 0:
                s = x["q"][b, i].double() @ k[:see].T / math.sqrt(D_QK)
                lse[:, i] = torch.logsumexp(s, -1)
                o[i] = torch.softmax(s, -1) @ k[:see, :D_V]
        outs.append(o)
        lses.append(lse)
    return torch.stack(outs), torch.stack(lses)
