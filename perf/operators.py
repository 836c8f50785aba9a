"""The serving operators around a decode step's cache and its logits, as cases that can be timed and checked.

``listed()`` names the cases, ``draw`` gives more of the same ranges, ``prepare`` makes what a program
holds before the call, ``run`` is one pass (``own``: through the package's entry points; else in plain
torch operations), ``exact`` the same results in 64 bits, ``work`` the bytes and flops of one pass.

Kinds:
  cache    a batch's new prompt tokens into the slots' cache rows, and the slots' whole context back out as bf16
  decode   a decode step's attention over per-slot caches: norms, rotary, cache write, softmax, gate
  prefix   the same for slots that continue a prefix they share
  sample   one token per row of logits: temperature, top-k, top-p, min-p, given random numbers

A cache keeps the 64 tokens of a block in the order in which the attention kernels read them (``_k_at``, ``_v_at``).
In e4m3 each (token, kv head) row has one power-of-two scale 2^e, kept as the byte e + 127: e is the smallest integer
with max |x| <= 448 * 2^e over the row's finite values (at least -126; 0 for a row of zeros).
"""
import math

import numpy as np
import torch

own = False

PKG = "910b_e2e_accleration_by_codex_amd"
EPS = 1e-6
BF, F8, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8
CACHE = {"fp8": F8, "bf16": BF}
DTYPES = {"bf16": BF, "fp16": torch.float16, "fp32": torch.float32}


def _pkg():
    import importlib
    return importlib.import_module(PKG)


def listed():
    return [
        # the next prefill chunk of one prompt (517 tokens behind 2048) at the 27B attention shape: stored, and the
        # context read back for the chunk's own attention
        dict(name="cache_fp8_continue_517", kind="cache", cache="fp8", dtype="bf16", prompts=1, lo=517, hi=517, start=2048,
             kv=4, hd=256, heads_first=True),
        # a batch of 16 fresh prompts admitted at once
        dict(name="cache_fp8_16prompts", kind="cache", cache="fp8", dtype="bf16", prompts=16, lo=200, hi=1500, start=0,
             kv=4, hd=256, heads_first=True),
        # one request in flight, a short context: launches and host time
        dict(name="decode_fp8_1slot", kind="decode", cache="fp8", slots=1, heads=24, kv=4, hd=256, rd=64, ctx_lo=353,
             ctx_hi=353),
        # the continuous-batching step, 16 slots with contexts of 512 to 4096
        dict(name="decode_fp8_16", kind="decode", cache="fp8", slots=16, heads=24, kv=4, hd=256, rd=64, ctx_lo=512,
             ctx_hi=4096),
        # the same on a cache that keeps bf16
        dict(name="decode_bf16_16", kind="decode", cache="bf16", slots=16, heads=24, kv=4, hd=256, rd=64, ctx_lo=512,
             ctx_hi=4096),
        # long documents in every slot
        dict(name="decode_fp8_16_long", kind="decode", cache="fp8", slots=16, heads=24, kv=4, hd=256, rd=64, ctx_lo=16384,
             ctx_hi=32768),
        # four agents behind a short system prompt, a small model's heads
        dict(name="prefix_bf16_4", kind="prefix", cache="bf16", slots=4, heads=4, kv=2, hd=64, rd=16, prefixes=1,
             prefix_len=353, ctx_lo=1, ctx_hi=130),
        # 16 slots behind one tool description of 8192 tokens
        dict(name="prefix_fp8_16", kind="prefix", cache="fp8", slots=16, heads=24, kv=4, hd=256, rd=64, prefixes=1,
             prefix_len=8192, ctx_lo=64, ctx_hi=1024),
        # 64 slots over two long documents: the product is large enough to be bound by the matrix units
        dict(name="prefix_fp8_64", kind="prefix", cache="fp8", slots=64, heads=24, kv=4, hd=256, rd=64, prefixes=2,
             prefix_len=16384, ctx_lo=64, ctx_hi=512),
        # one request's next token, every filter on
        dict(name="sample_1", kind="sample", dtype="bf16", rows=1, vocab=248320, mode="all", masked=0.0),
        # a step of 16 slots, each request with parameters of its own (greedy ones among them)
        dict(name="sample_16", kind="sample", dtype="bf16", rows=16, vocab=248320, mode="mixed", masked=0.0),
        # 64 slots' logits in fp32 under a grammar that forbids a third of the vocabulary
        dict(name="sample_64_fp32", kind="sample", dtype="fp32", rows=64, vocab=151936, mode="mixed", masked=0.33),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "prefix", "sample"])
    if kind == "sample":
        rows = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=rows, vocab=_log_int(rng, 1000, 248320),
                    mode=rng.choice(["plain", "all", "mixed", "greedy"]), masked=rng.choice([0.0, 0.0, 0.33, 0.99]))
    hd, kv, cache = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice(["fp8", "fp8", "bf16"])
    if kind == "cache":
        prompts, hi, start = _log_int(rng, 1, 16), _log_int(rng, 1, 1500), rng.choice([0, 1, _log_int(rng, 2, 4096)])
        return dict(kind=kind, cache=cache, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), prompts=prompts,
                    lo=max(1, hi // rng.choice([1, 2, 7])), hi=hi, start=start, kv=kv, hd=hd, heads_first=rng.random() < 0.5)
    heads, rd = kv * rng.choice([1, 2, 3, 4, 6, 7, 8, 16]), rng.choice([0, hd // 4, hd // 4, hd // 2, hd])
    if kind == "decode":
        slots = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(64, min(32768, 16 * 32768 * 4 * 256 // (slots * kv * hd) // (2 if cache == "bf16" else 1))))
        return dict(kind=kind, cache=cache, slots=slots, heads=heads, kv=kv, hd=hd, rd=rd, ctx_lo=max(1, hi // rng.choice([1, 2, 8])),
                    ctx_hi=hi)
    slots, hi = _log_int(rng, 2, 64), _log_int(rng, 1, 1024)
    most = min(16384, 64 * 24 * 256 * 16384 // (slots * heads * hd))
    return dict(kind=kind, cache=cache, slots=slots, heads=heads, kv=kv, hd=hd, rd=rd, prefixes=rng.choice([1, 1, 2, 3]),
                prefix_len=_log_int(rng, 16, most), ctx_lo=max(1, hi // rng.choice([1, 2, 8])), ctx_hi=hi)


# ---- the cache's blocks ---------------------------------------------------------------------------
def _k_at(t, d, hd, fp8):
    """Where token t's dim d lies in a K row of T * hd values: blocks of 64 tokens, in them 16-byte pieces of e values
    of one token, token 16 a + 4 i + r at [piece / 4][i][piece % 4][4 a + r]."""
    e = 16 if fp8 else 8
    piece, x = d // e, t % 64
    a, i, r = x // 16, x // 4 % 4, x % 4
    return t // 64 * (64 * hd) + (((piece // 4 * 4 + i) * 4 + piece % 4) * 16 + 4 * a + r) * e + d % e


def _v_at(t, d, hd, fp8):
    """Where token t's dim d lies in a V row: blocks of 64 tokens, in them 16 dims at a time.  e4m3: [dim][16 a + x];
    bf16: token 16 a + 8 u + x at [u][dim][a][x]."""
    x, m = t % 64, d % 16
    if fp8:
        return t // 64 * (64 * hd) + d // 16 * 1024 + m * 64 + x
    return t // 64 * (64 * hd) + d // 16 * 1024 + ((x // 8 % 2 * 16 + m) * 4 + x // 16) * 8 + x % 8


def _k_rows(c, hd):
    """A K cache [R, kv, T / 64, 64 hd] as [R, kv, T, hd]."""
    R, kv, B = c.shape[:3]
    e = 16 if c.dtype == F8 else 8
    x = c.view(U8 if c.dtype == F8 else c.dtype).view(R, kv, B, hd // (4 * e), 4, 4, 4, 4, e)  # [piece / 4][i][piece % 4][a][r][e]
    return x.permute(0, 1, 2, 6, 4, 7, 3, 5, 8).reshape(R, kv, B * 64, hd).view(c.dtype)


def _v_rows(c, hd):
    """A V cache [R, kv, T / 64, 64 hd] as [R, kv, T, hd]."""
    R, kv, B = c.shape[:3]
    if c.dtype == F8:
        x = c.view(U8).view(R, kv, B, hd // 16, 16, 64).permute(0, 1, 2, 5, 3, 4)
    else:
        x = c.view(R, kv, B, hd // 16, 2, 16, 4, 8).permute(0, 1, 2, 6, 4, 7, 3, 5)
    return x.reshape(R, kv, B * 64, hd).view(c.dtype)


def _scales(e):
    return torch.exp2(e.float() - 127)


def _quantised(x):
    """fp32 rows [..., hd] -> e4m3 codes and the bytes of their scales."""
    finite = x.isfinite()
    top = x.abs().where(finite, torch.zeros_like(x)).amax(-1)
    m, ex = torch.frexp(top)
    e = torch.where(top > 0, (ex - 8 - (m <= 0.875).int()).clamp_min(-126), torch.zeros_like(ex))
    y = torch.ldexp(x, -e[..., None]).where(finite, torch.full_like(x, float("nan")))
    return y.to(F8), (e + 127).to(U8)


# ---- inputs ---------------------------------------------------------------------------------------
class _Rand:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda:0")
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def n(self, *shape, scale=1.0, dtype=BF):
        return (torch.randn(*shape, generator=self.g, device=self.dev) * scale).to(dtype)

    def u(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.g, device=self.dev) * (hi - lo) + lo

    def i(self, lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=self.g, device=self.dev)


def _spread(n, lo, hi):
    """n whole numbers over [lo, hi], in a mixed order: a batch's lengths belong to the case, not to the seed."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    return [v[i * step % n] for i in range(n)]


def _new_cache(r, rows, kv, hd, length, kind):
    """A cache that has been written everywhere: rows as a model's normalised keys and its values have them."""
    B = -(-length // 64)
    shape = (rows, kv, B, 64 * hd)
    if kind == "bf16":
        return dict(k=r.n(*shape), v=r.n(*shape), ks=None, vs=None)
    x = {}
    for name in ("k", "v"):
        # a row's largest of hd values is near 2.8 sigma: with the scale's exponent -7 it lies between 224 and 448
        x[name] = torch.empty(shape, dtype=F8, device=r.dev)
        for i in range(rows):
            x[name][i] = r.n(*shape[1:], scale=100.0, dtype=torch.float32).clamp_(-448, 448).to(F8)
        x[name + "s"] = r.i(118, 121, rows, kv, B * 64).to(U8)
    return x


def prepare(case, seed):
    r = _Rand(seed)
    kind = case["kind"]
    if kind == "sample":
        n, V = case["rows"], case["vocab"]
        # a step's logits: a broad body and a few hundred tokens that stand out
        l = r.n(n, V, scale=2.0, dtype=torch.float32)
        l += 6.0 * (r.u(n, V) < 200.0 / V)
        if case["masked"]:
            l.masked_fill_(r.u(n, V) < case["masked"], float("-inf"))
        s = dict(case=case, logits=l.to(DTYPES[case["dtype"]]), u=r.u(n), temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
        if case["mode"] == "all":
            s.update(temperature=0.75, top_k=50, top_p=0.95, min_p=0.02)
        elif case["mode"] == "greedy":
            s.update(temperature=0.0)
        elif case["mode"] == "mixed":  # per request: a quarter each greedy, unfiltered, nucleus only, everything
            q = torch.arange(n, device=r.dev) % 4
            s.update(temperature=torch.where(q == 3, 0.0, r.u(n, lo=0.5, hi=1.5)),
                     top_k=torch.where(q == 2, r.i(2, 100, n), 0).int(), top_p=torch.where(q > 0, r.u(n, lo=0.7, hi=0.99), 1.0),
                     min_p=torch.where(q == 2, r.u(n, lo=0.0, hi=0.1), 0.0))
        return s
    kv, hd = case["kv"], case["hd"]
    if kind == "cache":
        n = case["prompts"]
        lens, starts = _spread(n, case["lo"], case["hi"]), _spread(n, case["start"] // 2, case["start"])
        rows = [2 * i + 1 for i in range(n)]  # a serving batch's slots: the prompts sit in every other row
        cu, ctx = [0], [0]
        for a, b in zip(lens, starts):
            cu.append(cu[-1] + a)
            ctx.append(ctx[-1] + a + b)
        dt = DTYPES[case["dtype"]]
        # as a prefill leaves them: [tokens, kv, hd], or a view of a model cache's [kv, tokens, hd]
        new = [r.n(kv, cu[-1], hd, dtype=dt).transpose(0, 1) if case["heads_first"] else r.n(cu[-1], kv, hd, dtype=dt)
               for _ in range(2)]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=r.dev)  # noqa: E731
        return dict(case=case, new_k=new[0], new_v=new[1], rows=i32(rows), cu=i32(cu), start=i32(starts), ctx=i32(ctx),
                    total=ctx[-1], **_new_cache(r, 2 * n + 1, kv, hd, max(a + b for a, b in zip(lens, starts)), case["cache"]))
    n, nh, rd = case["slots"], case["heads"], case["rd"]
    s = dict(case=case, proj=r.n(n, (2 * nh + 2 * kv) * hd), qn=r.n(hd, scale=0.1), kn=r.n(hd, scale=0.1),
             inv=1.0 / (10000.0 ** (torch.arange(0, rd, 2, device=r.dev, dtype=torch.float32) / max(rd, 1))),
             **_new_cache(r, n, kv, hd, case["ctx_hi"] + 16, case["cache"]))
    pos = torch.tensor(_spread(n, case["ctx_lo"], case["ctx_hi"]), device=r.dev) - 1
    if kind == "prefix":
        p = case["prefixes"]
        c = _new_cache(r, p, kv, hd, case["prefix_len"], case["cache"])
        s.update(pk=c["k"], pv=c["v"], pks=c["ks"], pvs=c["vs"],
                 plen=torch.tensor(_prefix_lens(case), dtype=torch.int32, device=r.dev),
                 pof=(torch.arange(n, device=r.dev) % p).int())
        pos = pos + s["plen"].long()[s["pof"].long()]
    s["pos"] = pos
    return s


def _prefix_lens(case):
    return [max(1, case["prefix_len"] - 37 * i) for i in range(case["prefixes"])]


# ---- run ------------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s)
    if kind == "sample":
        return _plain_sample(s)
    if kind == "cache":
        return _plain_cache(s)
    return _plain_attention(s)


def _own(s):
    p, case = _pkg(), s["case"]
    if case["kind"] == "sample":
        return p.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    cache = p.KVCache(s["k"], s["v"], s["ks"], s["vs"])
    if case["kind"] == "cache":
        p.kv_cache_store(cache, s["new_k"], s["new_v"], s["rows"], s["cu"], s["start"])
        return p.kv_cache_load(cache, s["rows"], s["ctx"], total_tokens=s["total"])
    prefix = p.SharedPrefix(p.KVCache(s["pk"], s["pv"], s["pks"], s["pvs"]), s["plen"], s["pof"]) if "pof" in s else None
    if "work" not in s:  # a program keeps its workspace
        s["work"] = p.cached_attn_workspace(cache, case["heads"], prefix)
    o = p.cached_decode_attention(s["proj"], s["pos"], s["qn"], s["kn"], s["inv"], cache, case["heads"], case["rd"], EPS,
                                  work=s["work"], prefix=prefix)
    return dict(out=o, k=s["k"], v=s["v"], ks=s["ks"], vs=s["vs"])


def _put(c, e, at, rows, heads, t, x):
    """x [m, kv, hd] fp32 -> one side of the cache (c: its tensor, e: its scales' bytes or None), token t[m] of row rows[m];
    at: _k_at or _v_at."""
    hd = x.shape[-1]
    fp8 = c.dtype == F8
    place = at(t[:, None, None], torch.arange(hd, device=x.device), hd, fp8)
    flat = (c.view(U8) if fp8 else c).view(c.shape[0], c.shape[1], -1)
    if fp8:
        code, ex = _quantised(x)
        e[rows[:, None], heads, t[:, None]] = ex
        x = code.view(U8)
    flat[rows[:, None, None], heads[:, None], place] = x.to(flat.dtype)


def _get(c, e, at, rows, heads, t, hd):
    """Token t[m] of row rows[m] of one side of the cache: bf16 [m, kv, hd]."""
    place = at(t[:, None, None], torch.arange(hd, device=t.device), hd, c.dtype == F8)
    flat = (c.view(U8) if c.dtype == F8 else c).view(c.shape[0], c.shape[1], -1)
    x = flat[rows[:, None, None], heads[:, None], place].view(c.dtype).float()
    if e is not None:
        x = x * _scales(e[rows[:, None], heads, t[:, None]])[..., None]
    return x.to(BF)


def _plain_cache(s):
    case = s["case"]
    kv, hd = case["kv"], case["hd"]
    heads = torch.arange(kv, device=s["cu"].device)
    i = torch.arange(s["new_k"].shape[0], device=s["cu"].device)
    q = torch.searchsorted(s["cu"], i, right=True) - 1
    rows, t = s["rows"][q].long(), i - s["cu"][q] + s["start"][q]
    _put(s["k"], s["ks"], _k_at, rows, heads, t, s["new_k"].float())
    _put(s["v"], s["vs"], _v_at, rows, heads, t, s["new_v"].float())
    i = torch.arange(s["total"], device=i.device)
    q = torch.searchsorted(s["ctx"], i, right=True) - 1
    rows, t = s["rows"][q].long(), i - s["ctx"][q]
    return _get(s["k"], s["ks"], _k_at, rows, heads, t, hd), _get(s["v"], s["vs"], _v_at, rows, heads, t, hd)


def _plain_attention(s):
    case = s["case"]
    n, nh, kv, hd, rd = case["slots"], case["heads"], case["kv"], case["hd"], case["rd"]
    x, pos = s["proj"].float(), s["pos"]
    heads = torch.arange(kv, device=x.device)

    def normed(y, w):
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * (1 + w.float())

    ang = pos.double()[:, None, None] * s["inv"].double()
    cos, sin = ang.cos().float(), ang.sin().float()

    def turned(y):
        a, b = y[..., :rd // 2], y[..., rd // 2:rd]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., rd:]), -1)

    qg = x[:, :2 * nh * hd].view(n, nh, 2 * hd)
    q, gate = turned(normed(qg[..., :hd], s["qn"])), qg[..., hd:]
    k, v = x[:, 2 * nh * hd:].view(n, 2, kv, hd).unbind(1)
    own_pos = pos - s["plen"].long()[s["pof"].long()] if "pof" in s else pos
    rows = torch.arange(n, device=x.device)
    _put(s["k"], s["ks"], _k_at, rows, heads, own_pos, turned(normed(k, s["kn"])))
    _put(s["v"], s["vs"], _v_at, rows, heads, own_pos, v)

    def sides(k, ks, v, vs):
        k, v = _k_rows(k, hd).float(), _v_rows(v, hd).float()
        return (k, v) if ks is None else (k * _scales(ks)[..., None], v * _scales(vs)[..., None])

    k, v = sides(s["k"], s["ks"], s["v"], s["vs"])
    T, G = k.shape[2], nh // kv
    q = q.view(n, kv, G, hd) * hd ** -0.5
    sc = q @ k.transpose(-1, -2).contiguous()
    sc = sc.masked_fill(torch.arange(T, device=x.device) > own_pos[:, None, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    if "pof" in s:  # every slot's heads against every prefix, the others' masked
        pk, pv = sides(s["pk"], s["pks"], s["pv"], s["pvs"])
        P, L = pk.shape[0], pk.shape[2]
        allq = q.transpose(0, 1).reshape(1, kv, n * G, hd)
        ps = (allq @ pk.transpose(-1, -2).contiguous()).view(P, kv, n, G, L)
        mine = (s["pof"] == torch.arange(P, device=x.device)[:, None])[:, None, :, None, None]
        inside = (torch.arange(L, device=x.device) < s["plen"][:, None])[:, None, None, None, :]
        ps = ps.masked_fill(~(mine & inside), float("-inf"))
        top = torch.maximum(top, ps.amax((0, 4)).transpose(0, 1)[..., None])
        ps = (ps - top.transpose(0, 1)).exp()
    sc = (sc - top).exp()
    o, total = sc @ v, sc.sum(-1, keepdim=True)
    if "pof" in s:
        o = o + (ps.view(P, kv, n * G, L) @ pv).sum(0).view(kv, n, G, hd).transpose(0, 1)
        total = total + ps.sum((0, 4)).transpose(0, 1)[..., None]
    o = (o / total).view(n, nh, hd) / (1 + (-gate).exp())
    return dict(out=o.reshape(n, nh * hd).to(BF), k=s["k"], v=s["v"], ks=s["ks"], vs=s["vs"])


def _plain_sample(s):
    n, V = s["logits"].shape
    dev = s["logits"].device
    col = lambda v: torch.as_tensor(v, device=dev, dtype=torch.float64).expand(n)[:, None]  # noqa: E731
    t, k, p, m, u = (col(s[x]) for x in ("temperature", "top_k", "top_p", "min_p", "u"))
    l = s["logits"].double()
    l = l.where(~l.isnan(), torch.full_like(l, float("-inf")))
    top = l.amax(-1, keepdim=True)
    none = top[:, 0] == float("-inf")
    greedy = (l == top).int().argmax(-1)
    w = ((l - top) / t.where(t > 0, torch.ones_like(t))).exp()
    w = w.where(l != top, torch.ones_like(w))
    by, at = torch.sort(l, dim=-1, descending=True, stable=True)
    w = w.gather(-1, at)
    rank = torch.arange(V, device=dev)
    keep = (by > float("-inf")) & ((rank < k) | (k <= 0))
    w = w * keep
    before = w.cumsum(-1) - w
    keep &= (before < p * w.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)
    keep &= (w >= m) | (rank == 0)
    w = torch.zeros_like(l).scatter(-1, at, w * keep)
    c = w.cumsum(-1)
    drawn = (c <= u * c[:, -1:]).sum(-1).clamp_max(V - 1)
    token = torch.where(t[:, 0] > 0, drawn, greedy)
    return token.where(~none, torch.full_like(token, -1))


# ---- 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "cache":
        return _exact_cache(s)
    return _exact_attention(s)


def _exact_rounded(x, kind):
    """What a cache of this kind holds for rows x (float64): (values, codes, bytes of the scales)."""
    if kind == "bf16":
        y = x.to(BF).double()
        return y, y, None
    e = torch.zeros(x.shape[:-1], dtype=torch.float64, device=x.device)
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top / 448)).clamp_min(-126)
    e = e - (top <= 448 * torch.exp2(e - 1)).double() + (top > 448 * torch.exp2(e)).double()  # the logarithm's last bit
    e = e.where(top > 0, torch.zeros_like(e)).clamp_min(-126)
    y = x * torch.exp2(-e)[..., None]
    # the nearest multiple of the step at |y|: 2^(exponent - 3), and 2^-9 below 2^-6; ties to even
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    code = torch.round(y / step) * step
    return code * torch.exp2(e)[..., None], code, (e + 127).to(U8)


def _exact_cache(s):
    """Sequence by sequence: the rows that were there, then the new ones as the cache rounds them."""
    case = s["case"]
    kv, hd = case["kv"], case["hd"]
    old_k, old_v = _exact_sides(s, "", hd)
    cu, start, rows = s["cu"].tolist(), s["start"].tolist(), s["rows"].tolist()
    out = []
    for old, new in ((old_k, s["new_k"]), (old_v, s["new_v"])):
        parts = []
        for i, row in enumerate(rows):
            parts.append(old[row, :, :start[i]].transpose(0, 1))
            parts.append(_exact_rounded(new[cu[i]:cu[i + 1]].double(), case["cache"])[0])
        out.append(torch.cat(parts))
    return tuple(out)


def _exact_sides(s, p, hd):
    """The values [R, kv, T, hd] (float64) that a cache holds, token by token and dim by dim from the layout's formula."""
    out = []
    for name, at in (("k", _k_at), ("v", _v_at)):
        c, e = s[p + name], s[p + name + "s"]
        R, kv, B = c.shape[:3]
        place = at(torch.arange(B * 64, device=c.device)[:, None], torch.arange(hd, device=c.device), hd, c.dtype == F8)
        flat = (c.view(U8) if c.dtype == F8 else c).view(R, kv, -1)
        x = torch.empty(R, kv, B * 64, hd, dtype=torch.float64, device=c.device)
        for i in range(R):
            x[i] = flat[i][:, place.reshape(-1)].view(c.dtype).double().view(kv, B * 64, hd)
            if e is not None:
                x[i] *= torch.exp2(e[i].double() - 127)[..., None]
        out.append(x)
    return out


def _exact_attention(s):
    case = s["case"]
    n, nh, kv, hd, rd = case["slots"], case["heads"], case["kv"], case["hd"], case["rd"]
    G = nh // kv
    proj, inv = s["proj"].double(), s["inv"].double()

    def prepared(y, w, p):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * (1.0 + w.double())
        z = torch.view_as_complex(torch.stack((y[:, :rd // 2], y[:, rd // 2:rd]), -1).contiguous())
        z = z * torch.polar(torch.ones_like(inv), inv * p)
        return torch.cat((z.real, z.imag, y[:, rd:]), -1)

    out = torch.empty(n, nh * hd, dtype=torch.float64, device=proj.device)
    heads = torch.arange(kv, device=proj.device)
    dims = torch.arange(hd, device=proj.device)
    fp8 = case["cache"] == "fp8"
    # the state after the step: what it held, with the new token's values in place
    codes = {name: s[name].double() for name in ("k", "v")}
    bytes_ = {name: None if s[name + "s"] is None else s[name + "s"].clone() for name in ("k", "v")}
    prefix = _exact_sides(s, "p", hd) if "pof" in s else None
    pos = s["pos"].tolist()
    for i in range(n):
        one = {name: s[name][i:i + 1] if s[name] is not None else None for name in ("k", "v", "ks", "vs")}
        sides = _exact_sides(one, "", hd)
        r = int(s["pof"][i]) if "pof" in s else -1
        before = int(s["plen"][r]) if r >= 0 else 0
        t = pos[i] - before
        row = proj[i]
        new = {"k": prepared(row[2 * nh * hd:(2 * nh + kv) * hd].view(kv, hd), s["kn"], pos[i]),
               "v": row[(2 * nh + kv) * hd:].view(kv, hd)}
        for j, (name, at) in enumerate((("k", _k_at), ("v", _v_at))):
            value, code, ex = _exact_rounded(new[name], case["cache"])
            sides[j][0, :, t] = value
            codes[name].view(n, kv, -1)[i][heads[:, None], at(t, dims, hd, fp8)] = code
            if fp8:
                bytes_[name][i, :, t] = ex
        qg = row[:2 * nh * hd].view(nh, 2 * hd)
        q = prepared(qg[:, :hd], s["qn"], pos[i]).view(kv, G, hd)
        k, v = sides[0][0, :, :t + 1], sides[1][0, :, :t + 1]
        if r >= 0:
            k, v = torch.cat((prefix[0][r, :, :before], k), 1), torch.cat((prefix[1][r, :, :before], v), 1)
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd), -1)
        out[i] = (torch.matmul(p, v).reshape(nh, hd) * torch.sigmoid(qg[:, hd:])).reshape(-1)
    return dict(out=out, k=codes["k"], v=codes["v"], ks=bytes_["k"], vs=bytes_["v"])


def _exact_sample(s):
    """Row by row on the host, sums in extended precision."""
    n = s["logits"].shape[0]
    par = {x: torch.as_tensor(s[x], dtype=torch.float64).cpu().expand(n).numpy() for x in ("temperature", "top_k", "top_p", "min_p", "u")}
    logits = s["logits"].float().cpu().numpy()
    out = []
    for i in range(n):
        t, k, p, m, u = (par[x][i] for x in ("temperature", "top_k", "top_p", "min_p", "u"))
        l = np.where(np.isnan(logits[i]), -np.inf, logits[i]).astype(np.longdouble)
        best = int(np.argmax(l))
        if l[best] == -np.inf or t <= 0:
            out.append(-1 if l[best] == -np.inf else best)
            continue
        order = np.argsort(-l, kind="stable")
        order = order[l[order] > -np.inf]
        if k > 0:
            order = order[:int(k)]
        w = np.exp((l[order] - l[best]) / np.longdouble(t))
        count = len(order)
        if p < 1:
            count = max(1, int(np.searchsorted(np.cumsum(w), np.longdouble(p) * w.sum(), side="left")) + 1)
        order, w = order[:count], w[:count]
        order, w = order[(w >= m) | (order == best)], w[(w >= m) | (order == best)]
        by_index = np.argsort(order)
        c = np.cumsum(w[by_index])
        at = min(int(np.searchsorted(c, np.longdouble(u) * c[-1], side="right")), len(c) - 1)
        out.append(int(order[by_index][at]))
    return torch.tensor(out, device=s["logits"].device)


# ---- work -----------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * (4 if case["dtype"] == "fp32" else 2) + 16 * case["rows"], flops=4 * n)
    kv, hd = case["kv"], case["hd"]
    row = 2 * kv * (hd + 1 if case["cache"] == "fp8" else 2 * hd)  # bytes of one token's K and V in the cache
    if kind == "cache":
        new, old = sum(_spread(case["prompts"], case["lo"], case["hi"])), sum(_spread(case["prompts"], case["start"] // 2, case["start"]))
        size = 4 if case["dtype"] == "fp32" else 2
        return dict(bytes=new * (2 * kv * hd * size + row) + (new + old) * (row + 4 * kv * hd), flops=2 * kv * hd * (2 * new + old))
    n, nh = case["slots"], case["heads"]
    own_ctx = sum(_spread(n, case["ctx_lo"], case["ctx_hi"]))
    shared = _prefix_lens(case) if kind == "prefix" else [0]
    seen = own_ctx + sum(shared[i % len(shared)] for i in range(n))
    return dict(bytes=(own_ctx + sum(shared)) * row + n * (2 * nh + 2 * kv) * hd * 2 + n * nh * hd * 2 + n * row,
                flops=4 * seen * nh * hd)
