"""GPU tests of the KV cache: packed prompts stored (bf16, and quantised to e4m3) and loaded, against the oracle's
quantisation and layout, exactly: codes, scales and what no sequence covers."""
import pytest
import torch

from oracle import serving_oracle as so

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
pytestmark = pytest.mark.gpu


def bits(c):
    return c.cpu().view(torch.uint8 if c.dtype == F8 else torch.int16)


def filled(gdn, R, kv, hd, T, dtype, dev, seed=0):
    """A cache whose every byte is something."""
    g = torch.Generator().manual_seed(seed)
    c = gdn.KVCache.empty(R, kv, hd, T, dtype=dtype, device=dev)
    for x in (c.k, c.v):
        b = x.view(torch.uint8) if dtype == F8 else x.view(torch.int16)
        b.copy_(torch.randint(0, 100, b.shape, generator=g))
    if dtype == F8:
        c.k_exp.copy_(torch.randint(100, 130, c.k_exp.shape, generator=g))
        c.v_exp.copy_(torch.randint(100, 130, c.v_exp.shape, generator=g))
    return c


def expect(c, k, v, rows, cu, start):
    """The cache's tensors after a store, from the oracle (c: before, moved to the CPU)."""
    R, kv, B, w = c.k.shape
    hd, T, fp8 = w // 64, B * 64, c.k.dtype == F8
    out = []
    for side, cache, exp, x in (("k", c.k, c.k_exp, k), ("v", c.v, c.v_exp, v)):
        vals = cache.cpu().float().reshape(R, kv, T * hd)
        exp = None if exp is None else exp.cpu().clone()
        at = so.table(T, hd, side, fp8)
        for s, r in enumerate(rows):
            if not 0 <= r < R:
                continue
            for i in range(cu[s], cu[s + 1]):
                t = start[s] + i - cu[s]
                if not 0 <= t < T:
                    continue
                y = x[i].cpu()
                if fp8:
                    q, e = so.quantise(y)
                    exp[r, :, t] = (e + 127).to(torch.uint8)
                    y = q * torch.exp2(-e.double())[:, None]
                vals[r][:, at[t]] = (y if fp8 else y.to(BF)).float()
        out += [vals.reshape(R, kv, B, w).to(c.k.dtype), exp]
    return out


def check(c, want):
    for got, w in zip((c.k, c.k_exp, c.v, c.v_exp), want):
        if w is None:
            assert got is None
        elif w.dtype == torch.uint8:
            assert torch.equal(got.cpu(), w)
        else:
            g = got.cpu()
            same = (bits(g) == bits(w)) | (g.float().isnan() & w.float().isnan()) | ((g.float() == 0) & (w.float() == 0))
            assert same.all()


CASES = [  # rows, lengths, starts, T
    ([0], [1], [0], 64),
    ([2, 0], [64, 65], [0, 0], 128),
    ([1, 2, 0], [3, 0, 130], [61, 5, 0], 192),       # an empty sequence; starts inside a block
    ([0, 1], [100, 17], [63, 127], 256),
    ([2, 2], [50, 50], [0, 50], 128),                # two pieces of one row that share a block
    ([0, -1, 5, 1], [40, 9, 9, 40], [-7, 0, 0, 100], 128),  # rows and positions outside the cache
]


@pytest.mark.parametrize("dtype", [F8, BF])
@pytest.mark.parametrize("hd,kv", [(64, 3), (128, 1), (256, 2)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_store_and_load(gdn, dev, dtype, hd, kv, case):
    rows, lens, starts, T = CASES[case]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    g = torch.Generator().manual_seed(hd + case)
    k, v = (torch.randn(cu[-1], kv, hd, generator=g).mul(torch.exp2(torch.randint(-20, 20, (cu[-1], kv, 1), generator=g).float())).to(BF)
            for _ in range(2))
    c = filled(gdn, 3, kv, hd, T, dtype, dev)
    want = expect(c, k, v, rows, cu, starts)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    gdn.kv_cache_store(c, k.to(dev), v.to(dev), i32(rows), i32(cu), i32(starts))
    check(c, want)
    gk, gv = gdn.kv_cache_load(c, i32(rows), i32(cu), i32(starts), total_tokens=cu[-1])
    for got, side, vals, exp in ((gk, "k", want[0], want[1]), (gv, "v", want[2], want[3])):
        full = so.unpack(vals, exp, side)
        ref = torch.zeros(cu[-1], kv, hd, dtype=torch.float64)
        for s, r in enumerate(rows):
            for i in range(cu[s], cu[s + 1]):
                t = starts[s] + i - cu[s]
                if 0 <= r < 3 and 0 <= t < T:
                    ref[i] = full[r, :, t]
        assert torch.equal(got.cpu().double(), ref)


@pytest.mark.parametrize("src", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("dtype", [F8, BF])
def test_store_input_types_and_strides(gdn, dev, src, dtype):
    """fp32 / fp16 / bf16 rows as a transposed view of [kv, tokens, hd], a slice at an odd offset (copied) and dense rows give
    the same cache; host lists and device tensors too."""
    kv, hd, n = 2, 128, 77
    g = torch.Generator().manual_seed(3)
    base = torch.randn(2, n, kv, hd, generator=g).to(src)
    got = []
    for form in range(3):
        x = base.to(dev)
        if form == 1:
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif form == 2:
            y = torch.zeros(2, n, kv, hd + 3, dtype=src, device=dev)
            y[..., 3:] = x
            x = y[..., 3:]
        c = filled(gdn, 2, kv, hd, 128, dtype, dev)
        if form:
            gdn.kv_cache_store(c, x[0], x[1], torch.tensor([1, 0]), [0, 40, n], torch.tensor([5, 0]))
        else:
            gdn.kv_cache_store(c, x[0], x[1], gdn.Rows([1, 0], 2, 2, dev), gdn.Varlen([0, 40, n], n, dev),
                               torch.tensor([5, 0], dtype=torch.int32, device=dev))
        got.append(c)
    check(got[0], expect(filled(gdn, 2, kv, hd, 128, dtype, dev), base[0], base[1], [1, 0], [0, 40, n], [5, 0]))
    for c in got[1:]:
        assert torch.equal(bits(c.k), bits(got[0].k)) and torch.equal(bits(c.v), bits(got[0].v))


def test_store_equal_lengths_many_sequences(gdn, dev):
    """More sequences than a wave looks at at a time, without cu_seqlens and start."""
    n, kv, hd = 150, 1, 64
    x = torch.randn(2, 3 * n, kv, hd, generator=torch.Generator().manual_seed(4)).to(BF)
    c = filled(gdn, n, kv, hd, 64, F8, dev)
    want = expect(c, x[0], x[1], list(range(n)), list(range(0, 3 * n + 1, 3)), [0] * n)
    gdn.kv_cache_store(c, x[0].to(dev), x[1].to(dev), list(range(n)))
    check(c, want)


def test_store_special_values(gdn, dev):
    """Rows of zeros, of subnormals, of the largest values, at the borders of a scale, with infinities and NaN; every bf16
    value against one fixed maximum."""
    hd = 64
    rows = [torch.zeros(hd)]
    for top in (448.0, 449.0, 450.0, 2.0 ** -126, 2.0 ** -133, 3.3e38, 1.75 * 2 ** -118, 1.0):
        r = torch.linspace(-1, 1, hd) * top
        r[0] = top
        rows.append(r)
    bad = torch.linspace(-3, 3, hd)
    bad[3], bad[4], bad[5] = float("inf"), float("-inf"), float("nan")
    rows += [bad, torch.full((hd,), float("nan")), torch.full((hd,), float("inf"))]
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(BF).float()
    every = every[every.abs() <= 448]
    every = every[: every.numel() // (hd - 1) * (hd - 1)].view(-1, hd - 1)
    rows = torch.stack(rows).to(BF)
    every = torch.cat((every, torch.full((every.shape[0], 1), 448.0)), 1).to(BF)
    x = torch.cat((rows, every))[:, None]
    c = filled(gdn, 1, 1, hd, x.shape[0], F8, dev)
    want = expect(c, x, x.flip(0), [0], [0, x.shape[0]], [0])
    gdn.kv_cache_store(c, x.to(dev), x.flip(0).contiguous().to(dev), [0])
    check(c, want)


def test_far_positions(gdn, dev):
    """A row of more than 2^31 bytes: its end is written and read where it belongs."""
    T, hd = 2 ** 23 + 64 * 8, 256  # 2^31 bytes and a little
    c = gdn.KVCache.empty(2, 1, hd, T, dtype=F8, device=dev)
    x = torch.randn(2, 70, 1, hd, generator=torch.Generator().manual_seed(5)).to(BF)
    gdn.kv_cache_store(c, x[0].to(dev), x[1].to(dev), [1], start=[T - 70])
    k, v = gdn.kv_cache_load(c, [1], [0, 70], start=[T - 70])
    for got, ref in ((k, x[0]), (v, x[1])):
        assert torch.equal(got.cpu().double(), so.quantise(ref)[0])
    assert not c.k[0].view(torch.uint8).any() and not c.v[0].view(torch.uint8).any()
    tail = gdn.KVCache(*(y[1:, :, -2:].contiguous() for y in (c.k, c.v)), *(y[1:, :, -128:].contiguous() for y in (c.k_exp, c.v_exp)))
    blank = gdn.KVCache.empty(1, 1, hd, 128, dtype=F8, device=dev)
    check(tail, expect(blank, x[0], x[1], [0], [0, 70], [58]))


@pytest.mark.parametrize("dtype", [F8, BF])
def test_graph_of_store_and_load(gdn, dev, dtype):
    """Store and load captured with their batch on the device, replayed on other rows, lengths and starts (a batch that
    ends before the packed tokens do: what lies behind is not written)."""
    kv, hd, T, total = 2, 64, 256, 150
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    rows, cu, start = i32([0, 2]), i32([0, 70, 150]), i32([0, 10])
    k, v = (torch.randn(total, kv, hd, generator=torch.Generator().manual_seed(i)).to(BF).to(dev) for i in range(2))
    c, d = (gdn.KVCache.empty(3, kv, hd, T, dtype=dtype, device=dev) for _ in range(2))

    def both():
        gdn.kv_cache_store(c, k, v, rows, cu, start)
        return gdn.kv_cache_load(c, rows, cu, start, total_tokens=total)
    graph = gdn.GDNDecodeGraph(both, device=dev)
    for t in (c.k, c.v, c.k_exp, c.v_exp):
        if t is not None:
            t.view(torch.uint8).fill_(127)
    for t in (d.k, d.v, d.k_exp, d.v_exp):
        if t is not None:
            t.view(torch.uint8).fill_(127)
    for r, n, s in (([0, 2], [70, 150], [0, 10]), ([1, 0], [1, 149], [255, 64]), ([2, 2], [33, 100], [100, 133])):
        rows.copy_(i32(r))
        cu.copy_(i32([0] + n))
        start.copy_(i32(s))
        k.copy_(torch.randn(k.shape, generator=torch.Generator().manual_seed(n[0])))
        gk, gv = graph.replay()
        torch.cuda.synchronize()
        gdn.kv_cache_store(d, k[:n[1]], v[:n[1]], r, [0] + n, s)
        for x, y in zip(c, d):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        wk, wv = gdn.kv_cache_load(d, r, [0] + n, s)
        assert torch.equal(gk[:n[1]], wk) and torch.equal(gv[:n[1]], wv)


def test_refusals(gdn, dev):
    c = gdn.KVCache.empty(2, 2, 64, 128, device=dev)
    x = torch.zeros(10, 2, 64, dtype=BF, device=dev)
    for args, err in (((c, x, x[:5], [0]), "one dtype"), ((c, x, x.float(), [0]), "one dtype"), ((c, x, x, [2]), "rows"),
                      ((c, x, x, [0], [0, 9]), "cu_seqlens"), ((c, x, x, [0, 1], [0, 11, 10]), "cu_seqlens"),
                      ((c, x, x, [0, 1, 0]), "divide"), ((c, x, x, [0], None, [0, 1]), "start"),
                      ((c, x, x, torch.zeros(1, dtype=torch.int64, device=dev)), "int32"),
                      ((c._replace(v=c.v[:1]), x, x, [0]), "contiguous tensors"),
                      ((c._replace(k_exp=None), x, x, [0]), "k_exp"), ((c._replace(k=c.k.transpose(0, 1)), x, x, [0]), "contiguous")):
        with pytest.raises(ValueError, match=err):
            gdn.kv_cache_store(*args)
    with pytest.raises(TypeError):
        gdn.kv_cache_store(c, x.double(), x.double(), [0])
    with pytest.raises(ValueError, match="total_tokens"):
        gdn.kv_cache_load(c, [0], None)
    gdn.kv_cache_store(c, x[:0], x[:0], [])
    k, v = gdn.kv_cache_load(c, [0], [0, 0])
    assert k.shape == v.shape == (0, 2, 64)
