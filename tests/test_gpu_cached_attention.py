"""GPU tests of decode attention over bf16 and e4m3 caches, with and without shared prefixes, against the oracle in 64
bits.

Tolerance of an output (relative 2-norm over a slot's heads): the query, the probabilities and the output are each rounded
to bf16 once, at most 2^-8 a value and about 0.4 of that in the mean square.  The last enters as it is; the others enter
scores of unit variance and sums of many terms, where such errors average: 3 * 0.4 * 2^-8 = 0.0047, so 0.01 holds with room
for single slots.  A new key's code may differ by a step where the fp32 norm and rotation land on the other side of a tie."""
import importlib

import pytest
import torch

from conftest import PKG_NAME, rel_l2
from oracle import serving_oracle as so

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
TOL, EPS = 1e-2, 1e-6
pytestmark = pytest.mark.gpu


def make(N, nh, kv, hd, T, fp8, seed, rd=None):
    g = torch.Generator().manual_seed(seed)
    rd = hd // 4 if rd is None else rd
    x = dict(proj=torch.randn(N, (2 * nh + 2 * kv) * hd, generator=g).to(BF), qn=(0.1 * torch.randn(hd, generator=g)).to(BF),
             kn=(0.1 * torch.randn(hd, generator=g)).to(BF), rd=rd,
             inv=1.0 / (10000.0 ** (torch.arange(0, rd, 2).float() / max(rd, 1))))
    for side in ("k", "v"):
        x[side], x[side + "e"] = so.pack(torch.randn(N, kv, T, hd, generator=g).double() * (2 if side == "v" else 1), side, fp8)
    return x


def on_gpu(gdn, x, dev):
    return gdn.KVCache(x["k"].to(dev), x["v"].to(dev), *(None if x[e] is None else x[e].to(dev) for e in ("ke", "ve")))


def run(gdn, dev, x, pos, nh, prefix=None, **kw):
    c = on_gpu(gdn, x, dev)
    out = gdn.cached_decode_attention(x["proj"].to(dev), torch.tensor(pos, device=dev), x["qn"].to(dev), x["kn"].to(dev),
                                      x["inv"].to(dev), c, nh, x["rd"], EPS, prefix=prefix, **kw)
    return out, c


def reference(x, pos, nh, fp8, prefix=None):
    k, v = so.unpack(x["k"], x["ke"], "k"), so.unpack(x["v"], x["ve"], "v")
    out, raw = so.decode_attention(x["proj"], pos, x["qn"], x["kn"], x["inv"], k, v, nh, x["rd"], EPS, fp8, prefix)
    return out, raw, k, v


def check_cache(c, x, k, v, raw, at, T):
    """The new tokens are where they belong, as the cache rounds them; nothing else changed."""
    gk = so.unpack(c.k.cpu(), None if c.k_exp is None else c.k_exp.cpu(), "k")
    gv = so.unpack(c.v.cpu(), None if c.v_exp is None else c.v_exp.cpu(), "v")
    assert torch.equal(torch.nan_to_num(gv, nan=1e9), torch.nan_to_num(v, nan=1e9))
    for n, t in enumerate(at):
        if 0 <= t < T:
            ulp = 2.0 ** -4 if c.k.dtype == F8 else 2.0 ** -8   # half a step, relative
            # ... and below e4m3's smallest normal, half of 2^-9 of the row's scale (at most max / 224)
            small = raw[n].abs().amax(-1, keepdim=True) * (2.0 ** -10 / 224 if c.k.dtype == F8 else 0)
            assert ((gk[n, :, t] - raw[n]).abs() <= (raw[n].abs() * ulp + small) * 1.001 + 1e-6).all()
            assert rel_l2(gk[n, :, t], k[n, :, t]) <= 1e-3
            gk[n, :, t] = k[n, :, t]
    assert torch.equal(torch.nan_to_num(gk, nan=1e9), torch.nan_to_num(k, nan=1e9))


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("nh,kv,hd,pos,T,rd", [
    (24, 4, 256, [0, 63, 64, 255, 256, 1300], 1344, 64),
    (4, 2, 64, [5, 17, 9], 64, 16),
    (8, 1, 128, [700, 3], 704, 128),
    (2, 2, 128, [511, 515], 576, 0),
    (16, 1, 64, [130], 192, 32),     # 16 heads a group
    (7, 1, 128, [1, 2, 300], 320, 64),
    (9, 3, 256, [2047, 100], 2048, 128),
])
def test_against_oracle(gdn, dev, fp8, nh, kv, hd, pos, T, rd):
    x = make(len(pos), nh, kv, hd, T, fp8, hd + nh + T, rd)
    out, c = run(gdn, dev, x, pos, nh)
    ref, raw, k, v = reference(x, pos, nh, fp8)
    for n in range(len(pos)):
        assert rel_l2(out[n], ref[n]) <= TOL, pos[n]
    check_cache(c, x, k, v, raw, pos, T)


@pytest.mark.parametrize("fp8", [True, False])
def test_edges_and_garbage(gdn, dev, fp8):
    """Positions at the edges of a block, a wave's turn and a range, with NaN codes, infinite and NaN scales in everything
    behind each slot's position; a negative position writes nothing and gives zero; one behind the cache writes nothing and
    attends to all of it."""
    nh, kv, hd, T = 6, 1, 128, 640
    pos = [0, 1, 15, 16, 62, 63, 64, 127, 128, 255, 256, 319, 511, 639, -1, 700]
    N = len(pos)
    x = make(N, nh, kv, hd, T, fp8, 5)
    for side in ("k", "v"):
        at = so.table(T, hd, side, fp8)
        b = x[side].view(torch.uint8 if fp8 else torch.int16).view(N, kv, -1)
        for n, p in enumerate(pos[:-1]):
            b[n][:, at[max(p, 0):].reshape(-1)] = 0x7f if fp8 else 0x7f80 if n % 2 else 0x7fc0
            if fp8:
                x[side + "e"][n, :, max(p, 0):] = 255 if n % 2 else 254
    out, c = run(gdn, dev, x, pos, nh)
    ref, raw, k, v = reference(x, pos, nh, fp8)
    assert not out.isnan().any()
    assert torch.equal(out[N - 2].cpu().float(), torch.zeros(nh * hd))
    for n in range(N):
        if pos[n] >= 0:
            assert rel_l2(out[n], ref[n]) <= TOL, pos[n]
    for got, was in ((c.k, x["k"]), (c.v, x["v"])):
        view = lambda y: y.cpu().view(torch.uint8 if fp8 else torch.int16)  # noqa: E731
        assert torch.equal(view(got)[-2:], view(was)[-2:])


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("nh,kv,hd,of,plen,own,T,Tp", [
    (24, 4, 256, [0] * 5, [700], [1, 64, 65, 300, 2], 320, 704),
    (4, 2, 64, [0, 1, 0, -1, 1, 2, 0], [64, 130, 1], [3, 9, 1, 70, 64, 20, 128], 128, 192),
    (16, 1, 128, [1] * 9 + [0] * 3, [65, 257], [5] * 12, 64, 320),      # many rows: several tiles
    (8, 8, 64, [0, 3, 0], [0, 64], [7, 8, 9], 64, 64),                  # an empty prefix; a number that names none
    (6, 1, 256, [0, 0], [5000], [4, 200], 256, 5056),
])
def test_shared_prefix(gdn, dev, fp8, nh, kv, hd, of, plen, own, T, Tp):
    N, P = len(of), len(plen)
    x = make(N, nh, kv, hd, T, fp8, nh + Tp)
    px = make(P, nh, kv, hd, Tp, fp8, nh + Tp + 1)
    for side in ("k", "v"):  # what lies behind a prefix's end may be anything
        b = px[side].view(torch.uint8 if fp8 else torch.int16).view(P, kv, -1)
        at = so.table(Tp, hd, side, fp8)
        for r, n in enumerate(plen):
            b[r][:, at[n:].reshape(-1)] = 0x7f if fp8 else 0x7fc0
    full = [plen[r] if 0 <= r < P else 0 for r in of]
    pos = [a + b - 1 for a, b in zip(full, own)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    prefix = gdn.SharedPrefix(on_gpu(gdn, px, dev), i32(plen), i32(of))
    out, c = run(gdn, dev, x, pos, nh, prefix)
    pk, pv = so.unpack(px["k"], px["ke"], "k"), so.unpack(px["v"], px["ve"], "v")
    ref, raw, k, v = reference(x, pos, nh, fp8, (pk, pv, plen, of))
    for n in range(N):
        assert rel_l2(out[n], ref[n]) <= TOL, (n, of[n])
    check_cache(c, x, k, v, raw, [o - 1 for o in own], T)
    if P == 1 and 64 % 64 == plen[0] % 64:
        return
    # the same tokens without sharing: each slot's prefix copied in front of its own
    if min(full) >= 0 and fp8 is False and hd == 64:
        T2 = (max(full) + max(own) + 63) // 64 * 64
        y = dict(x)
        for side, p, o in (("k", pk, so.unpack(x["k"], None, "k")), ("v", pv, so.unpack(x["v"], None, "v"))):
            z = torch.zeros(N, kv, T2, hd, dtype=torch.float64)
            for n in range(N):
                if full[n]:
                    z[n, :, :full[n]] = p[of[n], :, :full[n]]
                z[n, :, full[n]:full[n] + own[n]] = o[n, :, :own[n]]
            y[side], y[side + "e"] = so.pack(z, side, fp8)
        out2, _ = run(gdn, dev, y, pos, nh)
        assert rel_l2(out, out2) <= TOL


def test_prefix_positions(gdn, dev):
    """A slot whose position lies inside its prefix attends to the prefix alone and writes nothing; a negative one gives
    zero; lengths outside the prefix cache are cut to it."""
    nh, kv, hd = 4, 2, 64
    x, px = make(4, nh, kv, hd, 64, True, 1), make(2, nh, kv, hd, 128, True, 2)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    prefix = gdn.SharedPrefix(on_gpu(gdn, px, dev), i32([100, 999]), i32([0, 0, 1, 1]))
    pos = [40, -1, 130, 127]
    out, c = run(gdn, dev, x, pos, nh, prefix)
    p = (so.unpack(px["k"], px["ke"], "k"), so.unpack(px["v"], px["ve"], "v"), [100, 128], [0, 0, 1, 1])
    ref, raw, k, v = reference(x, pos, nh, True, p)
    assert not out[1].any()
    for n in (0, 2, 3):
        assert rel_l2(out[n], ref[n]) <= TOL
    check_cache(c, x, k, v, raw, [-1, -1, 2, -1], 64)


def test_infinite_values(gdn, dev):
    """An infinity in the new token's value row (bf16 cache) stays one in its output column, the other columns match."""
    nh, kv, hd, T = 6, 1, 128, 128
    pos = [0, 5, 62, 63, 64, 100]
    x = make(len(pos), nh, kv, hd, T, False, 3)
    x["proj"][:, (2 * nh + kv) * hd + 3] = float("inf")
    x["proj"][:, :2 * nh * hd].view(-1, nh, 2, hd)[:, :, 1, 3] = 0.5
    out, _ = run(gdn, dev, x, pos, nh)
    ref, *_ = reference(x, pos, nh, False)
    out, ref = out.cpu().view(len(pos), nh, hd), ref.view(len(pos), nh, hd)
    assert (out[:, :, 3] == float("inf")).all()
    keep = torch.arange(hd) != 3
    for n in range(len(pos)):
        assert rel_l2(out[n][:, keep], ref[n][:, keep]) <= TOL


def test_far_angles(gdn, dev):
    """Rotary at positions where a float's angle is off by radians: the keys match the oracle's."""
    nh, kv, hd, T = 2, 1, 64, 64
    plen = 64 * 15625  # a prefix of a million tokens
    x = make(2, nh, kv, hd, T, False, 4, rd=64)
    pc = gdn.KVCache.empty(1, kv, hd, plen, dtype=BF, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pos = [plen, plen + 37]
    out, c = run(gdn, dev, x, pos, nh, gdn.SharedPrefix(pc, i32([plen]), i32([0, 0])))
    pk = torch.zeros(1, kv, plen, hd, dtype=torch.float64)
    ref, raw, k, v = reference(x, pos, nh, False, (pk, pk, [plen], [0, 0]))
    check_cache(c, x, k, v, raw, [0, 37], T)


def test_from_partials(gdn, dev):
    """Fed the projection's split-K partials: the same output and cache, bit for bit."""
    cb = importlib.import_module(PKG_NAME + ".cb_engine")
    nh, kv, hd, H, N = 24, 4, 256, 5120, 7
    x = make(N, nh, kv, hd, 512, True, 6)
    g = torch.Generator().manual_seed(60)
    h = torch.randn(N, H, generator=g).to(BF).to(dev)
    w = cb.PackedWeight((0.05 * torch.randn((2 * nh + 2 * kv) * hd, H, generator=g)).to(BF).to(dev))
    pos = torch.randint(0, 512, (N,), generator=g).to(dev)
    part = cb.decode_linear_partial(h, w)
    assert part.splits > 1
    got = []
    for proj in (cb.decode_linear(h, w), part):
        c = on_gpu(gdn, x, dev)
        o = gdn.cached_decode_attention(proj, pos, x["qn"].to(dev), x["kn"].to(dev), x["inv"].to(dev), c, nh, x["rd"], EPS)
        got.append((o, c))
    assert torch.equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_matches_the_bf16_slot_cache(gdn, dev):
    """On the same history, a bf16 KVCache and gqa_decode_attention's transposed cache give the same attention."""
    cb = importlib.import_module(PKG_NAME + ".cb_engine")
    nh, kv, hd, T = 8, 2, 128, 512
    pos = [0, 100, 300, 511]
    x = make(4, nh, kv, hd, T, False, 8)
    out, _ = run(gdn, dev, x, pos, nh)
    kt = so.unpack(x["k"], None, "k").to(BF).transpose(2, 3).contiguous().to(dev)
    v = so.unpack(x["v"], None, "v").to(BF).to(dev)
    old = cb.gqa_decode_attention(x["proj"].to(dev), torch.tensor(pos, device=dev), x["qn"].to(dev), x["kn"].to(dev),
                                  x["inv"].to(dev), kt, v, nh, kv, hd, x["rd"], EPS)
    assert rel_l2(out, old) <= TOL


def test_graph_replays_as_positions_advance(gdn, dev):
    """A captured step with a kept workspace, replayed as positions and the prefix assignment change in place, equals eager
    steps on a copy of the cache; other eager work runs between."""
    nh, kv, hd, T, N = 8, 2, 128, 256, 5
    x, px = make(N, nh, kv, hd, T, True, 9), make(2, nh, kv, hd, 192, True, 10)
    c1, c2, pc = on_gpu(gdn, x, dev), on_gpu(gdn, x, dev), on_gpu(gdn, px, dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    plen, of = i32([150, 64]), i32([0, 1, 0, -1, 0])
    pos = torch.tensor([150, 70, 160, 3, 350], device=dev)
    prefix = gdn.SharedPrefix(pc, plen, of)
    proj = x["proj"].to(dev)
    par = (x["qn"].to(dev), x["kn"].to(dev), x["inv"].to(dev))
    work = gdn.cached_attn_workspace(c1, nh, prefix)
    graph = gdn.GDNDecodeGraph(lambda: gdn.cached_decode_attention(proj, pos, *par, c1, nh, x["rd"], EPS, work=work, prefix=prefix),
                               device=dev)
    for i in range(4):
        proj.copy_(torch.randn(proj.shape, generator=torch.Generator().manual_seed(i)))
        got = graph.replay().clone()
        torch.cuda.synchronize()
        want = gdn.cached_decode_attention(proj, pos, *par, c2, nh, x["rd"], EPS, prefix=prefix)
        assert torch.equal(got, want)
        assert torch.equal(c1.k_exp, c2.k_exp) or i == 0
        pos += 1
        if i == 1:
            of.copy_(i32([1, 1, 0, 0, -1]))
            pos += 90
    assert torch.equal(got, want)


def test_other_stream_and_strided_projection(gdn, dev):
    nh, kv, hd, T, N = 4, 2, 64, 128, 3
    x = make(N, nh, kv, hd, T, True, 12)
    pos = [3, 64, 127]
    want, _ = run(gdn, dev, x, pos, nh)
    wide = torch.zeros(N, x["proj"].shape[1] + 24, dtype=BF, device=dev)
    wide[:, 8:-16] = x["proj"].to(dev)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        y = dict(x, proj=wide[:, 8:-16])
        got, _ = run(gdn, dev, y, pos, nh)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("N,P", [(400, 300), (1024, 1024), (1024, 3)])
def test_many_slots_and_prefixes(gdn, dev, N, P):
    """As many slots and prefixes as a call takes; prefixes without slots, slots without a prefix, empty prefixes."""
    nh, kv, hd, T, Tp = 2, 1, 64, 64, 128
    g = torch.Generator().manual_seed(N + P)
    x, px = make(N, nh, kv, hd, T, True, N), make(P, nh, kv, hd, Tp, True, P)
    plen = torch.randint(0, Tp + 1, (P,), generator=g)
    of = torch.randint(-1, P + 1, (N,), generator=g)
    full = torch.where((of >= 0) & (of < P), plen[of.clamp(0, P - 1)], 0)
    pos = full + torch.randint(0, T, (N,), generator=g)
    prefix = gdn.SharedPrefix(on_gpu(gdn, px, dev), plen.int().to(dev), of.int().to(dev))
    out, c = run(gdn, dev, x, pos.tolist(), nh, prefix)
    p = (so.unpack(px["k"], px["ke"], "k"), so.unpack(px["v"], px["ve"], "v"), plen.tolist(), of.tolist())
    ref, raw, k, v = reference(x, pos.tolist(), nh, True, p)
    for n in range(N):
        assert rel_l2(out[n], ref[n]) <= TOL, n
    check_cache(c, x, k, v, raw, (pos - full).tolist(), T)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -60, 30.0])
def test_queries_of_any_size(gdn, dev, fp8, scale):
    """A query of zeros attends to all tokens alike; tiny ones nearly so; rows between the slots differ by many powers of
    two (the query's norm weights are -1 + scale; half of the slots' rows are scaled below the norm's eps)."""
    nh, kv, hd, T, N = 6, 1, 128, 192, 4
    x = make(N, nh, kv, hd, T, fp8, 15)
    x["qn"] = torch.full((hd,), scale - 1.0).to(BF) if scale in (0.0, 30.0) else x["qn"]
    if scale == 30.0:  # scores of a few units all the same
        x["proj"][:, :2 * nh * hd] *= 2.0 ** -18
    if 0 < scale < 1:
        x["proj"][::2, :2 * nh * hd] *= scale
    pos = [0, 70, 128, 191]
    out, _ = run(gdn, dev, x, pos, nh)
    ref, _, _, _ = reference(x, pos, nh, fp8)
    for n in range(N):
        assert rel_l2(out[n], ref[n]) <= TOL, pos[n]


def test_one_projection_for_all_slots_and_no_slots(gdn, dev):
    nh, kv, hd, T, N = 4, 2, 64, 64, 5
    x = make(N, nh, kv, hd, T, False, 14)
    x["proj"] = x["proj"][:1].expand(N, -1)
    pos = [0, 3, 9, 40, 63]
    c = on_gpu(gdn, x, dev)
    args = (torch.tensor(pos, device=dev), x["qn"].to(dev), x["kn"].to(dev), x["inv"].to(dev))
    out = gdn.cached_decode_attention(x["proj"][:1].to(dev).expand(N, -1), *args, c, nh, x["rd"], EPS)
    ref, _, _, _ = reference(x, pos, nh, False)
    for n in range(N):
        assert rel_l2(out[n], ref[n]) <= TOL, pos[n]
    none = gdn.KVCache(c.k[:0], c.v[:0])
    assert gdn.cached_decode_attention(x["proj"][:0].to(dev), args[0][:0], *args[1:], none, nh, x["rd"], EPS).shape == (0, nh * hd)


def test_refusals(gdn, dev):
    nh, kv, hd, N = 4, 2, 64, 2
    x = make(N, nh, kv, hd, 64, True, 13)
    c = on_gpu(gdn, x, dev)
    a = dict(proj=x["proj"].to(dev), pos=torch.zeros(N, dtype=torch.int64, device=dev), q_norm=x["qn"].to(dev), k_norm=x["kn"].to(dev),
             inv_freq=x["inv"].to(dev), cache=c, n_heads=nh, rotary_dim=16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    b16 = gdn.KVCache.empty(1, kv, hd, 64, dtype=BF, device=dev)
    for kw, err in ((dict(proj=a["proj"][:, :-1]), "proj"), (dict(pos=a["pos"].int()), "pos"), (dict(n_heads=8), "proj"),
                    (dict(q_norm=x["qn"][:5].to(dev)), "q_norm"), (dict(inv_freq=x["inv"][:3].to(dev)), "inv_freq"),
                    (dict(prefix=gdn.SharedPrefix(b16, i32([1]), i32([0, 0]))), "prefix cache"),
                    (dict(prefix=gdn.SharedPrefix(c, i32([1]), i32([0, 0]))), "length"),
                    (dict(prefix=gdn.SharedPrefix(c, i32([1, 1]), i32([0, 0]).long())), "prefix.of"),
                    (dict(work=torch.zeros(16)), "work")):
        with pytest.raises(ValueError, match=err):
            gdn.cached_decode_attention(**{**a, **kw})
    with pytest.raises(gdn.GDNError, match="workspace"):
        gdn.cached_decode_attention(**a, work=torch.zeros(16, dtype=torch.uint8, device=dev))
