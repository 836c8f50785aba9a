"""GPU tests of cached decode attention where a wave works through several blocks of a range, and of its precision, against
the formula in 64 bits on what the cache holds after the call.

Tolerance of an output (relative 2-norm over a slot's heads): rounding it to bf16 puts a value off by at most half a step, in
the mean square 2^-7 / sqrt(12) = 0.00226 of a value at the lower end of its binade (less above it).  What else there is lies
far below: probabilities in two bf16 parts, the first cut off, are off by at most 2^-15, about 2^-17 in the mean square, a query
in such parts the same, times scores of a few units, and the sums are fp32.  0.0024 leaves 6 % for the chance of a few hundred
values; probabilities and a query rounded to bf16 once give 0.0031."""
import math

import pytest
import torch

from conftest import rel_l2
from oracle import serving_oracle as so

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
TOL, EPS = 2.4e-3, 1e-6
pytestmark = pytest.mark.gpu


def cache_of(gdn, dev, R, kv, hd, T, fp8, seed, rise=0):
    """A cache written everywhere; rise: the keys' scale goes up by 2^rise over a row, so that the largest scores come late
    (below 0: early)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    c = gdn.KVCache.empty(R, kv, hd, T, F8 if fp8 else BF, dev)
    T = c.length
    up = (torch.arange(T, device=dev) * (rise / T)).round()  # whole powers of two
    up = up - up.max().clamp_min(0) + 1 if rise else up
    for side, x, e in (("k", c.k, c.k_exp), ("v", c.v, c.v_exp)):
        for r in range(R):
            y = torch.randn(x.shape[1:], generator=g, device=dev)
            if fp8:
                x[r] = (100 * y).clamp_(-448, 448).to(F8)
            else:
                y = y.view(kv, -1, 64 * hd)
                x[r] = (y * torch.exp2(up.view(-1, 64)[:, 0])[:, None] if side == "k" else y).to(BF)
        if fp8:
            e.copy_(torch.randint(119, 122, e.shape, generator=g, device=dev))
            if side == "k":
                e.copy_((e.float() + up).to(torch.uint8))
    return c


def values(c, side, r, n):
    """The first n tokens of row r of a cache's side: float64 [kv, n, hd] on its device."""
    x, e = (c.k, c.k_exp) if side == "k" else (c.v, c.v_exp)
    hd, fp8 = c.head_dim, c.k.dtype == F8
    blocks = (n + 63) // 64
    one = so.table(64, hd, side, fp8).to(x.device)  # of one block
    y = x[r, :, :blocks].float().double()[..., one.reshape(-1)].reshape(x.shape[1], blocks * 64, hd)[:, :n]
    return y if e is None else y * torch.exp2(e[r, :, :n].double() - 127)[..., None]


def reference(x, pos, nh, c, prefix=None):
    """The gated output [N, nh hd] in float64 from the cache as it stands after the call."""
    N, kv, hd, T = c.k.shape[0], c.k.shape[1], c.head_dim, c.length
    out = []
    for n in range(N):
        qg = x["proj"][n].double()[:2 * nh * hd].view(nh, 2 * hd)
        q = so.rms_rope(qg[:, :hd], x["qn"], pos[n], x["inv"], x["rd"], EPS).view(kv, nh // kv, hd).to(c.k.device)
        r = int(prefix.of[n]) if prefix is not None else -1
        plen = int(prefix.length[r]) if r >= 0 else 0
        own = min(pos[n] - plen + 1, T)
        k, v = values(c, "k", n, own), values(c, "v", n, own)
        if r >= 0:
            k, v = (torch.cat((values(prefix.cache, s, r, plen), y), 1) for s, y in (("k", k), ("v", v)))
        p = torch.softmax(q @ k.transpose(1, 2).contiguous() / math.sqrt(hd), -1)
        out.append(((p @ v).reshape(nh, hd).cpu() * torch.sigmoid(qg[:, hd:])).reshape(-1))
    return torch.stack(out)


def inputs(N, nh, kv, hd, seed, rd=None, qn=None):
    g = torch.Generator().manual_seed(seed)
    rd = hd // 4 if rd is None else rd
    return dict(proj=torch.randn(N, (2 * nh + 2 * kv) * hd, generator=g).to(BF),
                qn=(0.1 * torch.randn(hd, generator=g)).to(BF) if qn is None else torch.full((hd,), qn).to(BF),
                kn=(0.1 * torch.randn(hd, generator=g)).to(BF), rd=rd, inv=1.0 / (10000.0 ** (torch.arange(0, rd, 2).float() / max(rd, 1))))


def call(gdn, dev, x, pos, nh, c, prefix=None):
    return gdn.cached_decode_attention(x["proj"].to(dev), torch.tensor(pos, device=dev), x["qn"].to(dev), x["kn"].to(dev),
                                       x["inv"].to(dev), c, nh, x["rd"], EPS, prefix=prefix)


def blocks_a_wave(kv, G, own, plens=(), of=()):
    """(of slots' own tokens, of prefixes): the most blocks that a wave takes, by the plan's rule."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    wgs = 256 // kv + 1
    tiles = [up(sum(r == p for r in of) * G, 32) for p in range(len(plens))]
    each = up(sum(up(n, 64) for n in own) + sum(2 * t * up(n, 64) for t, n in zip(tiles, plens)), wgs)
    pre, own = up(each, 8), up(up(each, 4) if each >= 48 else each, 4)
    return own, pre


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("rise", [0, 4, -4])
@pytest.mark.parametrize("nh,kv,hd,own,waves", [
    (16, 8, 64, [4001, 7777, 12345, 20000, 65, 9999], 7),
    (8, 8, 128, [5000, 3, 8191, 8192, 8193], 4),
    (12, 4, 256, [6500, 9001, 7000], 2),
    (64, 32, 64, [13500, 15001], 4),                 # 50 blocks a workgroup: cut into four
])
def test_several_blocks_a_wave(gdn, dev, fp8, rise, nh, kv, hd, own, waves):
    """Running maxima that change from block to block, the next block's keys, values and scales, masks behind full blocks."""
    assert blocks_a_wave(kv, nh // kv, own)[0] == waves
    x = inputs(len(own), nh, kv, hd, hd + len(own))
    c = cache_of(gdn, dev, len(own), kv, hd, max(own), fp8, nh + rise, rise)
    pos = [n - 1 for n in own]
    out = call(gdn, dev, x, pos, nh, c)
    ref = reference(x, pos, nh, c)
    for n in range(len(own)):
        assert rel_l2(out[n], ref[n]) <= TOL, pos[n]


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("rise", [0, 4, -4])
@pytest.mark.parametrize("nh,kv,hd,of,plen,waves", [
    (64, 16, 64, [0, 1] * 8, [5000, 3001], 3),
    (32, 32, 64, [0] * 24 + [1, -1, 2], [4033, 700, 64], 4),
    (48, 16, 128, [0] * 30, [3333], 3),              # three tiles
    (24, 12, 256, [1, 0, 1, 1, 1, 0], [2500, 9000], 3),
])
def test_several_blocks_a_wave_of_a_prefix(gdn, dev, fp8, rise, nh, kv, hd, of, plen, waves):
    own = [1 + 37 * n % 300 for n in range(len(of))]
    assert blocks_a_wave(kv, nh // kv, own, plen, of)[1] == waves
    x = inputs(len(of), nh, kv, hd, hd + len(of))
    c = cache_of(gdn, dev, len(of), kv, hd, 300, fp8, nh)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    prefix = gdn.SharedPrefix(cache_of(gdn, dev, len(plen), kv, hd, max(plen), fp8, nh + 1, rise), i32(plen), i32(of))
    pos = [o - 1 + (plen[r] if r >= 0 else 0) for o, r in zip(own, of)]
    out = call(gdn, dev, x, pos, nh, c, prefix)
    ref = reference(x, pos, nh, c, prefix)
    for n in range(len(of)):
        assert rel_l2(out[n], ref[n]) <= TOL, (n, of[n])


@pytest.mark.parametrize("fp8", [True, False])
def test_a_million_shared_tokens(gdn, dev, fp8):
    """Far positions' angles, and sums over a million tokens."""
    nh, kv, hd, plen = 4, 1, 64, 64 * 15625 - 5
    x = inputs(2, nh, kv, hd, 4, rd=64)
    c = cache_of(gdn, dev, 2, kv, hd, 64, fp8, 1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    prefix = gdn.SharedPrefix(cache_of(gdn, dev, 1, kv, hd, plen, fp8, 2), i32([plen]), i32([0, 0]))
    pos = [plen, plen + 37]
    out = call(gdn, dev, x, pos, nh, c, prefix)
    ref = reference(x, pos, nh, c, prefix)
    for n in range(2):
        assert rel_l2(out[n], ref[n]) <= TOL, n


@pytest.mark.parametrize("behind", [False, True])
@pytest.mark.parametrize("fp8", [True, False])
def test_large_scores(gdn, dev, fp8, behind):
    """Scores of about 400 (a query norm weight of 128), and several tokens within one unit of each other at the top: a
    query of 11 bits (2^-11 / sqrt(12) of a value in the mean square) has scores off by 0.015, and so the probabilities by more
    than 1 %.  In two bf16 parts: 128 * 2^-17.7 = 0.0006."""
    nh, kv, hd, T, N = 3, 3, 128, 8192, 4
    x = inputs(N, nh, kv, hd, 21, qn=127.0)
    c = cache_of(gdn, dev, N, kv, hd, T, fp8, 22)
    if behind:  # the same history as a prefix for each slot
        p = gdn.KVCache(*(None if y is None else y.clone() for y in c))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        prefix, c = gdn.SharedPrefix(p, i32([T] * N), i32(range(N))), gdn.KVCache.empty(N, kv, hd, 64, F8 if fp8 else BF, dev)
        pos = [T] * N
    else:
        p, prefix, pos = c, None, [T - 1] * N
    # of the highest 40 scores the largest group within one unit is made the top: what lies above it gets another token's key
    for n in range(N):
        k = values(p, "k", n, T)
        qg = x["proj"][n].double()[:2 * nh * hd].view(nh, 2 * hd)
        q = so.rms_rope(qg[:, :hd], x["qn"], pos[n], x["inv"], x["rd"], EPS).to(dev)
        s = (q[:, None] * k).sum(-1) / math.sqrt(hd)
        at = so.table(T, hd, "k", fp8).to(dev)
        for h in range(kv):
            low = int((s[h].abs()).argmin())
            high = (s[h] > s[h].sort(descending=True).values[40]).nonzero()[:, 0]
            order = high[s[h][high].argsort()]
            top = max(range(len(order)), key=lambda i: int(((s[h][order] <= s[h][order[i]]) & (s[h][order] > s[h][order[i]] - 1)).sum()))
            flat = (p.k.view(torch.uint8) if fp8 else p.k)[n, h].view(-1)
            for t in order[top + 1:].tolist():
                flat[at[t]] = flat[at[low]].clone()
                if fp8:
                    p.k_exp[n, h, t] = p.k_exp[n, h, low]
    out = call(gdn, dev, x, pos, nh, c, prefix)
    ref = reference(x, pos, nh, c, prefix)
    for n in range(N):
        assert rel_l2(out[n], ref[n]) <= TOL, n
