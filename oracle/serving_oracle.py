"""CPU oracle of the serving operators in 64 bits: the KV cache's layout and quantisation, decode attention over it
(optionally behind a shared prefix), and sampling.  Written from the formulas in include/gdn_mi355x.h, element by element
where that is affordable."""
import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn


def quantise(x):
    """Rows x [..., hd] -> (values, exponent): code * 2^e with e the smallest integer >= -126 such that max|x| <= 448 * 2^e
    over the finite values (0 for zeros), codes to nearest even, what is not finite NaN.  All float64 / int."""
    x = x.double()
    fin = x.isfinite()
    top = torch.where(fin, x.abs(), 0.0).amax(-1)
    e = torch.full(top.shape, -126, dtype=torch.int64)
    for k in range(-126, 121):  # the smallest that holds
        e = torch.where(top > 448.0 * 2.0 ** k, k + 1, e)
    e = torch.where(top == 0, 0, e)
    y = torch.where(fin, x, 0.0) * torch.exp2(-e.double())[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    code = torch.round(y / step) * step  # torch.round: ties to even
    return torch.where(fin, code * torch.exp2(e.double())[..., None], float("nan")), e


def unit_of(t, d, hd, side, fp8):
    """Index of token t's dim d in a cache row of one kv head (values), from the header's formulas."""
    E = 16 if fp8 else 8
    b, x = divmod(t, 64)
    if side == "k":
        p = d // E
        a, i, r = x // 16, x // 4 % 4, x % 4
        unit, low = ((p // 4 * 4 + i) * 4 + p % 4) * 16 + 4 * a + r, d % E
    elif fp8:
        unit, low = d * 4 + x // 16, x % 16
    else:
        a, u = x // 16, x // 8 % 2
        unit, low = ((2 * (d // 16) + u) * 16 + d % 16) * 4 + a, x % 8
    return b * 64 * hd + unit * E + low


_tables = {}


def table(T, hd, side, fp8):
    """[T, hd] of unit_of."""
    key = (T, hd, side, fp8)
    if key not in _tables:
        one = torch.tensor([[unit_of(t, d, hd, side, fp8) for d in range(hd)] for t in range(64)])
        _tables[key] = torch.cat([one + b * 64 * hd for b in range(T // 64)])
    return _tables[key]


def unpack(c, exp, side):
    """A cache side [R, kv, T / 64, 64 hd] (with its exponent bytes) -> float64 values [R, kv, T, hd]."""
    R, kv, B, w = c.shape
    hd, fp8 = w // 64, c.dtype == F8
    v = c.cpu().float().double().reshape(R, kv, -1)[..., table(B * 64, hd, side, fp8).reshape(-1)].reshape(R, kv, B * 64, hd)
    return v if exp is None else v * torch.exp2(exp.cpu().double() - 127)[..., None]


def pack(x, side, fp8):
    """Values [R, kv, T, hd] -> (cache side [R, kv, T / 64, 64 hd], exponent bytes or None)."""
    R, kv, T, hd = x.shape
    at = table(T, hd, side, fp8).reshape(-1)
    exp = None
    if fp8:
        v, e = quantise(x)
        exp, x = (e + 127).to(torch.uint8), v * torch.exp2(-e.double())[..., None]
    out = torch.zeros(R, kv, T * hd, dtype=torch.float32)
    out[..., at] = x.reshape(R, kv, T * hd).float()
    return out.to(F8 if fp8 else torch.bfloat16).reshape(R, kv, T // 64, 64 * hd), exp


def rms_rope(x, w, pos, inv_freq, rd, eps):
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1 + w.double())
    ang = pos * inv_freq.double()
    h = rd // 2
    a, b = x[..., :h], x[..., h:rd]
    return torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., rd:]), -1)


def decode_attention(proj, pos, qn, kn, inv, k, v, nh, rd, eps, fp8, prefix=None):
    """k, v: float64 [N, kv, T, hd], updated in place with the new token as the cache holds it; prefix: (k, v [P, kv, Tp,
    hd], length, of).  Returns the gated output [N, nh * hd] in float64 and the new keys before they were rounded."""
    N, kv, T, hd = k.shape
    G = nh // kv
    out = torch.zeros(N, nh, hd, dtype=torch.float64)
    raw = torch.zeros(N, kv, hd, dtype=torch.float64)
    hold = (lambda y: quantise(y)[0]) if fp8 else (lambda y: y.to(torch.bfloat16).double())
    for n in range(N):
        p = int(pos[n])
        if p < 0:
            continue
        row = proj[n].double()
        r = int(prefix[3][n]) if prefix is not None else -1
        r = r if prefix is not None and 0 <= r < prefix[0].shape[0] else -1
        plen = min(max(int(prefix[2][r]), 0), prefix[0].shape[2]) if r >= 0 else 0
        at = p - plen
        raw[n] = rms_rope(row[2 * nh * hd:(2 * nh + kv) * hd].view(kv, hd), kn, p, inv, rd, eps)
        if 0 <= at < T:
            k[n, :, at] = hold(raw[n])
            v[n, :, at] = hold(row[(2 * nh + kv) * hd:].view(kv, hd))
        own = min(max(at + 1, 0), T)
        qg = row[:2 * nh * hd].view(nh, 2 * hd)
        q = rms_rope(qg[:, :hd], qn, p, inv, rd, eps).view(kv, G, hd)
        kk, vv = k[n, :, :own], v[n, :, :own]
        if r >= 0:
            kk, vv = torch.cat((prefix[0][r, :, :plen], kk), 1), torch.cat((prefix[1][r, :, :plen], vv), 1)
        pr = torch.softmax(q @ kk.transpose(1, 2) / math.sqrt(hd), -1)
        out[n] = (pr @ vv).reshape(nh, hd) * torch.sigmoid(qg[:, hd:])
    return out.view(N, nh * hd), raw


def sample(logits, u, temperature, top_k, top_p, min_p):
    """Row by row in extended precision, by sorting."""
    N, V = logits.shape
    col = lambda x: np.broadcast_to(np.asarray(x, dtype=np.float64), (N,))  # noqa: E731
    t, k, p, m, u = (col(x) for x in (temperature, top_k, top_p, min_p, u))
    out = []
    for n in range(N):
        l = logits[n].float().numpy().astype(np.longdouble)
        l = np.where(np.isnan(l), -np.inf, l)
        best = int(np.argmax(l))
        if l[best] == -np.inf:
            out.append(-1)
            continue
        if not t[n] > 0:
            out.append(best)
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(l == l[best], 1.0, np.exp((l - l[best]) / np.longdouble(t[n])))
        order = np.argsort(-l, kind="stable")
        order = order[l[order] > -np.inf]
        if 0 < k[n] < V:
            order = order[:int(k[n])]
        if p[n] < 1:
            c = np.cumsum(w[order])
            # the mass to reach is a double, p times the mass rounded: 0.9 as a double lies 2.2e-17 above 0.9, so 0.9 of 40
            # equal weights is 36 + 8.9e-16 exactly, and 36 (not 37 tokens) as the nearest double
            order = order[:max(1, int(np.searchsorted(c, np.longdouble(p[n] * np.float64(c[-1])))) + 1)]
        order = np.sort(order[(w[order] >= m[n]) | (l[order] == l[best])])
        c = np.cumsum(w[order])
        x = min(max(float(u[n]) if u[n] == u[n] else 0.0, 0.0), 1 - 2.0 ** -53)
        out.append(int(order[min(int(np.searchsorted(c, np.longdouble(x) * c[-1], side="right")), len(c) - 1)]))
    return torch.tensor(out)
