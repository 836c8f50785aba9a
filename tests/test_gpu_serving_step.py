"""GPU tests of the serving operators in a run: a prompt's keys and values stored chunk by chunk and read back, a hybrid
stack decoding over the caches (bf16, e4m3, behind a shared prefix) and sampling its tokens, eager and as one graph."""
import importlib

import pytest
import torch

from conftest import PKG_NAME, rel_l2
from oracle import serving_oracle as so

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
pytestmark = pytest.mark.gpu


def hybrid():
    return importlib.import_module(PKG_NAME + ".hybrid_decode")


def small(**kw):
    return hybrid().HybridConfig(**{**dict(hidden=256, layers=4, full_every=4, gdn_k_heads=2, gdn_v_heads=4, gdn_head=128, conv_k=4,
                                           attn_heads=4, kv_heads=2, attn_head=64, mlp=512, vocab=1000), **kw})


def inputs(N, H, n, dev, seed=7):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(N, H, generator=g).to(BF).to(dev) for _ in range(n)], [torch.rand(N, generator=g).to(dev) for _ in range(n)]


def test_bf16_cache_matches_the_default(gdn, dev):
    """The same stack over KVCaches in bf16 and over the transposed caches: the same logits (the attention rounds its
    probabilities and output apart: within 2^-8 each, through one of four layers)."""
    hd, cfg = hybrid(), small()
    a = hd.HybridDecoder(cfg, 3, [5, 17, 64], 8, dev, seed=3)
    b = hd.HybridDecoder(cfg, 3, [5, 17, 64], 8, dev, seed=3, cache_dtype=BF)
    for x in inputs(3, cfg.hidden, 4, dev)[0]:
        assert rel_l2(b.step(x), a.step(x)) <= 2e-2
    assert torch.equal(a.pos, b.pos)


def test_e4m3_cache(gdn, dev):
    """Over e4m3 caches the attention layer's output is the oracle's on what the caches hold, step after step."""
    hd, cfg = hybrid(), small(layers=1, full_every=1, mlp=0, vocab=0)
    m = hd.HybridDecoder(cfg, 2, [3, 62], 8, dev, seed=4, cache_dtype=F8, keep_plain=True)
    L = m.layers[0]
    cb = importlib.import_module(PKG_NAME + ".cb_engine")
    k, v = (so.unpack(c.cpu(), e.cpu(), s) for c, e, s in ((L.cache.k, L.cache.k_exp, "k"), (L.cache.v, L.cache.v_exp, "v")))
    for x in inputs(2, cfg.hidden, 3, dev)[0]:
        proj = cb.decode_linear(x, L.qkv_p).cpu()
        pos = m.pos.tolist()
        got = m.attention(L, x).cpu()
        m.pos += 1
        o, _ = so.decode_attention(proj, pos, L.q_norm.cpu(), L.k_norm.cpu(), m.inv_freq.cpu(), k, v, cfg.attn_heads,
                                   m.rotary_dim, cfg.eps, True)
        assert rel_l2(got, o @ L.o.cpu().double().t()) <= 1e-2


@pytest.mark.parametrize("dtype", [BF, F8])
def test_shared_prefix_in_the_stack(gdn, dev, dtype):
    """Slots behind a shared prefix give what slots with the prefix copied in front of their own tokens give."""
    hd, cfg, P, ctx = hybrid(), small(), 100, [5, 17, 40]
    a = hd.HybridDecoder(cfg, 3, ctx, 8, dev, seed=5, cache_dtype=dtype, prefix_ctx=P)
    b = hd.HybridDecoder(cfg, 3, ctx, 8, dev, seed=5, cache_dtype=dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for La, Lb in zip(a.layers, b.layers):
        # (the prefix is drawn in between, so the two stacks' later weights differ: b takes a's)
        for name in vars(La):
            if name not in ("cache", "prefix"):
                setattr(Lb, name, getattr(La, name))
        if La.full:
            Lb.cache = gdn.KVCache.empty(3, 2, 64, P + a.max_ctx, dtype, dev)
            pk, pv = gdn.kv_cache_load(La.prefix.cache, [0], [0, P])
            ok, ov = gdn.kv_cache_load(La.cache, [0, 1, 2], [0, a.max_ctx, 2 * a.max_ctx, 3 * a.max_ctx])
            for n in range(3):
                sl = slice(n * a.max_ctx, (n + 1) * a.max_ctx)
                gdn.kv_cache_store(Lb.cache, torch.cat((pk, ok[sl])), torch.cat((pv, ov[sl])), i32([n]))
    b.pos += P
    b.final_norm, b.lm_head_p = a.final_norm, a.lm_head_p
    b.attn_work = gdn.cached_attn_workspace(next(L for L in b.layers if L.full).cache, cfg.attn_heads)
    for s in (a, b):
        s.slots.reset()
    for x in inputs(3, cfg.hidden, 3, dev)[0]:
        assert rel_l2(a.step(x), b.step(x)) <= 2e-2


def test_graph_draws_the_tokens_too(gdn, dev):
    """The captured step over e4m3 caches behind a prefix, tokens drawn in it: the same logits and tokens as eager steps,
    replay after replay with eager work between, and the tokens the oracle's on those logits."""
    hd, cfg = hybrid(), small()
    mk = lambda: hd.HybridDecoder(cfg, 3, [5, 17, 9], 16, dev, seed=6, cache_dtype=F8, prefix_ctx=70)  # noqa: E731
    eager, graphed = mk(), mk()
    xs, us = inputs(3, cfg.hidden, 5, dev)
    inp, u = xs[0].clone(), us[0].clone()
    temperature = torch.tensor([0.8, 0.0, 1.2], device=dev)
    par = dict(temperature=temperature, top_k=40, top_p=0.9, min_p=0.01)
    graph = hd.HybridDecodeGraph(graphed, inp, u, **par)
    eager.step(xs[0])
    for x, r in zip(xs[1:], us[1:]):
        inp.copy_(x)
        u.copy_(r)
        out = graph.replay()
        want = eager.step(x)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(graph.tokens, eager.sample(want, r, **par))
        assert torch.equal(graph.tokens.cpu(), so.sample(want.cpu(), r.cpu().numpy(), temperature.cpu().numpy(), 40, 0.9, 0.01))
        for a, b in zip(eager.layers, graphed.layers):
            if a.full:
                assert all(torch.equal(x1.view(torch.uint8), x2.view(torch.uint8)) for x1, x2 in zip(a.cache, b.cache))


def test_chunked_prefill_round_trip(gdn, dev):
    """A prompt that arrives in chunks as HF leaves it ([kv, tokens, hd]): stored chunk by chunk, the context read back for
    each chunk equals what storing it at once gives; then a token is decoded behind it."""
    kv, hd, lens = 2, 128, [100, 64, 1, 130]
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(kv, sum(lens), hd, generator=g).to(BF).to(dev).transpose(0, 1) for _ in range(2))
    once, parts = (gdn.KVCache.empty(3, kv, hd, sum(lens) + 1, F8, dev) for _ in range(2))
    gdn.kv_cache_store(once, k, v, [1])
    at = 0
    for n in lens:
        gdn.kv_cache_store(parts, k[at:at + n], v[at:at + n], [1], start=[at])
        at += n
        ck, cv = gdn.kv_cache_load(parts, [1], [0, at])
        wk, wv = gdn.kv_cache_load(once, [1], [0, at])
        assert torch.equal(ck, wk) and torch.equal(cv, wv)
    assert rel_l2(ck, k) <= 0.03  # e4m3: at most 2^-4 a value, about 0.4 of that in the mean square
    for a, b in zip(once, parts):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_decoder_refuses_a_prefix_without_a_cache(gdn, dev):
    with pytest.raises(ValueError, match="cache_dtype"):
        hybrid().HybridDecoder(small(), 2, [3, 4], 4, dev, prefix_ctx=10)


def test_calls_at_once_on_two_streams(gdn, dev):
    """Attention and sampling on two streams at once, each with a workspace of its own, give what they give alone; a
    workspace that has served other sizes gives the same."""
    nh, kv, hd, N, V = 8, 2, 128, 12, 20000
    width = (2 * nh + 2 * kv) * hd
    g = torch.Generator().manual_seed(3)
    side = []
    for i in range(2):
        c = gdn.KVCache.empty(N, kv, hd, 1024, device=dev)
        k, v = (torch.randn(N * 1000, kv, hd, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
        gdn.kv_cache_store(c, k, v, list(range(N)))
        side.append(dict(c=c, proj=torch.randn(N, width, generator=g).to(torch.bfloat16).to(dev),
                         pos=torch.randint(0, 1000, (N,), generator=g).to(dev), l=torch.randn(N, V, generator=g).to(dev),
                         u=torch.rand(N, generator=g).to(dev), aw=gdn.cached_attn_workspace(c, nh),
                         sw=gdn.sample_workspace(2 * N, V, dev)))
    w = torch.zeros(hd, dtype=torch.bfloat16, device=dev)
    inv = 1.0 / (10000.0 ** (torch.arange(0, 32, 2, device=dev).float() / 32))

    def step(s, own=True):
        kw, sw = (dict(work=s["aw"]), s["sw"]) if own else ({}, None)
        return (gdn.cached_decode_attention(s["proj"], s["pos"], w, w, inv, s["c"], nh, 32, **kw),
                gdn.sample_tokens(s["l"], s["u"], 0.8, 50, 0.9, work=sw))
    want = [step(s, False) for s in side]
    gdn.sample_tokens(side[0]["l"].repeat(2, 1), side[0]["u"].repeat(2), work=side[0]["sw"])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in side]
    for _ in range(5):
        got = []
        for s, st in zip(side, streams):
            with torch.cuda.stream(st):
                got.append([step(s) for _ in range(3)])
        torch.cuda.synchronize()
        for i, x in enumerate(got):
            for a, t in x:
                assert torch.equal(a, want[i][0]) and torch.equal(t, want[i][1])
