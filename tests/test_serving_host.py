"""CPU checks of the serving operators (KV cache, attention over it, sampling): refusals before any GPU call, the C ABI's
argument checks, and the oracle against itself and against torch."""
import ctypes
import importlib

import pytest
import torch

from conftest import PKG_NAME
from oracle import serving_oracle as so

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def test_public_names(gdn):
    for name in ("KVCache", "SharedPrefix", "kv_cache_store", "kv_cache_load", "cached_attn_workspace",
                 "cached_decode_attention", "sample_tokens", "sample_workspace"):
        assert hasattr(gdn, name) and name in gdn.__all__


@pytest.mark.parametrize("dtype", [F8, BF])
def test_cpu_tensors_are_refused(gdn, dtype):
    c = gdn.KVCache.empty(2, 2, 64, 100, dtype=dtype, device="cpu")
    assert c.length == 128 and c.head_dim == 64 and c.k.shape == (2, 2, 2, 64 * 64)
    x = torch.zeros(5, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="no CPU fallback"):
        gdn.kv_cache_store(c, x, x, [0])
    with pytest.raises(ValueError, match="no CPU fallback"):
        gdn.kv_cache_load(c, [0], [0, 5])
    with pytest.raises(ValueError, match="no CPU fallback"):
        gdn.cached_attn_workspace(c, 4)
    with pytest.raises(ValueError, match="no CPU fallback"):
        gdn.cached_decode_attention(torch.zeros(2, 12 * 64, dtype=BF), torch.zeros(2, dtype=torch.int64), torch.zeros(64),
                                    torch.zeros(64), torch.ones(8), c, 4, 16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        gdn.sample_tokens(torch.zeros(2, 10), torch.zeros(2))


def test_cache_sizes_and_types(gdn):
    for bad in (dict(head_dim=96), dict(length=0), dict(n_rows=0)):
        with pytest.raises(ValueError):
            gdn.KVCache.empty(**{**dict(n_rows=1, kv_heads=1, head_dim=64, length=64, device="cpu"), **bad})
    with pytest.raises(TypeError):
        gdn.KVCache.empty(1, 1, 64, 64, dtype=torch.float16, device="cpu")


def test_c_abi_refuses(gdn):
    """Argument checks run on the host, before any HIP call."""
    h = importlib.import_module(PKG_NAME + "._lib").lib()
    p, f = ctypes.c_void_p(256), ctypes.c_float

    def store(dtype=3, hd=128, T=64, xk=p, stride=256, indt=1, nseq=1, total=4, cu=None, rows=p):
        return h.gdn_kv_store(xk, stride, 128, p, 256, 128, indt, p, p, p, p, dtype, 2, 2, hd, T, rows, cu, None, nseq, total, None)
    for kw, rc, msg in ((dict(dtype=2), 1, b"bf16 or e4m3"), (dict(hd=96), 2, b"head_dim"), (dict(T=100), 1, b"multiple of 64"),
                        (dict(xk=ctypes.c_void_p(264)), 1, b"16-byte"), (dict(stride=129), 1, b"16-byte"), (dict(indt=7), 1, b"input dtype"),
                        (dict(nseq=3), 1, b"divide"), (dict(rows=None), 1, b"null")):
        assert store(**kw) == rc and msg in h.gdn_last_error(), kw
    assert store(total=0) == 0 and store(nseq=0) == 0
    rc = h.gdn_kv_load(p, p, None, None, 3, 2, 2, 128, 64, p, None, None, 1, 4, p, p, None)
    assert rc == 1 and b"null" in h.gdn_last_error()

    def attn(proj=p, stride=12 * 64, dtype=3, T=64, P=0, hd=64, nh=4, kv=2, rd=16, work=1 << 40, plen=None, ke=p, N=2):
        return h.gdn_attn_cached(proj, stride, None, 0, p, p, p, p, p, p, ke, p, dtype, T, p, p, p, p, plen, plen, P, 64, p,
                                 nh * hd, p, work, N, nh, kv, hd, rd, f(1e-6), None)
    for kw, rc, msg in ((dict(proj=None), 1, b"null"), (dict(stride=64), 1, b"projection"), (dict(dtype=0), 1, b"bf16 or e4m3"),
                        (dict(T=65), 1, b"multiple of 64"), (dict(hd=96), 2, b"head_dim"), (dict(nh=34), 2, b"16 query heads"),
                        (dict(nh=5), 1, b"head counts"), (dict(rd=15), 1, b"rotary"), (dict(work=16), 1, b"workspace"),
                        (dict(P=1), 1, b"prefix"), (dict(ke=None), 1, b"null")):
        assert attn(**kw) == rc and msg in h.gdn_last_error(), kw
    assert attn(N=0) == 0
    assert h.gdn_attn_cached_workspace_bytes(16, 24, 4, 256, 100, 0, 0) == -1
    assert h.gdn_attn_cached_workspace_bytes(16, 24, 4, 256, 128, 1, 128) > h.gdn_attn_cached_workspace_bytes(16, 24, 4, 256, 128, 0, 0) > 0

    def sample(logits=p, stride=1000, dtype=1, t1=1.0, p1=1.0, m1=0.0, N=2, V=1000, work=1 << 40):
        return h.gdn_sample(logits, stride, dtype, p, 0, None, None, None, None, t1, 0, p1, m1, p, N, V, p, work, None)
    for kw, rc, msg in ((dict(logits=None), 1, b"null"), (dict(stride=999), 1, b"stride"), (dict(dtype=3), 1, b"fp32, bf16"),
                        (dict(t1=float("nan")), 1, b"temperature"), (dict(p1=1.5), 1, b"top_p"), (dict(m1=-0.1), 1, b"min_p"),
                        (dict(V=0), 1, b"sizes"), (dict(work=16), 1, b"workspace")):
        assert sample(**kw) == rc and msg in h.gdn_last_error(), kw
    assert sample(N=0) == 0


def test_c_abi_limits_and_workspaces(gdn):
    """A call takes 1024 slots and prefixes and 8388608 logits a row; a workspace for many rows or slots holds fewer."""
    h = importlib.import_module(PKG_NAME + "._lib").lib()
    attn = lambda N, P=0, T=128, Tp=128: h.gdn_attn_cached_workspace_bytes(N, 24, 4, 256, T, P, Tp)  # noqa: E731
    assert attn(1024, 1024) > 0 and attn(1025) == -1 and attn(4, 1025) == -1
    sizes = [attn(n, 2, 32768, 16384) for n in range(0, 200)]
    assert sizes == sorted(sizes)
    assert h.gdn_sample_workspace_bytes(1, 8388608) > 0 and h.gdn_sample_workspace_bytes(1, 8388609) == -1
    for V in (1, 9000, 65537, 131072, 248320):
        sizes = [h.gdn_sample_workspace_bytes(n, V) for n in range(0, 1200)]
        assert sizes == sorted(sizes)
    sizes = [h.gdn_sample_workspace_bytes(500, v) for v in range(1, 300000, 997)]
    assert sizes == sorted(sizes)


def test_oracle_quantises_as_torch_does():
    """Codes are torch's own e4m3 rounding of x 2^-e, and e is the smallest that fits."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 64, generator=g) * torch.exp2(torch.randint(-40, 40, (200, 1), generator=g).float())
    x[0] = 0
    x[1, :4] = torch.tensor([448.0, -448.0, 449.0, 1e-3])
    x[2, 0] = 448.0
    x[2, 1:] = 1.0
    x[3, 5], x[3, 6] = float("inf"), float("nan")
    v, e = so.quantise(x)
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1).double()
    assert ((top <= 448 * torch.exp2(e.double())) & ((top > 448 * torch.exp2(e.double() - 1)) | (top == 0))).all()
    want = torch.ldexp(x, -e[:, None]).to(F8).double() * torch.exp2(e.double())[:, None]
    fin = x.isfinite()
    assert torch.equal(v[fin], want[fin]) and v[~fin].isnan().all()
    assert int(e[0]) == 0 and int(e[2]) == 0


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fp8", [True, False])
def test_oracle_layout_is_a_permutation(hd, fp8):
    for side in ("k", "v"):
        t = so.table(128, hd, side, fp8).reshape(-1)
        assert torch.equal(t.sort().values, torch.arange(128 * hd))
        x = torch.randn(1, 2, 128, hd, generator=torch.Generator().manual_seed(hd)).to(BF).double()
        c, e = so.pack(x, side, fp8)
        want = so.quantise(x)[0] if fp8 else x
        assert torch.equal(so.unpack(c, e, side), want)


def test_oracle_sampling_frequencies():
    """Tokens drawn over a grid of u have the filtered softmax's probabilities."""
    l = torch.tensor([[2.0, 1.0, 1.0, 0.0, -1.0, float("-inf"), 3.0, 0.5]])
    u = (torch.arange(4000) + 0.5) / 4000
    t = so.sample(l.expand(4000, -1), u.numpy(), 0.7, 6, 0.95, 0.05)
    w = torch.softmax(l[0] / 0.7, 0)
    keep = torch.tensor([True, True, True, False, False, False, True, False])  # top 6, 0.95 of it, then min_p 0.05
    assert ((t.unsqueeze(0) == torch.arange(8)[:, None]).float().mean(1) - w * keep / (w * keep).sum()).abs().max() < 2 / 4000
