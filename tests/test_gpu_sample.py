"""GPU tests of sampling against the oracle's sort in extended precision: the same token, every time."""
import pytest
import torch

from oracle import serving_oracle as so

BF = torch.bfloat16
pytestmark = pytest.mark.gpu


def logits_of(N, V, dtype, seed, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    if kind == "flat":
        l = torch.zeros(N, V)
    elif kind == "few":  # few distinct values: ties everywhere
        l = torch.randint(-3, 4, (N, V), generator=g).float()
    elif kind == "negative":
        l = -torch.rand(N, V, generator=g) * 20 - 1e-3
    else:
        l = torch.randn(N, V, generator=g) * 3
        l += 8 * (torch.rand(N, V, generator=g) < 30 / V)
    if kind == "masked":
        l[torch.rand(N, V, generator=g) < 0.9] = float("-inf")
    return l.to(dtype), torch.rand(N, generator=g)


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 255, 4096, 4097, 50001, 248320])
@pytest.mark.parametrize("par", [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.8, 20, 0.8, 0.05), (0.0, 5, 0.5, 0.5),
                                 (1.0, 0, 1.0, 0.2), (2.5, 3000000, 0.999, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0),
                                 (0.01, 0, 0.99, 0.0), (50.0, 1000, 0.5, 0.9)])
def test_against_oracle(gdn, dev, dtype, V, par):
    N = 5 if V < 100000 else 3
    l, u = logits_of(N, V, dtype, V + int(par[0] * 10))
    got = gdn.sample_tokens(l.to(dev), u.to(dev), *par)
    assert got.dtype == torch.int64 and torch.equal(got.cpu(), so.sample(l, u.numpy(), *par))


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["flat", "few", "negative", "masked"])
@pytest.mark.parametrize("par", [(1.0, 0, 1.0, 0.0), (1.0, 77, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (0.9, 500, 0.61, 0.01), (1.0, 0, 0.83, 0.5)])
def test_ties_and_masks(gdn, dev, dtype, kind, par):
    """Equal logits (the lowest index first), log-probabilities, and masks of -inf."""
    l, u = logits_of(40, 9001, dtype, 7, kind)
    got = gdn.sample_tokens(l.to(dev), u.to(dev), *par)
    assert torch.equal(got.cpu(), so.sample(l, u.numpy(), *par))


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_special_rows(gdn, dev, dtype):
    """Rows of -inf and NaN give -1; NaN and -inf are never taken; +inf takes all; -0 and 0 tie; the type's lowest value is
    a value; random numbers at and outside the borders."""
    V, inf, nan = 5000, float("inf"), float("nan")
    l = torch.randn(9, V, generator=torch.Generator().manual_seed(8))
    l[0] = -inf
    l[1] = nan
    l[2, ::2] = nan
    l[3] = -inf
    l[3, 4321] = -5.0
    l[4, 77] = l[4, 4500] = inf
    l[5] = -0.0
    l[5, 10:20] = 0.0
    l[6] = torch.finfo(dtype).min
    l[7] = -inf
    l[7, 100:103] = torch.finfo(dtype).min
    l = l.to(dtype)
    for par in ((1.0, 0, 1.0, 0.0), (0.6, 40, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (1e-30, 0, 0.9, 0.0), (1.0, 15, 1.0, 0.0)):
        for u0 in (0.0, 0.5, 1 - 2.0 ** -24, 1.0, -0.5, nan):
            u = torch.full((9,), u0)
            got = gdn.sample_tokens(l.to(dev), u.to(dev), *par)
            assert torch.equal(got.cpu(), so.sample(l, u.numpy(), *par)), (par, u0)


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_parameters_per_row(gdn, dev, dtype):
    """Every row with its own parameters, greedy and unfiltered rows beside filtered ones; tensors of other whole and
    floating types; a strided, unaligned view of the logits."""
    N, V = 24, 30011
    l, u = logits_of(N, V, dtype, 11)
    g = torch.Generator().manual_seed(12)
    i = torch.arange(N)
    t = torch.where(i % 5 == 0, 0.0, torch.rand(N, generator=g) * 2 + 0.1)
    t[7] = float("nan")
    k = torch.where(i % 3 == 0, 0, torch.randint(1, 200, (N,), generator=g))
    p = torch.where(i % 4 == 0, 1.0, torch.rand(N, generator=g))
    m = torch.where(i % 2 == 0, 0.0, torch.rand(N, generator=g) * 0.2)
    wide = torch.zeros(N, V + 13, dtype=dtype, device=dev)
    wide[:, 5:V + 5] = l.to(dev)
    got = gdn.sample_tokens(wide[:, 5:V + 5], u.double().to(dev), t.to(dev), k.to(dev), p.to(dev), m.to(dev))
    assert torch.equal(got.cpu(), so.sample(l, u.numpy(), t.numpy(), k.numpy(), p.numpy(), m.numpy()))
    again = gdn.sample_tokens(l.to(dev), u.to(dev), t.to(dev), k.int().to(dev), p.double().to(dev), m.to(dev))
    assert torch.equal(again, got)


def test_graph_and_stream(gdn, dev):
    """Captured with a kept workspace and replayed on new logits, with eager calls between; and on a stream of its own."""
    N, V = 6, 40000
    l, u = logits_of(N, V, BF, 20)
    par = (0.8, 60, 0.9, 0.02)
    ld, ud = l.to(dev), u.to(dev)
    work = gdn.sample_workspace(N, V, dev)
    graph = gdn.GDNDecodeGraph(lambda: gdn.sample_tokens(ld, ud, *par, work=work), device=dev)
    for seed in (20, 21, 22):
        l, u = logits_of(N, V, BF, seed)
        ld.copy_(l)
        ud.copy_(u)
        got = graph.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), so.sample(l, u.numpy(), *par))
        assert torch.equal(gdn.sample_tokens(ld, ud, *par), got)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got2 = gdn.sample_tokens(ld, ud, *par)
    torch.cuda.synchronize()
    assert torch.equal(got2, got)


@pytest.mark.parametrize("dtype,N,V", [(BF, 600, 20000), (torch.float32, 700, 9000), (torch.float16, 2500, 100), (torch.float32, 2, 1000003)])
def test_many_rows_and_long_ones(gdn, dev, dtype, N, V):
    """Rows of which a workgroup takes several chunks, rows shorter than that, and a row of many chunks; the workspace of
    these rows serves fewer as well."""
    l, u = logits_of(N, V, dtype, N)
    work = gdn.sample_workspace(N, V, dev)
    ld, ud = l.to(dev), u.to(dev)
    for par in ((1.0, 0, 1.0, 0.0), (0.9, 40, 0.9, 0.01)):
        want = so.sample(l, u.numpy(), *par)
        assert torch.equal(gdn.sample_tokens(ld, ud, *par, work=work).cpu(), want)
        n = N // 2
        assert torch.equal(gdn.sample_tokens(ld[:n], ud[:n], *par, work=work).cpu(), want[:n])


def test_one_row_for_all_and_wide_parameters(gdn, dev):
    """The same logits for every random number (a row stride of 0), an odd row start, and top_k in int64 past 32 bits."""
    l, u = logits_of(1, 5001, BF, 30)
    u = torch.rand(64, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    want = so.sample(l.expand(64, -1), u.numpy(), 1.0, 0, 0.9, 0.0)
    assert torch.equal(gdn.sample_tokens(l.to(dev).expand(64, -1), u.to(dev), 1.0, 0, 0.9).cpu(), want)
    l, u = logits_of(4, 3001, torch.float32, 31)
    k = torch.tensor([2 ** 32 + 5, 2 ** 31, -(2 ** 40), 5], device=dev)
    got = gdn.sample_tokens(l.to(dev)[:, 1:], u.to(dev), 1.0, k)
    assert torch.equal(got.cpu(), so.sample(l[:, 1:], u.numpy(), 1.0, [0, 0, 0, 5], 1.0, 0.0))
    with pytest.raises(TypeError, match="whole"):
        gdn.sample_tokens(l.to(dev), u.to(dev), 1.0, 2.5)
    with pytest.raises(TypeError, match="whole"):
        gdn.sample_tokens(l.to(dev), u.to(dev), 1.0, k.float())


def test_refusals(gdn, dev):
    l, u = torch.zeros(2, 10, device=dev), torch.zeros(2, device=dev)
    for args, kw in (((l[0], u), {}), ((l, u[:1]), {}), ((l, u.half()), {}), ((l, u, float("nan")), {}), ((l, u, float("inf")), {}),
                     ((l, u, 1.0, 0, 1.5), {}), ((l, u, 1.0, 0, 1.0, -0.1), {}), ((l, u, torch.ones(2)), {}),
                     ((l, u, torch.ones(3, device=dev)), {}), ((l, u), dict(work=torch.zeros(16)))):
        with pytest.raises(ValueError):
            gdn.sample_tokens(*args, **kw)
    with pytest.raises(TypeError):
        gdn.sample_tokens(l.double(), u)
    with pytest.raises(gdn.GDNError, match="workspace"):
        gdn.sample_tokens(l, u, work=torch.zeros(16, dtype=torch.uint8, device=dev))
    assert gdn.sample_tokens(l[:0], u[:0]).shape == (0,)
