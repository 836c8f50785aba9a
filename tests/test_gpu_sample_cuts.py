"""GPU tests of where sampling cuts: masses of many near-equal weights in batches of many rows, and a top_p that asks for all
that top_k left, against the oracle's sort in extended precision."""
import pytest
import torch

from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


def crowded(kind, N, V, dtype, seed):
    """Rows whose weights crowd together: thousands of them near the largest."""
    g = torch.Generator().manual_seed(seed)
    if kind == "halves":  # the first half a little above the second
        l = torch.full((N, V), 1.0)
        l[:, :V // 2] = 1.0625
    elif kind == "bulk":  # nine in ten equal, the others below them, a few above
        l = torch.where(torch.rand(N, V, generator=g) < 0.9, 1.0, 0.75)
        l[:, ::V // 7] = 1.5
    elif kind == "narrow":  # distinct values within a hundredth
        l = 4.5 + 0.02 * (torch.rand(N, V, generator=g) - 0.5)
    else:
        l = torch.full((N, V), -2.0)
    return l.to(dtype), torch.rand(N, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("kind,N,V", [("halves", 64, 248320), ("bulk", 64, 151936), ("narrow", 128, 248320), ("equal", 17, 248320),
                                      ("bulk", 256, 50001), ("halves", 1100, 8193)])
@pytest.mark.parametrize("par", [(1.0, 0, 0.3, 0.0), (1.0, 0, 0.5, 0.0), (0.7, 0, 0.9, 0.01), (1.0, 40000, 0.6, 0.0)])
def test_many_rows_of_crowded_weights(gdn, dev, dtype, kind, N, V, par):
    """A workgroup sums the weights of several chunks (2 to 8 of 8192 logits), and 65536 weights of 1 have to fit."""
    l, u = crowded(kind, N, V, dtype, N)
    got = gdn.sample_tokens(l.to(dev), u.to(dev), *par).cpu()
    some = torch.arange(0, N, N // 8)
    assert torch.equal(got[some], so.sample(l[some], u[some].numpy(), *par))


@pytest.mark.parametrize("dtype,V,T,N", [(torch.float32, 3000, 7.3, 65000), (torch.float16, 200, 7.3, 65000), (torch.bfloat16, 200, 7.3, 65000)])
@pytest.mark.parametrize("short", [2.0 ** -53, 2.0 ** -52])
def test_top_p_next_to_one_keeps_to_top_k(gdn, dev, dtype, V, T, N, short):
    """A top_p of one less a rounding or two asks for all that top_k left: its mass, summed along two descents, may differ in
    the last place, and still nothing below top_k's cut is taken.  Logits in descending order and the largest random number:
    the token is the last one kept."""
    g = torch.Generator(device=dev).manual_seed(V)
    l = torch.randn(N, V, generator=g, device=dev).mul(3).to(dtype).float().sort(-1, descending=True).values.to(dtype)
    k = torch.randint(1, V, (N,), generator=g, device=dev).int()
    u = torch.full((N,), 1 - 2.0 ** -53, dtype=torch.float64, device=dev)
    got = gdn.sample_tokens(l, u, T, k, 1 - short)
    assert int((got >= k).sum()) == 0


def test_parameters_in_fp64_are_not_rounded(gdn, dev):
    """A number and an fp64 tensor of it cut alike; in fp32 the same figures cut elsewhere."""
    top = torch.full((3,), 1 - 2.0 ** -53, dtype=torch.float64, device=dev)
    one = lambda x, dtype=torch.float64: torch.full((3,), x, dtype=dtype, device=dev)  # noqa: E731
    flat = torch.zeros(3, 10, device=dev)
    for p, want in ((0.3, 2), (0.6, 5)):  # 0.3 as fp32 is 0.30000001: a fourth token
        assert gdn.sample_tokens(flat, top, 1.0, 0, p).tolist() == [want] * 3
        assert gdn.sample_tokens(flat, top, 1.0, 0, one(p)).tolist() == [want] * 3
        assert gdn.sample_tokens(flat, top, 1.0, 0, one(p, torch.float32)).tolist() == [want + 1] * 3
    l = torch.tensor([[0.0, -1.0]], device=dev).expand(3, -1)
    m = 0.36787944  # exp(-1) is 0.3678794412; as fp32 0.3678794503
    assert gdn.sample_tokens(l, top, 1.0, 0, 1.0, m).tolist() == [1] * 3
    assert gdn.sample_tokens(l, top, 1.0, 0, 1.0, one(m)).tolist() == [1] * 3
    assert gdn.sample_tokens(l, top, 1.0, 0, 1.0, one(m, torch.float32)).tolist() == [0] * 3
    t, m = 1 + 1e-8, 0.367879443  # exp(-1 / t) is 0.3678794449; t as fp32 is 1
    assert gdn.sample_tokens(l, top, t, 0, 1.0, m).tolist() == [1] * 3
    assert gdn.sample_tokens(l, top, one(t), 0, 1.0, m).tolist() == [1] * 3
    assert gdn.sample_tokens(l, top, one(t, torch.float32), 0, 1.0, m).tolist() == [0] * 3


@pytest.mark.parametrize("t", [1e-40, 1e-61, 1e-268, 1e-300, 1e-306, 3e-308, 5e-324])
@pytest.mark.parametrize("base", [-5.0, 0.0, 7.0, -1e30])
def test_smallest_temperatures(gdn, dev, t, base):
    """A temperature at which (l - max) / temperature leaves doubles behind: the ties of the maximum share the draw, cut by
    top_k and top_p as at any other."""
    l = torch.full((8, 100), base * 2 if base < 0 else base - 1)
    l[:, [7, 20, 50, 93]] = base
    u = torch.arange(8) / 8
    for par in ((t, 0, 0.5, 0.0), (t, 3, 1.0, 0.0), (t, 0, 0.8, 0.1), (t, 30, 0.7, 0.0), (t, 0, 1.0, 0.0)):
        assert torch.equal(gdn.sample_tokens(l.to(dev), u.to(dev), *par).cpu(), so.sample(l, u.numpy(), *par)), par
