"""A KV cache call's batch as it comes from the host: rows, lengths and positions that do not fit the cache are refused."""
import importlib

import pytest
import torch

from conftest import PKG_NAME


def batch(gdn, rows, cu, start, total, n_rows=4, length=128):
    return importlib.import_module(PKG_NAME + ".kv_cache")._batch("call", rows, cu, start, total, n_rows, length, torch.device("cpu"))


@pytest.mark.parametrize("rows,cu,start,total", [
    ([0], [0, 5], [124], 5), ([0], [0, 5], [-1], 5), ([0], None, [100], 29), ([0], [0, 129], None, 129), ([0, 1], None, None, 258),
    ([0, 1], [0, 10, 20], [0, 2 ** 40], 20), ([1, 0], [0, 0, 128], [129, 0], 128), ([0, 1], None, torch.tensor([0, 120]), 20),
])
def test_positions_outside_are_refused(gdn, rows, cu, start, total):
    with pytest.raises(ValueError, match="does not lie in the cache's 128 positions"):
        batch(gdn, rows, cu, start, total)
    if cu is not None:
        with pytest.raises(ValueError, match="does not lie in the cache's 128 positions"):
            batch(gdn, rows, gdn.Varlen(cu, total, "cpu"), start, total)


def test_positions_inside(gdn):
    for rows, cu, start, total in (([0], [0, 5], [123], 5), ([0], None, None, 128), ([0, 3], [0, 0, 128], [128, 0], 128),
                                   ([0, 1], None, torch.tensor([[0], [118]]), 20), ([], None, None, 0), ([0, 1], None, [3, 128], 0)):
        r, c, s, n = batch(gdn, rows, cu, start, total)
        assert n == len(rows) and r.tolist() == rows
        assert (c is None) == (cu is None) and (c is None or c.tolist() == cu)
        assert (s is None) == (start is None) and (s is None or s.tolist() == torch.as_tensor(start).reshape(-1).tolist())


@pytest.mark.gpu
def test_calls_refuse(gdn, dev):
    """Through the public calls; positions on the device are cut to the cache instead."""
    c = gdn.KVCache.empty(2, 1, 64, 128, device=dev)
    x = torch.ones(10, 1, 64, device=dev)
    for call in (lambda **kw: gdn.kv_cache_store(c, x, x, [1], **kw), lambda **kw: gdn.kv_cache_load(c, [1], [0, 10], **kw)):
        with pytest.raises(ValueError, match="does not lie"):
            call(start=[119])
    before = [t.view(torch.uint8).clone() for t in c]
    gdn.kv_cache_store(c, x, x, [1], start=torch.tensor([128], dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, c))
    k, _ = gdn.kv_cache_load(c, [1], [0, 10], start=torch.tensor([125], dtype=torch.int32, device=dev))
    assert not k.any()
