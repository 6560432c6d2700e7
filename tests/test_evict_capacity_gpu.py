"""Evictions from a cache whose tables hold far more keys than its sequences have: the results are those of the tight cache."""
import pytest
import torch

from test_paged_gpu import Cache, plain_evict
from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# what one CTA of a cluster holds is 16384 keys: sequences that end in the first, at a border, in a later one
@pytest.mark.parametrize("capacity", [16385, 65536, 200000, 262144, 262145])
@pytest.mark.parametrize("ties", [False, True])
def test_capacity_does_not_matter(capacity, ties):
    page, n_keep, n_recent, n_sink = 64, 900, 250, 4
    lens = [n for n in (1, 0, 899, 900, 901, 2000, 16384, 16385, 32768, 32769, 40000, 130000) if n <= capacity]
    c = Cache(lens, 2, 64, page, seed=capacity % 1000)
    g = torch.Generator().manual_seed(capacity)
    w = torch.rand(len(lens), 2, capacity, generator=g)
    if ties:
        w = (w * 3).floor()
    table = torch.full((len(lens), -(-capacity // page)), -9, dtype=torch.int32)
    table[:, :min(c.table.shape[1], table.shape[1])] = c.table[:, :table.shape[1]]
    kp, vp = torch.nan_to_num(c.kp), torch.nan_to_num(c.vp)
    kt, vt, wd = kp.clone(), vp.clone(), w.to(DEV)
    new, kept = tnn.evictPaged(kp, vp, table.to(DEV), c.lens_dev, wd, n_keep, n_recent, n_sink, max_kv_seq=capacity)
    assert tnn.device_status(0, True) == 0
    assert new.tolist() == [min(n, n_keep) for n in lens]
    for b, n in enumerate(lens):
        if n <= n_keep:
            assert kept[b].tolist() == [list(range(n)) + [-1] * (n_keep - n)] * 2
            assert torch.equal(wd[b].cpu(), w[b])
            continue
        left = plain_evict(None, None, w[b, :, :n], n_keep, n_recent, n_sink)
        assert kept[b].tolist() == left
        for h in range(2):
            want = w[b, h].clone()
            want[:n] = 0
            want[:n_keep] = w[b, h, left[h]]
            assert torch.equal(wd[b, h].cpu(), want)
        # the rows, against the sequence alone in a cache of just its length
        one = w[b:b + 1, :, :n].to(DEV)
        tnn.evictPaged(kt, vt, c.table_dev[b:b + 1], c.lens_dev[b:b + 1], one, n_keep, n_recent, n_sink)
    assert torch.equal(kp, kt) and torch.equal(vp, vt)
