"""Arguments of the paged-cache calls that have to be refused, or whose default has to be what the documentation says."""
import math

import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def cache(n_pages=8, hkv=2, page=16, d=64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n_pages, hkv, page, d, generator=g).bfloat16().to(DEV) for _ in range(2)]


def test_weights_do_not_change_which_keys_are_seen():
    """The most keys of a sequence are what the table holds; sums for fewer of them need an explicit max_kv_seq."""
    kp, vp = cache()
    q = torch.randn(1, 4, 64, device=DEV).bfloat16()
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    lens = torch.tensor([120], dtype=torch.int32, device=DEV)
    o, lse = tnn.flashDecodePaged(q, kp, vp, table, lens)
    narrow = torch.zeros(1, 2, 100, device=DEV)
    with pytest.raises(ValueError):
        tnn.flashDecodePaged(q, kp, vp, table, lens, weights=narrow)
    with pytest.raises(ValueError):
        tnn.paged_decode_workspace_bytes(q, kp, vp, table, lens, weights=narrow)
    with pytest.raises(ValueError):
        tnn.flashDecodePaged(q, kp, vp, table, lens, max_kv_seq=101, weights=narrow)
    assert not narrow.any()
    for width in (128, 130):                                 # all the table can hold, or more
        w = torch.zeros(1, 2, width, device=DEV)
        o1, lse1 = tnn.flashDecodePaged(q, kp, vp, table, lens, weights=w)
        assert torch.equal(o1, o) and torch.equal(lse1, lse)
        assert math.isclose(float(w[0, :, :120].sum()), 4.0, rel_tol=1e-4) and not w[0, :, 120:].any()
    short = torch.tensor([90], dtype=torch.int32, device=DEV)
    o1, _ = tnn.flashDecodePaged(q, kp, vp, table, short, max_kv_seq=100, weights=narrow)
    o2, _ = tnn.flashDecodePaged(q, kp, vp, table, short, max_kv_seq=100)
    assert torch.equal(o1, o2) and math.isclose(float(narrow.sum()), 4.0, rel_tol=1e-4)
    assert tnn.device_status(0, True) == 0
