"""Dense decode calls that would read behind the cache are refused before any launch."""
import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(*shape):
    return torch.randn(*shape, device=DEV).bfloat16()


def test_refusals():
    q, kc, vc = randn(2, 4, 64), randn(2, 2, 40, 64), randn(2, 2, 40, 64)
    lens = torch.tensor([7, 40], dtype=torch.int32, device=DEV)
    n = tnn.launch_count()
    for kw in (dict(kv_len=41), dict(kv_len=2 ** 31 - 1), dict(kv_len=2 ** 32 + 5), dict(kv_lens=lens, kv_len=41), dict(kv_lens=lens[:1]),
               dict(kv_lens=lens.long()), dict(kv_lens=torch.stack([lens, lens], 1)[:, 0])):
        with pytest.raises(ValueError):
            tnn.flashDecodeDense(q, kc, vc, **kw)
    for bad in (0, -1, -2 ** 32 + 5):
        with pytest.raises(tnn.AttnError):
            tnn.flashDecodeDense(q, kc, vc, kv_len=bad)
    for k, v in ((kc[:1], vc), (kc, vc[:1]), (kc, vc[:, :1]), (kc, vc[:, :, :39]), (kc.float(), vc.float()), (randn(2, 2, 40, 128), vc)):
        with pytest.raises(ValueError):
            tnn.flashDecodeDense(q, k, v)
    with pytest.raises(ValueError):
        tnn.flashDecodeDense(q.float(), kc, vc)
    assert tnn.launch_count() == n


def test_a_larger_cache_is_fine():
    q, kc, vc = randn(2, 4, 64), randn(3, 2, 40, 64), randn(3, 2, 50, 64)
    o, lse = tnn.flashDecodeDense(q, kc, vc, kv_len=33)
    o2, lse2 = tnn.flashDecodeDense(q, kc[:2, :, :33].contiguous(), vc[:2, :, :33].contiguous())
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
