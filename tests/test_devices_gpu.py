"""Host tensors where the kernels follow a device pointer are refused before any launch."""
import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def refused(call):
    n = tnn.launch_count()
    with pytest.raises(ValueError):
        call()
    assert tnn.launch_count() == n


def randn(*shape):
    return torch.randn(*shape, device=DEV).bfloat16()


def test_forward_and_backward():
    q, k, v, d_o = (randn(1, 2, 64, 64) for _ in range(4))
    o, lse = tnn.attentionFwd(q, k, v)
    refused(lambda: tnn.attentionFwd(q, k, v, lse=torch.empty(1, 2, 64)))
    refused(lambda: tnn.attentionFwd(q, k, v, out=torch.empty(1, 2, 64, 64, dtype=torch.bfloat16)))
    refused(lambda: tnn.attentionFwd(q, k, v, key_mask=torch.ones(1, 64, dtype=torch.uint8)))
    need = 1 << 16
    refused(lambda: tnn.attentionBwd(q, k, v, o, lse, d_o, workspace=torch.empty(need)))
    refused(lambda: tnn.attentionBwd(q, k, v, o, lse, d_o, workspace=torch.empty(need), window_size=8, n_sink=2))
    refused(lambda: tnn.attentionBwd(q, k, v, o, lse, d_o, key_mask=torch.ones(1, 64, dtype=torch.uint8)))


def test_decode():
    q, kc, vc = randn(2, 4, 64), randn(2, 2, 40, 64), randn(2, 2, 40, 64)
    lens = torch.tensor([7, 40], dtype=torch.int32)
    refused(lambda: tnn.flashDecodeDense(q, kc, vc, kv_lens=lens))
    refused(lambda: tnn.flashDecodeDense(q, kc, vc, workspace=torch.empty(1 << 20, dtype=torch.uint8)))
    plan = tnn.DecodePlan([kc[0], kc[1]], [vc[0], vc[1]], 4)
    refused(lambda: tnn.flashDecode(q, plan, out=torch.empty(2, 4, 64, dtype=torch.bfloat16)))
    refused(lambda: tnn.flashDecode(q, plan, lse=torch.empty(2, 4)))
    refused(lambda: tnn.flashDecodeStatic(q, plan, lse=torch.empty(2, 4)))
    want, _ = tnn.flashDecodeDense(q, kc, vc)
    got, _ = tnn.flashDecode(q, plan, out=torch.empty_like(q), lse=torch.empty(2, 4, device=DEV))
    assert torch.allclose(got.float(), want.float(), atol=2e-2)
