"""Outputs of a ragged decode that are too small or of another type are refused before any launch."""
import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_outputs():
    k, v = [[torch.randn(2, n, 64, device=DEV).bfloat16() for n in (40, 7, 300)] for _ in range(2)]
    plan = tnn.DecodePlan(k, v, 4)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()

    def bf16(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)

    n = tnn.launch_count()
    for call in (tnn.flashDecode, tnn.flashDecodeStatic):
        for kw in (dict(out=bf16(2, 4, 64)), dict(out=bf16(3, 2, 64)), dict(out=bf16(3, 4, 32)), dict(out=bf16(3, 256)), dict(out=bf16(3, 4, 64).float()),
                   dict(out=bf16(3, 64, 4).transpose(1, 2)), dict(out=bf16(3, 4, 2, 64)), dict(lse=torch.zeros(2, 4, device=DEV)),
                   dict(lse=torch.zeros(3, 4, dtype=torch.float64, device=DEV)), dict(lse=torch.zeros(4, 3, device=DEV).t())):
            with pytest.raises(ValueError):
                call(q, plan, **kw)
    assert tnn.launch_count() == n
    want, stats = tnn.flashDecode(q, plan)
    wide, lse = bf16(3, 2, 4, 64), torch.zeros(3, 4, device=DEV)
    for call, out in ((tnn.flashDecode, bf16(3, 4, 64)), (tnn.flashDecodeStatic, bf16(3, 4, 64)), (tnn.flashDecode, bf16(3, 4, 1, 64)),
                      (tnn.flashDecode, wide[:, 1]), (tnn.flashDecode, bf16(4, 3, 64).transpose(0, 1))):
        call(q, plan, out=out, lse=lse)
        assert torch.equal(out.view(3, 4, 64) if out.is_contiguous() else out, want) and torch.equal(lse, stats)
    assert not wide[:, 0].any()
