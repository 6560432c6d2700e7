"""Prologue calls whose weight or positions are too short for what the kernel reads are refused before any launch."""
import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("paged", [False, True])
def test_short_weights_and_positions(paged):
    x = torch.randn(3, 2, 4, 128, device=DEV).bfloat16()
    out = torch.zeros(3, 4, 16, 128, dtype=torch.bfloat16, device=DEV)
    kw = dict(page_table=torch.arange(3, dtype=torch.int32, device=DEV).view(3, 1)) if paged else {}
    pos = torch.tensor([0, 3, 14], dtype=torch.int32, device=DEV)
    n = tnn.launch_count()
    for bad in (dict(norm_weight=torch.ones(127, device=DEV)), dict(norm_weight=torch.ones(64, device=DEV)), dict(positions=pos[:2]),
                dict(positions=torch.stack([pos, pos], 1)[:, 0])):
        with pytest.raises(ValueError):
            tnn.qkPrologue(x, out, **bad, **kw)
    assert tnn.launch_count() == n and not out.any()
    w = torch.rand(128, device=DEV) + 0.5
    tnn.qkPrologue(x, out, w, positions=pos, **kw)
    y = x.double().cpu()
    want = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.double().cpu()
    for b, p in enumerate(pos.tolist()):
        got = out[b, :, p:p + 2].transpose(0, 1).double().cpu()
        # one rounding to bf16; a sum of 128 squares and three products in 32 bits
        assert bool(((got - want[b]).abs() <= want[b].abs() * (2.0 ** -8 + 140 * 2.0 ** -24)).all())
