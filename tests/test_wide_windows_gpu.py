"""A sliding window at least as long as the keys hides nothing but the future, however large the number is: every call that
takes a window gives the bits of the call with a window of exactly the keys."""
import ctypes

import pytest
import torch

from tyr_b200 import _lib
from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# near and past 31 bits, past 32 (5 and 0 in the low bits), past what a C int could be cut down from
WINDOWS = [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 1]


def randn(*shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).bfloat16().to(DEV)


# one tile, several, heads shared and not; rows past the line from which no key block is shared by CTAs
@pytest.mark.parametrize("hq,hkv,s,d", [(2, 2, 100, 64), (4, 2, 300, 128), (2, 1, 2100, 64)])
@pytest.mark.parametrize("n_sink", [0, 3])
def test_forward_and_gradients(hq, hkv, s, d, n_sink):
    q, k, v, d_o = (randn(1, h, s, d, seed=i) for i, h in enumerate((hq, hkv, hkv, hq)))
    o, lse = tnn.attentionFwd(q, k, v, window_size=s, n_sink=n_sink)
    want = tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=s, n_sink=n_sink)
    assert all(bool(t.any()) for t in want)
    oc, lc = tnn.attentionFwd(q, k, v, window_size=s, n_sink=n_sink, check_mode=True)
    for window in WINDOWS:
        o1, lse1 = tnn.attentionFwd(q, k, v, window_size=window, n_sink=n_sink)
        assert torch.equal(o1, o) and torch.equal(lse1, lse), window
        o1, lse1 = tnn.attentionFwd(q, k, v, window_size=window, n_sink=n_sink, check_mode=True)
        assert torch.equal(o1, oc) and torch.equal(lse1, lc), window
        got = tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=window, n_sink=n_sink)
        for name, a, b in zip(("d_q", "d_k", "d_v"), got, want):
            assert torch.equal(a, b), (window, name)


def test_padding_mask_beside_a_wide_window():
    q, k, v, d_o = (randn(2, 2, 200, 64, seed=i) for i in range(4))
    mask = torch.ones(2, 200, dtype=torch.bool, device=DEV)
    mask[1, 150:] = False
    o, lse = tnn.attentionFwd(q, k, v, window_size=200, key_mask=mask)
    want = tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=200, key_mask=mask)
    for window in WINDOWS:
        o1, lse1 = tnn.attentionFwd(q, k, v, window_size=window, key_mask=mask)
        assert torch.equal(o1, o) and torch.equal(lse1, lse), window
        got = tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=window, key_mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), window


def test_typed_call():
    q, k, v = (randn(1, 4, 300, 64, seed=i) for i in range(3))
    want = tnn.scaledDotProductAttentionGQAWindow(q, k, v, window_size=300)
    for window in WINDOWS:
        assert torch.equal(tnn.scaledDotProductAttentionGQAWindow(q, k, v, window_size=window), want), window
    for bad in (0, -1, -2 ** 31, -2 ** 32, -2 ** 32 + 5):
        with pytest.raises(tnn.AttnError):
            tnn.scaledDotProductAttentionGQAWindow(q, k, v, window_size=bad)


def test_negative_windows_are_refused():
    q, k, v, d_o = (randn(1, 2, 64, 64, seed=i) for i in range(4))
    o, lse = tnn.attentionFwd(q, k, v)
    for bad in (-1, -2 ** 31, -2 ** 32, -2 ** 32 + 5):
        with pytest.raises(tnn.AttnError):
            tnn.attentionFwd(q, k, v, window_size=bad)
        with pytest.raises(tnn.AttnError):
            tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=bad)


def test_c_abi_with_the_greatest_window():
    """The C calls themselves, the one with first tokens given none of them too."""
    s, d = 200, 64
    q, k, v, d_o = (randn(1, 2, s, d, seed=i) for i in range(4))
    o, lse = tnn.attentionFwd(q, k, v, window_size=s)
    want = tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=s)
    L = _lib.load()
    got = [torch.zeros_like(t) for t in want]
    ws = torch.empty(int(L.tyr_b200_attn_backward_workspace_bytes(1, 2, s)), dtype=torch.uint8, device=DEV)
    a = _lib.BackwardArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), d_o=d_o.data_ptr(), lse=lse.data_ptr(),
                          d_q=got[0].data_ptr(), d_k=got[1].data_ptr(), d_v=got[2].data_ptr(), workspace=ws.data_ptr(),
                          workspace_bytes=ws.numel(), batch=1, n_head=2, n_kv_head=2, q_seq=s, kv_seq=s, head_dim=d, is_causal=1,
                          window_size=2 ** 31 - 1)
    for x in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        getattr(a, x + "_stride")[:] = [2 * s * d, s * d, d]
    st = torch.cuda.current_stream().cuda_stream
    for call in (lambda: L.tyr_b200_attn_backward(ctypes.byref(a), st), lambda: L.tyr_b200_attn_backward_sinks(ctypes.byref(a), 0, st)):
        for t in got:
            t.zero_()
        assert call() == 0
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert a.window_size == 2 ** 31 - 1
