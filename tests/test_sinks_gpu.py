"""First tokens that stay visible beside a sliding window, forward and backward on the GPU, against the definition in float64
(plain_sinks.py, which says where the tolerances come from)."""
import pytest
import torch

import plain_sinks as plain
from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def randn(*shape, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(*shape, generator=g).bfloat16()


@pytest.fixture(autouse=True)
def _status():
    yield
    assert tnn.device_status(0, True) == 0


def run_case(B, Hq, Hkv, S, D, window, n_sink, scale=None, grads=True):
    q, k, v, d_o = (randn(B, h, S, D, seed=S + 7 * i + window) for i, h in enumerate((Hq, Hkv, Hkv, Hq)))
    qd, kd, vd, dd = (t.to(DEV) for t in (q, k, v, d_o))
    o, lse = tnn.attentionFwd(qd, kd, vd, scale=scale, window_size=window, n_sink=n_sink)
    ro, rl, _, _, tol_o, tol_l = plain.forward(q, k, v, window, n_sink, scale)
    plain.check(o, ro, tol_o, "o")
    plain.check(lse, rl, tol_l, "lse")
    if grads:
        got = tnn.attentionBwd(qd, kd, vd, o, lse, dd, scale=scale, window_size=window, n_sink=n_sink)
        for g, (w, tol), name in zip(got, plain.backward(q, k, v, d_o, window, n_sink, scale), ("d_q", "d_k", "d_v")):
            plain.check(g, w, tol, name)


# one key and query, ends of tiles, windows below, at and above a tile, first tokens in one tile and in several
@pytest.mark.parametrize("S,window,n_sink", [(1, 1, 1), (2, 1, 1), (127, 5, 1), (128, 128, 4), (129, 1, 1), (300, 40, 4), (384, 128, 128),
                                             (640, 64, 129), (700, 1, 300), (900, 256, 4), (900, 257, 16), (1500, 130, 1), (1500, 2000, 4),
                                             (517, 128, 10 ** 12), (1111, 300, 200)])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 64), (2, 2, 128), (6, 2, 128)])
def test_against_the_definition(S, window, n_sink, Hq, Hkv, D):
    run_case(1, Hq, Hkv, S, D, window, min(n_sink, 10 ** 12))


# enough work items for the plain schedule of the forward, units of the backward cut and merged, several rounds
@pytest.mark.parametrize("B,Hq,Hkv,S,D,window,n_sink", [(1, 2, 1, 2300, 128, 128, 4), (1, 4, 2, 2177, 64, 1, 2), (2, 2, 2, 2048, 64, 300, 150),
                                                         (1, 1, 1, 4097, 128, 64, 1), (3, 8, 4, 700, 64, 100, 4), (40, 2, 1, 260, 128, 50, 4)])
def test_larger_launches(B, Hq, Hkv, S, D, window, n_sink):
    run_case(B, Hq, Hkv, S, D, window, n_sink, scale=0.11)


def test_no_first_tokens_is_the_windowed_call_and_all_is_the_causal_one():
    q, k, v, d_o = (randn(1, h, 600, 128, seed=h).to(DEV) for h in (4, 2, 2, 4))
    a, b = tnn.attentionFwd(q, k, v, window_size=100), tnn.attentionFwd(q, k, v, window_size=100, n_sink=0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # everything visible: the causal call, up to the order of sums
    o, lse = tnn.attentionFwd(q, k, v, window_size=5, n_sink=600)
    oc, lc = tnn.attentionFwd(q, k, v, is_causal=True)
    assert (o.float() - oc.float()).abs().max().item() <= 2e-2 and (lse - lc).abs().max().item() <= 1e-4
    o2 = tnn.scaledDotProductAttentionGQAWindowSinks(q, k, v, 0.0, False, True, 100, 3)
    o3, _ = tnn.attentionFwd(q, k, v, window_size=100, n_sink=3)
    assert torch.equal(o2, o3)


def test_check_mode():
    q, k, v = (randn(2, h, 333, 80, seed=h).float() for h in (4, 2, 2))
    o, lse = tnn.attentionFwd(q.to(DEV), k.to(DEV), v.to(DEV), check_mode=True, window_size=50, n_sink=37)
    ro, rl, *_ = plain.forward(q, k, v, 50, 37)
    assert (o.double().cpu() - ro).abs().max() <= 1e-5 * ro.abs().max() and (lse.double().cpu() - rl).abs().max() <= 1e-5 * rl.abs().max()


def test_strided_views_and_poisoned_surroundings():
    """[batch, seq, heads, dim] buffers with NaN heads between those that are read, outputs in views."""
    B, S, D, window, n_sink = 2, 700, 128, 90, 5
    big = torch.full((B, S, 12, D), float("nan"), dtype=torch.bfloat16)
    q, k, v = randn(B, 4, S, D, seed=1), randn(B, 2, S, D, seed=2), randn(B, 2, S, D, seed=3)
    big[:, :, 0:4], big[:, :, 5:7], big[:, :, 9:11] = (t.transpose(1, 2) for t in (q, k, v))
    dev = big.to(DEV).transpose(1, 2)
    qd, kd, vd = dev[:, 0:4], dev[:, 5:7], dev[:, 9:11]
    out = torch.full((B, S, 4, D), float("nan"), dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    o, lse = tnn.attentionFwd(qd, kd, vd, window_size=window, n_sink=n_sink, out=out)
    ro, rl, _, _, tol_o, tol_l = plain.forward(q, k, v, window, n_sink)
    plain.check(out, ro, tol_o, "o")
    plain.check(lse, rl, tol_l, "lse")
    d_o = randn(B, 4, S, D, seed=4)
    got = tnn.attentionBwd(qd, kd, vd, o, lse, d_o.to(DEV), window_size=window, n_sink=n_sink)
    for g, (w, tol), name in zip(got, plain.backward(q, k, v, d_o, window, n_sink), ("d_q", "d_k", "d_v")):
        plain.check(g, w, tol, name)


@pytest.mark.parametrize("D", [64, 128])
def test_one_order_of_sums_for_long_calls(D):
    B, S, at = 5, 2200, dict(window_size=150, n_sink=4)
    t = [randn(B, h, S, D, seed=h + i).to(DEV) for i, h in enumerate((4, 2, 2, 4))]

    def both(t):
        o, lse = tnn.attentionFwd(*t[:3], **at)
        return (o, lse) + tnn.attentionBwd(*t[:3], o, lse, t[3], **at)

    whole = both(t)
    for a, b in zip(whole, both(t)):
        assert torch.equal(a, b)
    for a, b in zip(whole, both([x[3:4] for x in t])):
        assert torch.equal(a[3:4], b)


def test_own_workspace_another_stream_and_a_graph():
    S, at = 2500, dict(window_size=100, n_sink=3)
    q, k, v, d_o = (randn(1, h, S, 64, seed=h + 9).to(DEV) for h in (4, 2, 2, 4))
    o, lse = tnn.attentionFwd(q, k, v, **at)
    want = tnn.attentionBwd(q, k, v, o, lse, d_o, **at)
    ws = torch.empty(tnn.backward_sinks_workspace_bytes(q, k, 100, 3) // 4, dtype=torch.float32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tnn.attentionBwd(q, k, v, o, lse, d_o, workspace=ws, **at)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, lse2 = tnn.attentionFwd(q, k, v, **at)
        got = tnn.attentionBwd(q, k, v, o2, lse2, d_o, workspace=ws, **at)
    for _ in range(2):
        ws.fill_(float("nan"))
        graph.replay()
    assert torch.equal(o2, o) and all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError):
        tnn.attentionBwd(q, k, v, o, lse, d_o, workspace=ws[:-1], **at)


def test_gradients_against_differences():
    """Directional derivatives of sum(dO * O), O from the definition in float64, against the kernels' gradients."""
    S, window, n_sink = 200, 30, 3
    x = [randn(1, h, S, 64, seed=20 + h + i) for i, h in enumerate((4, 2, 2))]
    d_o = randn(1, 4, S, 64, seed=30)
    dev = [t.to(DEV) for t in x]
    o, lse = tnn.attentionFwd(*dev, window_size=window, n_sink=n_sink)
    got = tnn.attentionBwd(*dev, o, lse, d_o.to(DEV), window_size=window, n_sink=n_sink)
    tols = plain.backward(*x, d_o, window, n_sink)
    for i in range(3):
        u = randn(*x[i].shape, seed=40 + i).double()
        h = 1e-4
        loss = [float((plain.forward(*[t.double() + s * h * u if a == i else t for a, t in enumerate(x)], window, n_sink)[0] * d_o.double()).sum())
                for s in (1, -1)]
        slope = (loss[0] - loss[1]) / (2 * h)
        tol = float((tols[i][1] * u.abs()).sum()) + 1e-5 * abs(slope)
        assert abs(slope - float((got[i].double().cpu() * u).sum())) <= tol


def test_refusals():
    q, k, v = (randn(1, h, 64, 64, seed=h).to(DEV) for h in (2, 2, 2))
    m = torch.ones(1, 64, dtype=torch.uint8, device=DEV)
    for kw in (dict(n_sink=4), dict(n_sink=-1, window_size=4), dict(n_sink=4, window_size=4, key_mask=m), dict(n_sink=4, window_size=-1)):
        with pytest.raises(tnn.AttnError):
            tnn.attentionFwd(q, k, v, **kw)
    with pytest.raises(tnn.AttnError):
        tnn.scaledDotProductAttentionGQAWindowSinks(q, k, v, window_size=0, n_sink=4)
    with pytest.raises(tnn.AttnError):
        tnn.attentionFwd(q[:, :, :32], k, v, window_size=4, n_sink=2)


def test_on_the_other_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs in one process")
    torch.cuda.set_device(0)
    t = [randn(1, h, 2500, 64, seed=h + i) for i, h in enumerate((4, 2, 2, 4))]
    got = []
    for dev in ("cuda:0", "cuda:1"):
        q, k, v, d_o = (x.to(dev) for x in t)
        o, lse = tnn.attentionFwd(q, k, v, window_size=90, n_sink=4)
        got.append([x.cpu() for x in (o, lse, *tnn.attentionBwd(q, k, v, o, lse, d_o, window_size=90, n_sink=4))])
    assert torch.cuda.current_device() == 0 and tnn.device_status(1, True) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("n_sink", [0, 2])
def test_a_window_past_32_bits_is_all_keys(n_sink):
    torch.manual_seed(21)
    q, k, v = (torch.randn(1, 4, 300, 64, device="cuda").bfloat16() for _ in range(3))
    want = tnn.scaledDotProductAttentionGQAWindowSinks(q, k, v, window_size=300, n_sink=n_sink)
    for window in (2 ** 31 - 1, 2 ** 32, 2 ** 32 + 5):
        assert torch.equal(tnn.scaledDotProductAttentionGQAWindowSinks(q, k, v, window_size=window, n_sink=n_sink), want), window
