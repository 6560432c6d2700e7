"""The paged KV cache on the GPU: append, single-token attention (window, first tokens, running sums of the weights) and
eviction, each against a plain implementation in float64, and a generating loop that uses all of them."""
import math

import pytest
import torch

from tyr_b200 import nn as tnn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = 2.0 ** -8          # half a step of bf16, relative
OUT_OF_RANGE = 4          # TYR_ATTN_STATUS_OUT_OF_RANGE


def randn(*shape, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(*shape, generator=g).bfloat16().to(DEV)


class Cache:
    """Pools with the sequences' pages scattered over them; rows that belong to no sequence are NaN."""

    def __init__(self, lens, n_kv_head, d, page, seed, layout="phrd", spare=3):
        need = [-(-n // page) for n in lens]
        g = torch.Generator().manual_seed(seed)
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g).int()
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.lens, self.page = list(lens), page
        self.k = [torch.randn(n, n_kv_head, d, generator=g).bfloat16() for n in lens]
        self.v = [torch.randn(n, n_kv_head, d, generator=g).bfloat16() for n in lens]
        order = {"phrd": (0, 1, 2, 3), "prhd": (0, 2, 1, 3), "hprd": (1, 0, 2, 3)}[layout]
        inverse = [order.index(i) for i in range(4)]
        shape = (n_pages, n_kv_head, page, d)
        # K and V in one allocation, K's strides are V's and neither is contiguous by itself
        both = torch.full((2,) + tuple(shape[i] for i in order), math.nan, dtype=torch.bfloat16)
        kp, vp = both[0].permute(inverse), both[1].permute(inverse)
        for b, n in enumerate(lens):
            j = torch.arange(n)
            kp[self.table[b, j // page].long(), :, j % page] = self.k[b]
            vp[self.table[b, j // page].long(), :, j % page] = self.v[b]
        both = both.to(DEV)
        self.kp, self.vp = both[0].permute(inverse), both[1].permute(inverse)
        assert self.kp.shape == shape
        self.table_dev = self.table.to(DEV)
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)


def definition(q, k, v, window=0, n_sink=0, scale=None):
    """One token over a sequence in float64: o, lse, the weights [n_head, keys], and what the errors are measured by."""
    n, hkv, d = k.shape
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    g = q.shape[0] // hkv
    scale = scale or d ** -0.5
    kh, vh = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("hd,jhd->hj", q, kh) * scale
    j = torch.arange(n)
    if window:
        s = s.masked_fill(~((j >= n - window) | (j < n_sink)), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.softmax(s, -1)
    o = torch.einsum("hj,jhd->hd", p, vh)
    # |scores| are off by at most d + 2 roundings of the sum of their products' magnitudes
    ds = (d + 2) * 2.0 ** -24 * scale * torch.einsum("hd,jhd->hj", q.abs(), kh.abs()).amax(-1)
    return o, lse, p, torch.einsum("hj,jhd->hd", p, vh.abs()), ds


def check_token(o, lse, want):
    """P is rounded to bf16 before the product with V and O once at the end; scores, sums and exponentials are in 32 bits."""
    ro, rl, _, mag, ds = want
    tol = mag * (2 * HALF + 2 * ds[:, None] + 2.0 ** -18)
    err = (o.double().cpu() - ro).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    err = (lse.double().cpu() - rl).abs()
    assert bool((err <= ds + 2.0 ** -20 * (1 + rl.abs())).all()), float(err.max())


@pytest.fixture(autouse=True)
def _status():
    yield
    assert tnn.device_status(0, True) == 0


# lengths around pages, tiles and chunks; page sizes below, at and above a tile, and no power of two
@pytest.mark.parametrize("lens", [[1], [1, 0, 2, 15, 16, 17], [64, 63, 65, 129, 300], [2051, 5, 700], [20000]])
@pytest.mark.parametrize("page,layout", [(1, "phrd"), (7, "prhd"), (16, "phrd"), (64, "hprd"), (100, "prhd"), (4096, "phrd")])
def test_decode_lengths_and_pages(lens, page, layout):
    for hq, hkv, d in [(8, 2, 128), (6, 6, 64)]:
        c = Cache(lens, hkv, d, page, seed=len(lens) + page, layout=layout)
        q = randn(len(lens), hq, d, seed=page)
        o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=max(lens))
        o2, lse2 = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, total_kv_len=sum(lens))
        for b, n in enumerate(lens):
            if n == 0:
                assert not o[b].any() and torch.isneginf(lse[b]).all() and not o2[b].any() and torch.isneginf(lse2[b]).all()
                continue
            want = definition(q[b], c.k[b], c.v[b])
            check_token(o[b], lse[b], want)
            check_token(o2[b], lse2[b], want)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (16, 2), (9, 1), (40, 2), (17, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_groups(hq, hkv, d):
    c = Cache([333, 40], hkv, d, 16, seed=hq)
    q = randn(2, hq, d, seed=hq)
    o, lse = tnn.flashDecodePaged(q.unsqueeze(2), c.kp, c.vp, c.table_dev, c.lens_dev, scale=0.3)
    assert o.shape == (2, hq, 1, d) and lse.shape == (2, hq, 1)
    for b in range(2):
        check_token(o[b, :, 0], lse[b, :, 0], definition(q[b], c.k[b], c.v[b], scale=0.3))


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (64, 4), (100, 37), (1000, 4), (3000, 16), (10 ** 12, 5), (2, 5000)])
@pytest.mark.parametrize("page", [16, 24])
def test_decode_window_and_first_tokens(window, n_sink, page):
    lens = [1, 3, 64, 101, 1500, 2600, 0]
    for hq, hkv, d in [(8, 2, 128), (4, 4, 64)]:
        c = Cache(lens, hkv, d, page, seed=window % 97 + n_sink)
        # pages out of sight are given back: their entries are no pages any more
        for b, n in enumerate(lens):
            for at in range(-(-n // page)):
                lo, hi = at * page, min((at + 1) * page, n)
                if lo >= n_sink and hi <= n - window:
                    c.table[b, at] = -1
        table = c.table.to(DEV)
        q = randn(len(lens), hq, d, seed=5)
        w = torch.rand(len(lens), hkv, 2600, device=DEV)
        w0 = w.clone()
        o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, table, c.lens_dev, max_kv_seq=2600, window_size=window, n_sink=n_sink, weights=w)
        o1, lse1 = tnn.flashDecodePaged(q, c.kp, c.vp, table, c.lens_dev, max_kv_seq=2600, window_size=window, n_sink=n_sink)
        assert torch.equal(o, o1) and torch.equal(lse, lse1)
        for b, n in enumerate(lens):
            if n == 0:
                assert not o[b].any() and torch.equal(w[b], w0[b])
                continue
            want = definition(q[b], c.k[b], c.v[b], min(window, 10 ** 6), n_sink)
            check_token(o[b], lse[b], want)
            check_sums(w[b], w0[b], want, hkv, n)


def check_sums(w, w0, want, hkv, n):
    """A weight is 2^(score - lse): the score's and the LSE's errors come in relative to it; one rounding for each addition."""
    _, rl, p, _, ds = want
    add = p.view(hkv, -1, n).sum(1)
    rel = (2 * ds + 2.0 ** -19 * (1 + rl.abs())).amax()
    got, base = w[:, :n].double().cpu(), w0[:, :n].double().cpu()
    assert bool(((got - base - add).abs() <= add * rel + (base + add) * 2.0 ** -23).all())
    assert torch.equal(w[:, n:], w0[:, n:])


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (20, 1, 128)])
def test_weights_add_up(hq, hkv, d):
    lens = [700, 1, 4100]
    c = Cache(lens, hkv, d, 32, seed=3)
    wide = torch.rand(3, hkv + 1, 4200, device=DEV)       # a view of a wider array
    w = wide[:, :hkv]
    w0, rest = w.clone(), wide[:, hkv:].clone()
    q = randn(3, hq, d, seed=8)
    _, lse = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=4100, weights=w, return_lse=False)
    assert lse is None
    for b, n in enumerate(lens):
        check_sums(w[b], w0[b], definition(q[b], c.k[b], c.v[b]), hkv, n)
    once = w.clone()
    w.copy_(w0)
    tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=4100, weights=w)
    assert torch.equal(w, once) and torch.equal(wide[:, hkv:], rest)


def test_bad_lengths_and_pages_are_reported():
    c = Cache([100, 200, 50, 70], 2, 64, 16, seed=1)
    q = randn(4, 4, 64, seed=2)
    lens = torch.tensor([100, 500, -3, 70], dtype=torch.int32, device=DEV)
    o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, lens, max_kv_seq=200)
    assert tnn.device_status(0, True) == OUT_OF_RANGE
    for b, n in ((0, 100), (1, 200), (3, 70)):
        check_token(o[b], lse[b], definition(q[b], c.k[b], c.v[b]))
    assert not o[2].any() and torch.isneginf(lse[2]).all()
    for entry in (-1, c.kp.shape[0], 2 ** 31 - 1):
        table = c.table_dev.clone()
        table[1, 5] = entry
        o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, table, c.lens_dev, max_kv_seq=200)
        assert tnn.device_status(0, True) == OUT_OF_RANGE
        assert torch.isnan(o[1]).all() and torch.isnan(lse[1]).all()
        for b in (0, 2, 3):
            check_token(o[b], lse[b], definition(q[b], c.k[b], c.v[b]))


def test_keys_that_score_minus_infinity_have_no_weight():
    c = Cache([90], 1, 64, 16, seed=4)
    q = randn(1, 2, 64, seed=4).abs() + 1
    c.k[0][:40] = -3e38                                     # the products overflow to -inf
    j = torch.arange(40)
    c.kp[c.table[0, j // 16].long().to(DEV), :, (j % 16).to(DEV)] = c.k[0][:40].to(DEV)
    w = torch.zeros(1, 1, 90, device=DEV)
    o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=90, weights=w)
    check_token(o[0], lse[0], definition(q[0], c.k[0][40:], c.v[0][40:]))
    assert not w[0, 0, :40].any() and (w[0, 0, 40:] > 0).all()


def test_strided_query_and_outputs_another_stream_and_a_graph():
    c = Cache([1000, 37], 2, 128, 16, seed=9)
    wide = randn(2, 3, 8, 128, seed=9)
    q = wide[:, 1]                                          # the query part of a fused projection
    o_wide = torch.zeros(2, 3, 8, 128, dtype=torch.bfloat16, device=DEV)
    o, lse = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=1000, out=o_wide[:, 1])
    assert not o_wide[:, 0].any() and not o_wide[:, 2].any()
    for b in range(2):
        check_token(o_wide[b, 1], lse[b], definition(q[b], c.k[b], c.v[b]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, _ = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=1000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, o)
    w = torch.zeros(2, 2, 1000, device=DEV)
    ws = torch.empty(tnn.paged_decode_workspace_bytes(q, c.kp, c.vp, c.table_dev, c.lens_dev, 1000, weights=w), dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, lse3 = tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=1000, weights=w, workspace=ws)
    for _ in range(2):
        graph.replay()
    assert torch.equal(o3, o) and torch.equal(lse3, lse)
    one = torch.zeros_like(w)
    tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=1000, weights=one)
    assert torch.equal(w, one + one)


# --------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,layout", [(1, "phrd"), (16, "prhd"), (100, "phrd")])
def test_append(d, page, layout):
    B, S, H, eps = 3, 37, 5, 1e-6
    start = [0, 15, 211]
    c = Cache([n + S for n in start], H, d, page, seed=d + page, layout=layout)
    before = c.kp.clone()
    g = torch.Generator().manual_seed(d)
    x = randn(B, S, H, d, seed=d)
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(DEV)
    ang = torch.arange(260.0)[:, None] * (10000.0 ** (-torch.arange(0, d, 2) / d))[None]
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    pos = torch.tensor(start, dtype=torch.int32, device=DEV)
    assert tnn.qkPrologue(x, c.kp, w, cos, sin, positions=pos, eps=eps, page_table=c.table_dev) is c.kp
    at = torch.tensor(start)[:, None] + torch.arange(S)[None]
    y = x.double().cpu()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double().cpu()
    y1, y2 = y[..., :d // 2], y[..., d // 2:]
    cs, sn = cos.double().cpu()[at][:, :, None], sin.double().cpu()[at][:, :, None]
    want = torch.cat([y1 * cs - y2 * sn, y1 * sn + y2 * cs], -1)
    mag = torch.cat([(y1 * cs).abs() + (y2 * sn).abs(), (y1 * sn).abs() + (y2 * cs).abs()], -1)
    page_of = torch.gather(c.table, 1, at // page).long().to(DEV)
    got = c.kp[page_of, :, (at % page).to(DEV)]
    # one rounding to bf16; before it the norm (a sum of d squares) and the rotation in 32 bits
    assert bool(((got.double().cpu() - want).abs() <= HALF * want.abs() + mag * (d + 8) * 2.0 ** -24).all())
    before[page_of, :, (at % page).to(DEV)] = got
    assert torch.equal(c.kp.view(torch.int16), before.view(torch.int16))     # nothing else was written
    # values: no norm, no rotation, a row of its own
    rows = torch.tensor([0, 9, 100], dtype=torch.int32, device=DEV)
    tnn.qkPrologue(x, c.vp, page_table=c.table_dev, rows=rows, position0=5000)
    at = torch.tensor([0, 9, 100])[:, None] + torch.arange(S)[None]
    page_of = torch.gather(c.table, 1, at // page).long().to(DEV)
    assert torch.equal(c.vp[page_of, :, (at % page).to(DEV)], x)
    # the rotary row by the position, the cache row by `rows`: the bits of the first call
    k2 = torch.zeros_like(c.kp)
    tnn.qkPrologue(x, k2, w, cos, sin, positions=pos, eps=eps, page_table=c.table_dev, rows=rows)
    assert torch.equal(k2[page_of, :, (at % page).to(DEV)], got)


def test_append_skips_rows_without_a_place():
    c = Cache([40, 40], 2, 64, 16, seed=2, spare=1)
    table = c.table_dev[:, :3].clone()
    table[0, 1] = c.kp.shape[0]                             # no page of the pool
    x = randn(2, 20, 2, 64, seed=3)
    for positions, good in (([10, 0], [(0, range(0, 6)), (1, range(20))]),            # rows 16.. of sequence 0 lie in the bad page
                            ([-4, 40], [(1, range(8))])):                              # before the first row; behind the last
        pool = torch.zeros_like(c.kp)
        tnn.qkPrologue(x, pool, positions=torch.tensor(positions, dtype=torch.int32, device=DEV), page_table=table)
        assert tnn.device_status(0, True) == OUT_OF_RANGE
        want = torch.zeros_like(pool)
        for b, tokens in good:
            for s in tokens:
                r = positions[b] + s
                want[table[b, r // 16], :, r % 16] = x[b, s]
        if positions[0] == -4:
            for s in range(4, 20):
                if (s - 4) // 16 != 1:
                    want[table[0, 0], :, s - 4] = x[0, s]
        assert torch.equal(pool, want)


# -------------------------------------------------------------------------------------------- eviction
def plain_evict(k, v, w, n_keep, n_recent, n_sink):
    """k, v [n, heads, d], w [heads, n]: what is left, per head."""
    n = w.shape[1]
    if n <= n_keep:
        return [list(range(n)) for _ in range(w.shape[0])]
    out = []
    for h in range(w.shape[0]):
        always = set(range(n_sink)) | set(range(n - n_recent, n))
        key = [(-math.inf if math.isnan(x) else x) for x in w[h].tolist()]
        nan = [math.isnan(x) for x in w[h].tolist()]
        rest = sorted((i for i in range(n) if i not in always), key=lambda i: (nan[i], -key[i], i))
        out.append(sorted(always | set(rest[:n_keep - len(always)])))
    return out


def evict_case(lens, hkv, d, page, n_keep, n_recent, n_sink, weights, layout="phrd", seed=0):
    c = Cache(lens, hkv, d, page, seed=seed, layout=layout)
    most = weights.shape[2]
    w = weights.to(DEV)
    k0, v0 = c.kp.clone(), c.vp.clone()
    new, kept = tnn.evictPaged(c.kp, c.vp, c.table_dev, c.lens_dev, w, n_keep, n_recent, n_sink, max_kv_seq=most)
    assert new.tolist() == [min(n, n_keep) for n in lens] and c.lens_dev.tolist() == list(lens)
    want_w = weights.clone()
    for b, n in enumerate(lens):
        left = plain_evict(c.k[b], c.v[b], weights[b, :, :n], n_keep, n_recent, n_sink)
        for h in range(hkv):
            ids = left[h]
            assert kept[b, h].tolist() == ids + [-1] * (n_keep - len(ids)), (b, h)
            if n > n_keep:
                row = weights[b, h, ids].clone()
                want_w[b, h, :n] = 0
                want_w[b, h, :n_keep] = row
            j = torch.arange(len(ids))
            at, off = c.table[b, j // page].long().to(DEV), (j % page).to(DEV)
            k0[at, h, off] = c.k[b][ids, h].to(DEV)
            v0[at, h, off] = c.v[b][ids, h].to(DEV)
    for got, want in ((c.kp, k0), (c.vp, v0)):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))     # every other row as it was, the NaN rows too
    assert torch.equal(w.cpu().view(torch.int32), want_w.view(torch.int32))


@pytest.mark.parametrize("n_keep,n_recent,n_sink", [(1, 0, 0), (1, 1, 0), (8, 4, 4), (100, 30, 4), (333, 0, 0), (1000, 999, 1), (500, 100, 0)])
@pytest.mark.parametrize("page,layout,d", [(16, "phrd", 128), (7, "prhd", 64), (1, "phrd", 256), (4096, "hprd", 128)])
def test_evict(n_keep, n_recent, n_sink, page, layout, d):
    g = torch.Generator().manual_seed(n_keep)
    lens = [n_keep, n_keep + 1, 1, 0, 1500, 1023]
    w = torch.exp(2 * torch.randn(6, 3, 1500, generator=g))
    evict_case(lens, 3, d, page, n_keep, n_recent, n_sink, w, layout, seed=n_keep)


@pytest.mark.parametrize("kind", ["equal", "few values", "zeros of both signs", "not numbers", "close together"])
def test_evict_ties_and_odd_weights(kind):
    g = torch.Generator().manual_seed(7)
    w = torch.rand(2, 2, 5000, generator=g)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few values":
        w = (w * 4).floor()
    elif kind == "zeros of both signs":
        w = torch.where(w < 0.5, -0.0, 0.0)
        w[:, :, ::100] = -1.0
        w[:, :, 50::100] = 1e-42                              # below the smallest normal number
    elif kind == "not numbers":
        w[w < 0.3] = math.nan
        w[(w > 0.3) & (w < 0.5)] = -math.inf
        w[w > 0.9] = math.inf
    else:
        w = 1 + torch.randint(0, 8, w.shape, generator=g) * 2.0 ** -23
    for n_keep in (700, 2400, 4999):
        evict_case([5000, 4100], 2, 64, 16, n_keep, 100, 4, w, seed=1)


# what one CTA holds, clusters of 2 to 16, and past them; ties across the CTAs' borders, sequences that end in an early CTA
@pytest.mark.parametrize("lens,n_keep", [([16384, 8192, 8193], 5000), ([16385, 16384, 20], 16384), ([40000, 17000], 16000), ([140000, 100000, 3000], 70000),
                                         ([262144, 200000], 1000), ([262145, 300], 200000)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long(lens, n_keep, ties):
    g = torch.Generator().manual_seed(n_keep)
    w = torch.rand(len(lens), 1, max(lens), generator=g)
    if ties:
        w = (w * 3).floor()
    evict_case(lens, 1, 64, 64, n_keep, n_keep // 3, 7, w, seed=4)


# enough (sequence, KV head) pairs for whole columns of 128 bytes per CTA; several steps of moves, ends inside a step
@pytest.mark.parametrize("d,page,layout", [(64, 16, "phrd"), (128, 7, "prhd"), (256, 100, "hprd")])
@pytest.mark.parametrize("n_keep,n_recent,n_sink", [(1, 0, 0), (130, 30, 4), (500, 0, 1), (127, 127, 0)])
def test_evict_many(d, page, layout, n_keep, n_recent, n_sink):
    g = torch.Generator().manual_seed(n_keep + d)
    lens = [int(n) for n in torch.randint(0, 900, (40,), generator=g)]
    w = torch.rand(40, 4, 900, generator=g)
    evict_case(lens, 4, d, page, n_keep, n_recent, n_sink, w[:, :, :max(lens)].contiguous(), layout, seed=d)
    assert 2 * (d // 64) * 4 * 40 >= 2 * torch.cuda.get_device_properties(0).multi_processor_count


def test_evict_many_with_a_bad_page():
    lens = [300] * 40
    c = Cache(lens, 4, 64, 16, seed=3)
    table = c.table_dev.clone()
    table[7, 3] = c.kp.shape[0]                             # rows 48.. of sequence 7 have no place
    k0 = c.kp.clone()
    w = torch.rand(40, 4, 300, device=DEV)
    sums = w.cpu()
    _, kept = tnn.evictPaged(c.kp, c.vp, table, c.lens_dev, w, 100, 10)
    assert tnn.device_status(0, True) == OUT_OF_RANGE
    for b in range(40):
        left = plain_evict(None, None, sums[b], 100, 10, 0)
        for h in range(4):
            assert kept[b, h].tolist() == left[h]
            for i, src in enumerate(left[h]):
                if b == 7 and (i // 16 == 3 or src // 16 == 3) and src != i:
                    if i // 16 != 3:                        # stays as it was
                        at, off = int(c.table[b, i // 16]), i % 16
                        assert torch.equal(c.kp[at, h, off].view(torch.int16), k0[at, h, off].view(torch.int16))
                    continue
                if b in (0, 7, 39):
                    assert torch.equal(c.kp[int(c.table[b, i // 16]), h, i % 16], c.k[b][src, h].to(DEV))
    other = int(c.table[7, 3])                              # the page that the table no longer names
    assert torch.equal(c.kp[other].view(torch.int16), k0[other].view(torch.int16))


def test_evict_large_and_reported():
    g = torch.Generator().manual_seed(11)
    evict_case([40000, 9000], 2, 64, 64, 8192, 1000, 4, torch.rand(2, 2, 40000, generator=g), seed=2)
    c = Cache([100, 100], 1, 64, 16, seed=3)
    w = torch.rand(2, 1, 100, device=DEV)
    lens = torch.tensor([-5, 400], dtype=torch.int32, device=DEV)
    new, kept = tnn.evictPaged(c.kp, c.vp, c.table_dev, lens, w, 50, 10)
    assert new.tolist() == [0, 50] and tnn.device_status(0, True) == OUT_OF_RANGE and (kept[0] == -1).all()
    c = Cache([100], 1, 64, 16, seed=3)
    table = c.table_dev.clone()
    table[0, 6] = -1
    k0 = c.kp.clone()
    tnn.evictPaged(c.kp, c.vp, table, c.lens_dev, torch.rand(1, 1, 100, device=DEV), 50, 10)   # rows 96.. have no place
    assert tnn.device_status(0, True) == OUT_OF_RANGE
    j = torch.arange(46, 50)
    at, off = c.table[0, j // 16].long().to(DEV), (j % 16).to(DEV)
    assert torch.equal(c.kp[at, 0, off], k0[at, 0, off])


# --------------------------------------------------------------------------------------- all of them
@pytest.mark.parametrize("window", [0, 60])
def test_generating_loop_with_a_budget(window):
    """Prompt into pages, tokens one by one with running sums, eviction when a budget is passed, then on: every step against
    attention in float64 over the keys that the loop should hold."""
    hq, hkv, d, page, budget = 8, 2, 64, 16, 90
    lens = [80, 33]
    c = Cache([0, 0], hkv, d, page, seed=1, spare=40)
    table = torch.arange(20, dtype=torch.int32).view(2, 10).to(DEV)
    c.kp.zero_(), c.vp.zero_()
    ang = torch.arange(400.0)[:, None] * (10000.0 ** (-torch.arange(0, d, 2) / d))[None]
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    w = torch.zeros(2, hkv, 160, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    xk, xv = randn(2, 80, hkv, d, seed=1), randn(2, 80, hkv, d, seed=2)
    tnn.qkPrologue(xk, c.kp, None, cos, sin, positions=zero, page_table=table)      # (rows behind a shorter prompt are overwritten)
    tnn.qkPrologue(xv, c.vp, page_table=table)

    def rows(pool, b, n):
        j = torch.arange(n, device=DEV)
        return pool[table[b, j // page].long(), :, j % page].cpu()

    held = [[(rows(c.kp, b, n)[:, h], rows(c.vp, b, n)[:, h], torch.zeros(n, dtype=torch.float64)) for h in range(hkv)]
            for b, n in enumerate(lens)]
    cached = torch.tensor(lens, dtype=torch.int32, device=DEV)
    text = cached.clone()
    for step in range(40):
        xk, xv, q = randn(2, 1, hkv, d, seed=100 + step), randn(2, 1, hkv, d, seed=200 + step), randn(2, hq, 1, d, seed=300 + step)
        tnn.qkPrologue(xk, c.kp, None, cos, sin, positions=text, page_table=table, rows=cached)
        tnn.qkPrologue(xv, c.vp, page_table=table, rows=cached)
        qr = torch.empty(2, hq, 1, d, dtype=torch.bfloat16, device=DEV)
        tnn.qkPrologue(q.transpose(1, 2), qr, None, cos, sin, positions=text, out_at_row0=True)
        cached, text = cached + 1, text + 1
        o, lse = tnn.flashDecodePaged(qr, c.kp, c.vp, table, cached, max_kv_seq=160, window_size=window, n_sink=4 if window else 0,
                                      weights=w)
        for b in range(2):
            n = int(cached[b])
            new_k, new_v = rows(c.kp, b, n)[-1], rows(c.vp, b, n)[-1]
            assert torch.equal(new_v, xv[b, 0].cpu())
            for h in range(hkv):
                k, v, s = held[b][h]
                k, v = torch.cat([k, new_k[None, h]]), torch.cat([v, new_v[None, h]])
                sel = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                want = definition(qr[b, sel, 0], k[:, None], v[:, None], window, 4 if window else 0)
                check_token(o[b, sel, 0], lse[b, sel, 0], want)
                held[b][h] = (k, v, torch.cat([s, torch.zeros(1, dtype=torch.float64)]) + want[2].sum(0))
                assert torch.allclose(w[b, h, :n].double().cpu(), held[b][h][2], rtol=1e-4, atol=1e-6)
        if int(cached.max()) >= 120:
            before = w.clone()
            cached, kept = tnn.evictPaged(c.kp, c.vp, table, cached, w, budget, 20, 4)
            for b in range(2):
                for h in range(hkv):
                    ids = [i for i in kept[b, h].tolist() if i >= 0]
                    assert ids == plain_evict(None, None, before[b, h:h + 1, :len(held[b][h][0])].cpu(), budget, 20, 4)[0]
                    held[b][h] = tuple(t[ids] for t in held[b][h])
    assert int(cached.max()) < int(text.max())                # the budget was passed on the way


def test_table_and_lengths_rewritten_between_calls():
    """The table and the lengths are the device's: each call sees what the kernel before it on the stream wrote."""
    page, n_pages, hkv, d = 16, 400, 2, 64
    g = torch.Generator().manual_seed(5)
    kp, vp = (torch.randn(n_pages, hkv, page, d, generator=g).bfloat16() for _ in range(2))
    kd, vd = kp.to(DEV), vp.to(DEV)
    q = randn(3, 4, d, seed=6)
    plans = [(torch.stack([torch.randperm(n_pages, generator=g)[:60] for _ in range(3)]).int(), torch.randint(1, 961, (3,), generator=g).int())
             for _ in range(12)]
    on_dev = [(t.to(DEV), n.to(DEV)) for t, n in plans]
    table, lens = torch.zeros(3, 60, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    ws = torch.empty(tnn.paged_decode_workspace_bytes(q, kd, vd, table, lens), dtype=torch.uint8, device=DEV)
    out = []
    for t, n in on_dev:
        table.copy_(t)
        lens.copy_(n)
        out.append(tnn.flashDecodePaged(q, kd, vd, table, lens, workspace=ws))
    for (t, n), (o, lse) in zip(plans, out):
        for b in range(3):
            j = torch.arange(int(n[b]))
            at = t[b, j // page].long()
            check_token(o[b], lse[b], definition(q[b], kp[at, :, j % page], vp[at, :, j % page]))


def test_calls_on_two_streams_with_workspaces_of_their_own():
    lens = [30000, 20000]
    c = Cache(lens, 2, 128, 16, seed=12)
    qs = [randn(2, 8, 128, seed=s) for s in (1, 2)]
    want = [tnn.flashDecodePaged(q, c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=30000) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(tnn.flashDecodePaged(qs[i], c.kp, c.vp, c.table_dev, c.lens_dev, max_kv_seq=30000))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i][0]) and torch.equal(l, want[i][1]) for o, l in got[i])


def test_loop_with_eviction_as_a_graph():
    """One captured step (append, attention with sums, the counters) replayed, and a captured eviction, against the eager calls."""
    hq, hkv, d, page, cap = 8, 2, 64, 16, 320
    xs = [(randn(2, 1, hkv, d, seed=10 + i), randn(2, 1, hkv, d, seed=60 + i), randn(2, hq, d, seed=110 + i)) for i in range(30)]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int().view(2, 20).to(DEV)

    def run(graphs):
        kp, vp = (torch.zeros(40, hkv, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        sums = torch.zeros(2, hkv, cap, device=DEV)
        n, n2 = torch.tensor([3, 200], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
        kept = torch.zeros(2, hkv, 150, dtype=torch.int32, device=DEV)
        xk, xv, q = (torch.zeros_like(t) for t in xs[0])
        o, lse = torch.zeros(2, hq, d, dtype=torch.bfloat16, device=DEV), torch.zeros(2, hq, device=DEV)
        ws = torch.empty(tnn.paged_decode_workspace_bytes(q, kp, vp, table, n, cap, weights=sums), dtype=torch.uint8, device=DEV)

        def step():
            tnn.qkPrologue(xk, kp, positions=n, page_table=table)
            tnn.qkPrologue(xv, vp, positions=n, page_table=table)
            n.add_(1)
            tnn.flashDecodePaged(q, kp, vp, table, n, max_kv_seq=cap, weights=sums, out=o, lse=lse, workspace=ws)

        def evict():
            tnn.evictPaged(kp, vp, table, n, sums, 150, 40, 4, max_kv_seq=cap, new_lens=n2, kept=kept)
            n.copy_(n2)

        if graphs:
            calls = []
            for f in (step, evict):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    f()
                calls.append(g.replay)
            one, drop = calls
        else:
            one, drop = step, evict
        seen = []
        for i, x in enumerate(xs):
            for to, t in zip((xk, xv, q), x):
                to.copy_(t)
            one()
            seen += [o.clone(), lse.clone()]
            if i % 10 == 9:
                drop()
                seen += [n.clone(), kept.clone(), kp.clone(), vp.clone(), sums.clone()]
        return seen

    eager, replayed = run(False), run(True)
    assert len(eager) == len(replayed) and all(torch.equal(a, b) for a, b in zip(eager, replayed))
    assert eager[-5].tolist() == [33, 150]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rotary", ["none", "halves", "pairs"])
def test_append_gives_the_bits_of_the_dense_call(d, rotary):
    B, S, H, page = 2, 53, 6, 24
    x, w = randn(B, S, H, d, seed=3).transpose(1, 2).contiguous().transpose(1, 2), torch.rand(d, device=DEV) + 0.5      # heads outer
    start = torch.tensor([40, 5], dtype=torch.int32, device=DEV)
    ang = torch.arange(100.0, device=DEV)[:, None] * torch.rand(d // 2, device=DEV)[None]
    cos, sin = ang.cos().contiguous(), ang.sin().contiguous()
    rot = {"none": {}, "halves": dict(cos=cos, sin=sin),
           "pairs": dict(pe=torch.stack([cos, -sin, sin, cos], -1).view(1, 100, d // 2, 2, 2).contiguous())}[rotary]
    dense = torch.zeros(B, H, 100, d, dtype=torch.bfloat16, device=DEV)
    tnn.qkPrologue(x, dense, w, positions=start, **rot)
    pool = torch.zeros(11, page, H, d, dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    table = torch.tensor([[9, 2, 7, 0, 4], [1, 10, 3, 8, 6]], dtype=torch.int32, device=DEV)
    tnn.qkPrologue(x, pool, w, positions=start, page_table=table, **rot)
    j = torch.arange(100, device=DEV)
    for b in range(B):
        assert torch.equal(pool[table[b, j // page].long(), :, j % page].transpose(0, 1), dense[b])


def test_pages_far_apart():
    """Pages 2^26 rows' worth of elements apart (offsets past 32 bits), V laid out in another way than K."""
    hkv, d, page, n_pages = 2, 64, 16, 40
    far = torch.empty(n_pages * 2 ** 26, dtype=torch.bfloat16, device=DEV)            # 5.4 GB
    kp = far.as_strided((n_pages, hkv, page, d), (2 ** 26, 2 ** 20, 1024, 1))
    vp = torch.zeros(hkv, n_pages, page, d, dtype=torch.bfloat16, device=DEV).transpose(0, 1)
    table = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=DEV).view(1, n_pages)
    xk, xv, q = randn(1, 600, hkv, d, seed=1), randn(1, 600, hkv, d, seed=2), randn(1, 4, d, seed=3)
    tnn.qkPrologue(xk, kp, page_table=table)
    tnn.qkPrologue(xv, vp, page_table=table)
    lens, w = torch.tensor([600], dtype=torch.int32, device=DEV), torch.zeros(1, hkv, 640, device=DEV)
    o, lse = tnn.flashDecodePaged(q, kp, vp, table, lens, weights=w)
    want = definition(q[0], xk[0].cpu(), xv[0].cpu())
    check_token(o[0], lse[0], want)
    sums = w.clone()
    lens, kept = tnn.evictPaged(kp, vp, table, lens, w, 300, 50, 4)
    for h, left in enumerate(plain_evict(None, None, sums[0, :, :600].cpu(), 300, 50, 4)):
        assert kept[0, h].tolist() == left
        j = torch.arange(300, device=DEV)
        at = table[0, j // page].long()
        assert torch.equal(kp[at, h, j % page], xk[0, left, h]) and torch.equal(vp[at, h, j % page], xv[0, left, h])
    del far


def test_calls_on_the_other_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs in one process")
    torch.cuda.set_device(0)
    c = Cache([500, 20000], 2, 64, 16, seed=4)
    q, w = randn(2, 4, 64, seed=5), torch.rand(2, 2, 20000, device=DEV)
    got = []
    for dev in ("cuda:0", "cuda:1"):
        kp, vp, table, lens, ws, qd = (t.to(dev).clone() for t in (c.kp, c.vp, c.table_dev, c.lens_dev, w, q))
        o, lse = tnn.flashDecodePaged(qd, kp, vp, table, lens, max_kv_seq=20000, weights=ws)
        new, kept = tnn.evictPaged(kp, vp, table, lens, ws, 400, 30, 4, max_kv_seq=20000)
        tnn.qkPrologue(qd.view(2, 1, 4, 64)[:, :, :2], kp, positions=new, page_table=table)
        got.append([t.cpu() for t in (o, lse, ws, new, kept)] + [kp.cpu().view(torch.int16)])
    assert torch.cuda.current_device() == 0 and tnn.device_status(1, True) == 0
    assert all(torch.equal(a, b) for a, b in zip(*got))
