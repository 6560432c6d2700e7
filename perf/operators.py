"""Attention with a bounded view of its keys, and the paged KV cache that such models generate from, as they are timed.

A case is a dict of plain values; "path" names the operator that one pass goes through:

  sinks   attention with a causal sliding window and a few first tokens that every later row still sees
  train   the same forward with its row statistics, then dQ, dK and dV
  append  norm + rotary of new keys and their rows, and the new values, into a paged cache at each sequence's row
  decode  one new token per sequence over a paged cache, optionally with the window and the first tokens,
          optionally adding the weight each cached key got to a running sum
  evict   keeps the first, the most recent and the most weighted keys of every (sequence, KV head) of a paged cache

With `own` false a pass is elementary torch operations in 32 bits, rounded once at the end.

Model shapes are the repository's own: a char-level GPT (6 heads of 64), Qwen3-0.6B and Qwen3-8B (grouped-query
attention, heads of 128, Q and K normalised per head), and the generic ones of perf/cases.py.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# query heads, KV heads, head_dim, Q and K normalised per head
SHAPES = {
    "char": (6, 6, 64, False),
    "mha64": (12, 12, 64, False),
    "gqa64": (32, 8, 64, False),
    "qwen3_0p6b": (16, 8, 128, True),
    "qwen3_8b": (32, 8, 128, True),
}
EPS = 1e-6


def listed():
    return [
        # one chat prompt of odd length through a windowed layer: latency, few work items
        {"name": "sinks_one_prompt", "path": "sinks", "shape": "qwen3_8b", "batch": 1, "seq": 517, "window": 128, "n_sink": 4},
        # a long document of odd length, a thousand keys of window
        {"name": "sinks_long_prompt", "path": "sinks", "shape": "qwen3_8b", "batch": 1, "seq": 9001, "window": 1024, "n_sink": 4},
        # the char-level training run with a window of a quarter of its sequence and one first token
        {"name": "train_char", "path": "train", "shape": "char", "batch": 64, "seq": 256, "window": 64, "n_sink": 1},
        # a training step's attention at the 0.6B shape
        {"name": "train_long", "path": "train", "shape": "qwen3_0p6b", "batch": 2, "seq": 4096, "window": 1024, "n_sink": 4},
        # the new key and value of one step of 64 generating sequences
        {"name": "append_token", "path": "append", "shape": "qwen3_8b", "batch": 64, "seq": 1, "max_row": 600, "page": 16},
        # four prompts into the cache, behind what is there
        {"name": "append_prompt", "path": "append", "shape": "qwen3_8b", "batch": 4, "seq": 4096, "max_row": 100, "page": 64},
        # one user, one token: latency
        {"name": "decode_one", "path": "decode", "shape": "qwen3_8b", "batch": 1, "min_len": 1537, "max_len": 1537,
         "len_seed": 0, "page": 16, "window": 0, "n_sink": 0, "weights": False},
        # a serving batch: ragged lengths as in the repository's decode benchmark
        {"name": "decode_64_ragged", "path": "decode", "shape": "qwen3_8b", "batch": 64, "min_len": 512, "max_len": 32768,
         "len_seed": 3, "page": 64, "window": 0, "n_sink": 0, "weights": False},
        # long generations through a windowed layer: most of each sequence is out of sight
        {"name": "decode_window", "path": "decode", "shape": "qwen3_0p6b", "batch": 32, "min_len": 100, "max_len": 40000,
         "len_seed": 7, "page": 16, "window": 4096, "n_sink": 4, "weights": False},
        # the step of a cache that will be evicted from: the keys' weights are summed up
        {"name": "decode_weights", "path": "decode", "shape": "qwen3_8b", "batch": 16, "min_len": 4096, "max_len": 8192,
         "len_seed": 5, "page": 32, "window": 0, "n_sink": 0, "weights": True},
        # one sequence brought back to its budget, many equal weights
        {"name": "evict_one", "path": "evict", "shape": "qwen3_0p6b", "batch": 1, "min_len": 2049, "max_len": 2049,
         "len_seed": 0, "page": 16, "n_keep": 1024, "n_recent": 256, "n_sink": 4, "ties": True},
        # a serving batch of ragged lengths, some of them still within the budget
        {"name": "evict_batch", "path": "evict", "shape": "qwen3_8b", "batch": 32, "min_len": 2000, "max_len": 16384,
         "len_seed": 9, "page": 64, "n_keep": 4096, "n_recent": 1024, "n_sink": 4, "ties": False},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# What a drawn case costs at most: (score-matrix entries of the plain form, bytes), by the listed cases' largest.
_CAPS = {"sinks": (32 * 9001 ** 2, 1e9), "train": (32 * 4096 ** 2, 1e9), "append": (0, 0.3e9), "decode": (0, 4.4e9), "evict": (0, 1.1e9)}
_PAGES = (1, 8, 16, 24, 32, 64, 100, 128, 256)


def draw(rng: random.Random) -> dict:
    while True:
        c = _draw(rng)
        w, cap = work(c), _CAPS[c["path"]]
        hq, hkv, d, _ = SHAPES[c["shape"]]
        if c["path"] in ("sinks", "train") and c["batch"] * hq * c["seq"] ** 2 > cap[0]:
            continue
        # (the plain form of a decode takes every sequence as long as the longest)
        if c["path"] == "decode" and c["batch"] * hkv * d * min(c["max_len"], (c["window"] + c["n_sink"]) or c["max_len"]) > 64 * 8 * 128 * 32768:
            continue
        if w["bytes"] <= cap[1]:
            return c


def _draw(rng: random.Random) -> dict:
    path = rng.choice(["sinks", "train", "append", "decode", "decode", "evict"])
    c = {"path": path, "shape": rng.choice(list(SHAPES))}
    if path in ("sinks", "train"):
        c["batch"] = _log_int(rng, 1, 64)
        c["seq"] = _log_int(rng, 16, 9001 if path == "sinks" else 4096)
        c["window"] = _log_int(rng, 1, 4096)
        c["n_sink"] = rng.choice([1, 2, 4, 4, 16, 64, 130, 300])
    elif path == "append":
        c["batch"] = _log_int(rng, 1, 64)
        c["seq"] = rng.choice([1, 1, _log_int(rng, 2, 4096)])
        c["max_row"] = _log_int(rng, 1, 2000)
        c["page"] = rng.choice(_PAGES)
    elif path == "decode":
        c["batch"] = _log_int(rng, 1, 96)
        c["max_len"] = _log_int(rng, 1, 40000)
        c["min_len"] = max(1, c["max_len"] // rng.choice([1, 2, 8, 64]))
        c["len_seed"] = rng.randrange(1 << 20)
        c["page"] = rng.choice(_PAGES)
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 8192)])
        c["n_sink"] = rng.choice([0, 1, 4, 16, 100]) if c["window"] else 0
        c["weights"] = rng.random() < 0.4
    else:
        c["batch"] = _log_int(rng, 1, 64)
        c["max_len"] = _log_int(rng, 16, 16384)
        c["min_len"] = max(1, c["max_len"] // rng.choice([1, 2, 8]))
        c["len_seed"] = rng.randrange(1 << 20)
        c["page"] = rng.choice(_PAGES)
        c["n_keep"] = _log_int(rng, 4, c["max_len"])
        c["n_sink"] = rng.choice([0, 1, min(4, c["n_keep"] // 2)])
        c["n_recent"] = rng.randint(0, c["n_keep"] - c["n_sink"])
        c["ties"] = rng.random() < 0.5
    return c


def _lengths(case) -> list:
    """Cached keys of each sequence of a decode or evict case, or rows before the new ones of an append (the case alone decides)."""
    if case["path"] == "append":
        r = random.Random(case["max_row"])
        return [r.randint(0, case["max_row"]) for _ in range(case["batch"])]
    r = random.Random(case["len_seed"])
    return [case["max_len"]] + [r.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"] - 1)]


def _visible(case, n: int) -> int:
    """Keys that the new token of a sequence of n keys sees."""
    if not case["window"]:
        return n
    begin = max(0, n - case["window"])
    return n - begin + min(case["n_sink"], begin)


# ------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape, norm=False):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    if norm:  # QK-norm models hand over vectors of unit root mean square
        t = (t.float() / torch.sqrt(t.float().pow(2).mean(-1, keepdim=True) + EPS)).bfloat16()
    return t


def _rotary(max_pos, d):
    inv = 1.0 / (1.0e6 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
    ang = torch.arange(max_pos, device="cuda", dtype=torch.float32)[:, None] * inv[None]
    return ang.cos().contiguous(), ang.sin().contiguous()


def _page_table(gen, rows, page):
    """(table [batch, most pages], number of pages): every sequence's pages scattered over the pool, -1 behind its last."""
    need = [-(-n // page) for n in rows]
    total, most = sum(need), max(max(need), 1)
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    at = torch.arange(most, device="cuda")[None]
    n = torch.tensor(need, device="cuda")[:, None]
    first = torch.cumsum(n, 0) - n
    table = torch.where(at < n, ids[(first + at).clamp(max=total - 1)], -1).to(torch.int32)
    return table.contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, d, norm = SHAPES[case["shape"]]
    path, b = case["path"], case["batch"]
    s = {"case": case}
    if path in ("sinks", "train"):
        s["q"] = _randn(gen, b, hq, case["seq"], d, norm=norm)
        s["k"] = _randn(gen, b, hkv, case["seq"], d, norm=norm)
        s["v"] = _randn(gen, b, hkv, case["seq"], d)
        s["d_o"] = _randn(gen, b, hq, case["seq"], d) if path == "train" else None
        return s
    lens = _lengths(case)
    grown = [n + case["seq"] for n in lens] if path == "append" else lens
    s["table"], pages = _page_table(gen, grown, case["page"])
    # K is cached as the model leaves it, after norm and rotation; the pool is one allocation for each of K and V
    s["k_pages"] = _randn(gen, pages, hkv, case["page"], d)
    s["v_pages"] = _randn(gen, pages, hkv, case["page"], d)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if path == "append":
        s["x_k"], s["x_v"] = _randn(gen, b, case["seq"], hkv, d), _randn(gen, b, case["seq"], hkv, d)
        s["w"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda") if norm else None
        s["cos"], s["sin"] = _rotary(max(grown), d)
        return s
    s["total"] = sum(lens)  # the host of a serving loop knows the lengths it hands over
    if path == "decode":
        s["q"] = _randn(gen, b, hq, d, norm=norm)
        s["weights"] = torch.rand(b, hkv, max(lens), generator=gen, device="cuda") if case["weights"] else None
    else:
        # sums of softmax weights: many small ones, a few large
        w = torch.exp(2.0 * torch.randn(b, hkv, max(lens), generator=gen, device="cuda"))
        s["weights"] = torch.round(w * 4) / 4 if case["ties"] else w
    return s


# ------------------------------------------------------------------------------------- the plain forms
def _scores(q, k, case):
    """Scaled scores of the rows that share a KV head, [batch, KV heads, group, seq, seq], -inf where a key is out of sight."""
    b, hq, n, d = q.shape
    s = (q.float().view(b, k.shape[1], -1, n, d) @ k.float()[:, :, None].transpose(-1, -2)) * (1.0 / math.sqrt(d))
    i = torch.arange(n, device=q.device)
    far = i[:, None] - i[None, :]
    return s.masked_fill_(~((far >= 0) & ((far < case["window"]) | (i < case["n_sink"])[None, :])), -math.inf)


def _plain_forward(q, k, v, case):
    """O and the scores' log-sum-exp in 32 bits, and the softmax."""
    p = _scores(q, k, case)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p = p.div_(l)
    return p @ v.float()[:, :, None], (m + l.log())[..., 0], p


def _plain_sinks(s):
    o, lse, _ = _plain_forward(s["q"], s["k"], s["v"], s["case"])
    return {"o": o.view(s["q"].shape).bfloat16(), "lse": lse.view(s["q"].shape[:3])}


def _plain_train(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, hq, n, d = q.shape
    scale = 1.0 / math.sqrt(d)
    o, lse, p = _plain_forward(q, k, v, s["case"])
    d_o = s["d_o"].float().view(o.shape)
    d_v = (p.transpose(-1, -2) @ d_o).sum(2)
    d_s = d_o @ v.float()[:, :, None].transpose(-1, -2)
    d_s = d_s.sub_((d_o * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    d_q = d_s @ k.float()[:, :, None]
    d_k = (d_s.transpose(-1, -2) @ q.float().view(o.shape)).sum(2)
    return {"o": o.view(q.shape).bfloat16(), "lse": lse.view(q.shape[:3]), "d_q": d_q.view(q.shape).bfloat16(),
            "d_k": d_k.bfloat16(), "d_v": d_v.bfloat16()}


def _at(table, rows, page):
    """Page and row within it of rows [batch, n] of the sequences."""
    rows = rows.clamp(min=0)
    return table.gather(1, rows // page).long(), rows % page


def _plain_append(s):
    page, (b, n, h, d) = s["case"]["page"], s["x_k"].shape
    rows = s["lens"].long()[:, None] + torch.arange(n, device="cuda")[None]
    at, off = _at(s["table"], rows, page)
    y = s["x_k"].float()
    if s["w"] is not None:
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * s["w"]
    y1, y2 = y[..., : d // 2], y[..., d // 2:]
    c, z = s["cos"][rows][:, :, None], s["sin"][rows][:, :, None]
    y = torch.cat([y1 * c - y2 * z, y1 * z + y2 * c], -1)
    s["k_pages"][at, :, off] = y.bfloat16()
    s["v_pages"][at, :, off] = s["x_v"]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_decode(s):
    c, q, table = s["case"], s["q"], s["table"]
    b, hq, d = q.shape
    hkv = s["k_pages"].shape[1]
    n = s["lens"].long()[:, None]
    begin = (n - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(n)
    first = begin.clamp(max=c["n_sink"])
    i = torch.arange(max(_visible(c, x) for x in _lengths(c)), device="cuda")[None]
    live = i < first + n - begin
    key = torch.where(i < first, i, i - first + begin).minimum(n - 1)
    at, off = _at(table, key, c["page"])
    k = s["k_pages"][at, :, off].transpose(1, 2).float()  # [batch, KV heads, keys, head_dim]
    x = (q.float().view(b, hkv, -1, d) @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del k
    x = x.masked_fill_(~live[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp_()
    l = e.sum(-1, keepdim=True)
    e = e / l
    o = e @ s["v_pages"][at, :, off].transpose(1, 2).float()
    out = {"o": o.view(b, hq, d).bfloat16(), "lse": (m + l.log()).view(b, hq)}
    if s["weights"] is not None:
        s["weights"].scatter_add_(2, key[:, None].expand(b, hkv, -1), e.sum(2))
        out["weights"] = s["weights"]
    return out


def _plain_evict(s):
    c, w, n = s["case"], s["weights"], s["lens"].long()[:, None, None]
    b, hkv, most = w.shape
    i = torch.arange(most, device="cuda")[None, None]
    # the keys by rank: those that always stay, then by weight (the lower position first among equals), then what is not there
    always = (i < c["n_sink"]) | ((i >= n - c["n_recent"]) & (i < n))
    rank = torch.sort(torch.where(i < n, torch.where(always, math.inf, w), -math.inf), dim=2, descending=True, stable=True).indices
    keep = min(c["n_keep"], most)
    slot = torch.arange(keep, device="cuda")[None, None]
    # (a sequence within its budget keeps its keys where they are)
    kept = torch.where(n <= c["n_keep"], slot, rank[:, :, :keep].sort(dim=2).values)
    left = n.clamp(max=c["n_keep"])
    src = torch.where(slot < left, kept, 0)
    dst = torch.where(slot < left, slot, 0)
    head = torch.arange(hkv, device="cuda")[None, :, None]
    pages = [_at(s["table"], x.reshape(b, -1), c["page"]) for x in (src, dst.expand(b, hkv, keep))]
    (sp, so), (dp, do) = [[t.view(b, hkv, keep) for t in x] for x in pages]
    s["k_pages"][dp, head, do] = s["k_pages"][sp, head, so]
    s["v_pages"][dp, head, do] = s["v_pages"][sp, head, so]
    moved = torch.where(i < n, 0.0, w)
    moved[:, :, :keep] = torch.where(slot < left, w.gather(2, src), moved[:, :, :keep])
    w.copy_(moved)
    none = torch.full((b, hkv, c["n_keep"] - keep), -1, dtype=torch.int32, device="cuda")
    return {"kv_lens": left[:, 0, 0].int(), "kept": torch.cat([torch.where(slot < left, kept, -1).int(), none], 2),
            "k_pages": s["k_pages"], "v_pages": s["v_pages"], "weights": w}


# --------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    path = c["path"]
    if not own:
        return {"sinks": _plain_sinks, "train": _plain_train, "append": _plain_append, "decode": _plain_decode,
                "evict": _plain_evict}[path](s)
    from tyr_b200 import nn
    if path == "sinks":
        o, lse = nn.attentionFwd(s["q"], s["k"], s["v"], window_size=c["window"], n_sink=c["n_sink"])
        return {"o": o, "lse": lse}
    if path == "train":
        at = {"window_size": c["window"], "n_sink": c["n_sink"]}
        o, lse = nn.attentionFwd(s["q"], s["k"], s["v"], **at)
        d_q, d_k, d_v = nn.attentionBwd(s["q"], s["k"], s["v"], o, lse, s["d_o"], **at)
        return {"o": o, "lse": lse, "d_q": d_q, "d_k": d_k, "d_v": d_v}
    if path == "append":
        at = {"positions": s["lens"], "page_table": s["table"]}
        nn.qkPrologue(s["x_k"], s["k_pages"], s["w"], s["cos"], s["sin"], eps=EPS, **at)
        nn.qkPrologue(s["x_v"], s["v_pages"], **at)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if path == "decode":
        o, lse = nn.flashDecodePaged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], max_kv_seq=c["max_len"],
                                     window_size=c["window"], n_sink=c["n_sink"], weights=s["weights"], total_kv_len=s["total"])
        return {"o": o, "lse": lse} if s["weights"] is None else {"o": o, "lse": lse, "weights": s["weights"]}
    lens, kept = nn.evictPaged(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["weights"], c["n_keep"], c["n_recent"],
                               c["n_sink"])
    return {"kv_lens": lens, "kept": kept, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "weights": s["weights"]}


# ------------------------------------------------------------------------------------ what it comes to
def work(case):
    hq, hkv, d, _ = SHAPES[case["shape"]]
    path, b = case["path"], case["batch"]
    row = 2 * d  # bytes of one bf16 row
    if path in ("sinks", "train"):
        n = case["seq"]
        pairs = b * sum(min(i + 1, case["window"] + min(case["n_sink"], max(0, i + 1 - case["window"]))) for i in range(n))
        q, kv, stat = b * hq * n * row, b * hkv * n * row, 4 * b * hq * n
        flops = 4 * d * hq * pairs
        if path == "sinks":
            return {"bytes": 2 * q + 2 * kv + stat, "flops": flops}
        # forward: Q, K, V in, O and statistics out; backward: those and dO in, the gradients out
        return {"bytes": 2 * q + 2 * kv + stat + (3 * q + 2 * kv + stat) + (q + 2 * kv), "flops": flops * 7 // 2}
    if path == "append":
        tokens = b * case["seq"]
        return {"bytes": 4 * tokens * hkv * row + 4 * d * min(tokens, max(_lengths(case)) + case["seq"]), "flops": 10 * tokens * hkv * d}
    if path == "decode":
        keys = sum(_visible(case, n) for n in _lengths(case))
        sums = 8 * keys * hkv if case["weights"] else 0  # read and written
        return {"bytes": 2 * keys * hkv * row + 2 * b * hq * row + 4 * b * hq + sums, "flops": 4 * keys * hq * d}
    over = [n for n in _lengths(case) if n > case["n_keep"]]
    # the weights in, the kept ones and the cleared rest out; the rows that move in and out, the first ones stay
    moved = len(over) * hkv * (case["n_keep"] - case["n_sink"])
    return {"bytes": 8 * sum(over) * hkv + 4 * moved * row + 4 * b * hkv * case["n_keep"], "flops": 2 * sum(over) * hkv + 1}


# ------------------------------------------------------------------------------------ from the definition
def exact(case, seed):
    """Outputs of the first pass on prepare(case, seed) in 64 bits, sequence by sequence; None where nothing is computed."""
    s = prepare(case, seed)
    path, page = case["path"], case["page"] if "page" in case else 0
    if path == "evict":
        return None
    if path == "append":
        kp = s["k_pages"].double()
        for b, n in enumerate(s["lens"].tolist()):
            y = s["x_k"][b].double()
            if s["w"] is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * s["w"].double()
            h = y.shape[-1] // 2
            pos = torch.arange(n, n + y.shape[0], device="cuda")
            cs, sn = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
            y = torch.cat([y[..., :h] * cs - y[..., h:] * sn, y[..., h:] * cs + y[..., :h] * sn], -1)
            kp[s["table"][b, pos // page].long(), :, pos % page] = y
        return {"k_pages": kp, "v_pages": None}
    q = s["q"].double()
    scale = q.shape[-1] ** -0.5
    if path == "decode":
        o, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
        w = s["weights"].double() if s["weights"] is not None else None
        group = q.shape[1] // s["k_pages"].shape[1]
        for b, n in enumerate(s["lens"].tolist()):
            j = torch.arange(n, device="cuda")
            if case["window"]:
                j = j[(j >= n - case["window"]) | (j < case["n_sink"])]
            at = s["table"][b, j // page].long()
            k, v = s["k_pages"][at, :, j % page].double(), s["v_pages"][at, :, j % page].double()
            x = torch.einsum("hgd,jhd->hgj", q[b].view(-1, group, q.shape[-1]), k) * scale
            lse[b] = torch.logsumexp(x, -1).view(-1)
            x = torch.softmax(x, -1)
            o[b] = torch.einsum("hgj,jhd->hgd", x, v).reshape(o[b].shape)
            if w is not None:
                w[b][:, j] += x.sum(1)
        return {"o": o, "lse": lse} if w is None else {"o": o, "lse": lse, "weights": w}
    b, hq, n, d = q.shape
    k, v = s["k"].double(), s["v"].double()
    group = hq // k.shape[1]
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = (j <= i) & ((i - j < case["window"]) | (j < case["n_sink"]))
    o, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda")
    d_q, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for x in range(b * hq):
        a, h = divmod(x, hq)
        kv = h // group
        sc = torch.where(seen, scale * q[a, h] @ k[a, kv].T, -math.inf)
        lse[a, h] = torch.logsumexp(sc, -1)
        p = torch.exp(sc - lse[a, h][:, None])
        o[a, h] = p @ v[a, kv]
        if path == "train":
            g = s["d_o"][a, h].double()
            d_v[a, kv] += p.T @ g
            g = p * (g @ v[a, kv].T - (g * o[a, h]).sum(-1, keepdim=True))
            d_q[a, h] = scale * g @ k[a, kv]
            d_k[a, kv] += scale * g.T @ q[a, h]
    return {"o": o, "lse": lse} if path == "sinks" else {"o": o, "lse": lse, "d_q": d_q, "d_k": d_k, "d_v": d_v}
