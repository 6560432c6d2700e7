"""Attention with a sliding window and first tokens that stay visible, from its definition in float64, with how far a kernel
may be off: bf16 inputs and outputs, P and dS rounded to bf16 for the matrix products, everything else in 32 bits."""
import math

import torch

HALF = 2.0 ** -8       # half a step of bf16, relative
SLACK = 1.01           # products of small terms, 32-bit sums


def seen(n, window, n_sink):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    return (j <= i) & ((i - j < window) | (j < n_sink))


def repeat(x, group):
    return x.repeat_interleave(group, 1)


def forward(q, k, v, window, n_sink, scale=None):
    """o, lse, P and what bounds the errors of o and lse."""
    q, k, v = q.double(), k.double(), v.double()
    n, d, group = q.shape[2], q.shape[3], q.shape[1] // k.shape[1]
    scale = scale or d ** -0.5
    kh, vh = repeat(k, group), repeat(v, group)
    m = seen(n, window, n_sink)
    s = (q @ kh.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    # a score is a sum of d products in 32 bits: off by at most (d + 2) roundings of the sum of their magnitudes
    ds = ((d + 2) * 2.0 ** -24 * scale * (q.abs() @ kh.abs().transpose(-1, -2)) * m).amax(-1)
    rel_p = 2 * ds + 2.0 ** -18 * (1 + lse.abs())              # of a weight: scores, LSE, the exponential
    tol_o = (p @ vh.abs()) * (2 * HALF + rel_p[..., None]) * SLACK   # P to bf16, O to bf16
    tol_lse = ds + 2.0 ** -20 * (1 + lse.abs())
    return p @ vh, lse, p, rel_p, tol_o, tol_lse


def backward(q, k, v, d_o, window, n_sink, scale=None):
    """[(gradient, how far it may be off)] of q, k, v."""
    o, lse, p, rel_p, tol_o, _ = forward(q, k, v, window, n_sink, scale)
    q, k, v, d_o = q.double(), k.double(), v.double(), d_o.double()
    b, hq, n, d = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    scale = scale or d ** -0.5
    kh, vh = repeat(k, group), repeat(v, group)

    def of_group(x):
        return x.view(b, hkv, group, n, d).sum(2)

    d_v = of_group(p.transpose(-1, -2) @ d_o)
    tol_v = of_group((p * (HALF + rel_p[..., None])).transpose(-1, -2) @ d_o.abs()) * SLACK + HALF * d_v.abs()
    d_p = d_o @ vh.transpose(-1, -2)
    d_s = scale * p * (d_p - (d_o * o).sum(-1, keepdim=True))
    # delta is formed from the rounded O; dP is a sum of d products in 32 bits
    e_delta = (d_o.abs() * tol_o).sum(-1, keepdim=True)
    e_dp = (d + 2) * 2.0 ** -24 * (d_o.abs() @ vh.abs().transpose(-1, -2))
    e_s = d_s.abs() * (HALF + rel_p[..., None]) + scale * p * (e_delta + e_dp)
    d_q, d_k = d_s @ kh, of_group(d_s.transpose(-1, -2) @ q)
    tol_q = (e_s @ kh.abs()) * SLACK + HALF * d_q.abs()
    tol_k = of_group(e_s.transpose(-1, -2) @ q.abs()) * SLACK + HALF * d_k.abs()
    return [(d_q, tol_q), (d_k, tol_k), (d_v, tol_v)]


def check(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), (what, float((err / tol.clamp(min=1e-300)).max()))
