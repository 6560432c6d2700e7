"""First tokens beside a sliding window, without a GPU: the plain form against differences, the refusals, and the number of
units that the backward cuts the first tokens' key blocks into."""
import ctypes
import os
import subprocess

import pytest
import torch

import plain_sinks as plain
from tyr_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_visibility_closed_forms():
    m = plain.seen(6, 2, 1)
    assert [r.nonzero().view(-1).tolist() for r in m] == [[0], [0, 1], [0, 1, 2], [0, 2, 3], [0, 3, 4], [0, 4, 5]]
    causal = torch.tril(torch.ones(6, 6, dtype=torch.bool))
    assert torch.equal(plain.seen(6, 6, 0), causal) and torch.equal(plain.seen(6, 1, 6), causal)
    assert torch.equal(plain.seen(6, 3, 3), causal) and not torch.equal(plain.seen(6, 2, 3), causal)


@pytest.mark.parametrize("n,window,n_sink", [(9, 3, 2), (7, 1, 1), (8, 20, 3)])
def test_plain_gradients_against_differences(n, window, n_sink):
    g = torch.Generator().manual_seed(n)
    x = [torch.randn(2, h, n, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2)]
    d_o = torch.randn(2, 4, n, 8, generator=g, dtype=torch.float64)
    grads = plain.backward(*x, d_o, window, n_sink, 0.4)
    for i in range(3):
        u = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        loss = [float((plain.forward(*[t + s * h * u if a == i else t for a, t in enumerate(x)], window, n_sink, 0.4)[0] * d_o).sum())
                for s in (1, -1)]
        assert abs((loss[0] - loss[1]) / (2 * h) - float((grads[i][0] * u).sum())) < 1e-7


def prefill_args(p, **kw):
    a = _lib.PrefillArgs(q=p, k=p, v=p, o=p, batch=1, n_head=4, n_kv_head=2, q_seq=8, kv_seq=8, head_dim=64, window_size=4)
    for name in ("q_stride", "k_stride", "v_stride", "o_stride"):
        getattr(a, name)[:] = [4 * 8 * 64, 8 * 64, 64]
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_refusals(built_lib):
    buf = ctypes.create_string_buffer(8192)
    p = ctypes.addressof(buf)
    p += (-p) % 16
    f = built_lib.tyr_b200_attn_prefill_sinks
    assert f(None, 1, None) == -1
    assert f(ctypes.byref(prefill_args(p)), -1, None) == -2
    assert f(ctypes.byref(prefill_args(p, window_size=0)), 2, None) == -2           # first tokens go with a window
    assert f(ctypes.byref(prefill_args(p, window_size=-3)), 2, None) == -2
    assert f(ctypes.byref(prefill_args(p, key_mask=p, key_mask_stride=8)), 2, None) == -2
    assert f(ctypes.byref(prefill_args(p, kv_seq=4)), 2, None) == -2                 # one sequence length
    assert f(ctypes.byref(prefill_args(p, head_dim=96)), 2, None) == -3
    assert f(ctypes.byref(prefill_args(p, q=p + 2)), 2, None) == -4
    assert f(ctypes.byref(prefill_args(p, batch=0)), 2, None) == 0                   # nothing to do
    g, need = built_lib.tyr_b200_attn_backward_sinks, built_lib.tyr_b200_attn_backward_sinks_workspace_bytes
    a = _lib.BackwardArgs(q=p, k=p, v=p, o=p, d_o=p, lse=p, d_q=p, d_k=p, d_v=p, batch=1, n_head=4, n_kv_head=2, q_seq=8, kv_seq=8,
                          head_dim=64, window_size=4)
    for name in ("q_stride", "k_stride", "v_stride", "o_stride", "do_stride", "dq_stride", "dk_stride", "dv_stride"):
        getattr(a, name)[:] = [4 * 8 * 64, 8 * 64, 64]
    assert g(None, 1, None) == -1 and need(None, 1) == -1
    assert g(ctypes.byref(a), -1, None) == -2 and need(ctypes.byref(a), -1) == -2
    plain_need = built_lib.tyr_b200_attn_backward_workspace_bytes(1, 4, 8)
    assert need(ctypes.byref(a), 0) == plain_need and plain_need < need(ctypes.byref(a), 2) <= plain_need + 512   # one key block: a counter only
    assert g(ctypes.byref(a), 2, None) == -7
    a.workspace, a.workspace_bytes = p, need(ctypes.byref(a), 2) - 1
    assert g(ctypes.byref(a), 2, None) == -7
    a.window_size = 0
    assert g(ctypes.byref(a), 2, None) == -2 and need(ctypes.byref(a), 2) == -2
    a.window_size, a.q_seq, a.kv_seq = 128, 8192, 8192
    base = built_lib.tyr_b200_attn_backward_workspace_bytes(1, 4, 8192)
    extra = need(ctypes.byref(a), 2) - base - 256
    assert extra > 0 and extra % (2 * 2 * 128 * 64 * 4) == 0                         # whole parts of both KV heads
    a.batch = 3
    assert need(ctypes.byref(a), 2) == 3 * (base + extra) + 256                      # as many parts whatever the batch
    a.batch = 0
    assert need(ctypes.byref(a), 2) == 0
    a.batch, a.head_dim = 1, 96
    assert need(ctypes.byref(a), 2) == -3


SWEEP = r"""
#include <cstdio>
#include "unit_parts.h"
using namespace tyr;
int main() {
  long long bad = 0, cut = 0;
  for (int blocks : {1, 2, 3, 7, 16, 64, 71, 500, 4096})
    for (int sink : {1, 2, 3, 40})
      for (int kv : {1, 2, 8, 64})
        for (int group : {1, 4, 16})
          for (int window : {1, 2, 100, 128, 1024, 100000, 524288})
            for (int sms : {148, 20, 1}) {
              if (sink > blocks) continue;
              const int parts = choose_sink_parts(blocks, blocks, kv, group, window, sink, sms);
              // at least one pair of every first block for each part: the last of them is seen by blocks - sink + 1 query blocks
              if (parts < 1 || parts > kMaxSinkParts || parts > (blocks - sink + 1) * group) ++bad;
              if (parts > 1) ++cut;
              // a window over everything makes all units alike in the causal order: nothing to cut but for a small launch
              const BwdSizes z{blocks, blocks, kv, kv * group, group, window, true, sink};
              const int cap[4] = {sms, sms / 2, sms / 4, sms / 8};
              const int p = choose_unit_parts(z, sms, cap);
              if (p != 1 && p != 2 && p != 4 && p != 8) ++bad;
            }
  std::printf("%lld %lld\n", bad, cut);
}
"""


def test_parts_of_the_first_tokens(tmp_path):
    src, exe = tmp_path / "sweep.cpp", tmp_path / "sweep"
    src.write_text(SWEEP)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "tyr_b200", "csrc"), str(src), "-o", str(exe)])
    bad, cut = map(int, subprocess.check_output([str(exe)]).split())
    assert bad == 0 and cut > 0
