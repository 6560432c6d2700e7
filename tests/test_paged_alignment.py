"""Misaligned arrays of 32-bit numbers are refused by the paged-cache calls before any launch (no GPU): a kernel's load from one
would fault."""
import ctypes

import pytest

from tyr_b200 import _lib

P, ALIGN = 1 << 20, -4


def table(at=P):
    return _lib.PageTable(table=at, table_stride=4, max_pages=4, n_pages=8, page_size=16)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_decode(built_lib, off):
    def call(**kw):
        a = _lib.PagedDecodeArgs(q=P, o=P, k=P, v=P, pages=table(), kv_lens=P, batch=1, n_head=2, n_kv_head=1, max_kv_seq=64, head_dim=64,
                                 weights=P)      # without a workspace: a call that passes all checks of its arrays ends there
        a.k_stride[:] = a.v_stride[:] = [16 * 64, 16 * 64, 64]
        a.q_stride[:] = a.o_stride[:] = [2 * 64, 64]
        a.weights_stride[:] = [64, 64]
        for k, v in kw.items():
            setattr(a, k, v)
        return built_lib.tyr_b200_attn_paged_decode(ctypes.byref(a), None)

    assert call() == -7
    for bad in (dict(pages=table(P + off)), dict(kv_lens=P + off), dict(lse=P + off), dict(weights=P + off)):
        assert call(**bad) == ALIGN, bad


@pytest.mark.parametrize("off", [1, 2, 3])
def test_evict(built_lib, off):
    def call(**kw):
        a = _lib.EvictArgs(k=P, v=P + 8 * 16 * 64 * 2, pages=table(), kv_lens=P, weights=P, new_lens=P + 64, kept=P, batch=1, n_kv_head=1,
                           max_kv_seq=64, head_dim=64, n_keep=8, n_recent=2, n_sink=1)
        a.k_stride[:] = a.v_stride[:] = [16 * 64, 16 * 64, 64]
        a.weights_stride[:] = [64, 64]
        for k, v in kw.items():
            setattr(a, k, v)
        return built_lib.tyr_b200_attn_paged_evict(ctypes.byref(a), None)

    for bad in (dict(pages=table(P + off)), dict(kv_lens=P + off), dict(new_lens=P + 64 + off), dict(kept=P + off), dict(weights=P + off)):
        assert call(**bad) == ALIGN, bad


@pytest.mark.parametrize("off", [1, 2, 3])
def test_append(built_lib, off):
    def call(pages, rows=None, positions=None):
        a = _lib.PrologueArgs(x=P, out=P, batch=2, seq=3, n_head=2, head_dim=64, positions=positions)
        a.x_stride[:] = [3 * 2 * 64, 2 * 64, 64]
        a.out_stride[:] = [2 * 16 * 64, 16 * 64, 64]
        return built_lib.tyr_b200_attn_qk_prologue_paged(ctypes.byref(a), ctypes.byref(pages), rows, None)

    assert call(table(P + off)) == ALIGN
    assert call(table(), rows=P + off) == ALIGN
    assert call(table(), positions=P + off) == ALIGN
