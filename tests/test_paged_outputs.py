"""A paged decode whose output rows share memory is refused before any launch (no GPU).  Every call here fails the next check, the
sums' alignment."""
import ctypes

import pytest

from tyr_b200 import _lib

SHAPE, ALIGN = -2, -4


@pytest.mark.parametrize("batch,heads,stride,rc", [
    (2, 4, [4 * 64, 64], ALIGN), (2, 4, [64, 2 * 64], ALIGN),              # either axis outermost
    (2, 4, [12 * 64, 64], ALIGN), (1, 1, [0, 0], ALIGN), (1, 4, [0, 64], ALIGN), (3, 1, [64, 0], ALIGN),
    (2, 4, [0, 64], SHAPE), (2, 4, [4 * 64, 0], SHAPE), (2, 4, [4 * 64, 63], SHAPE), (2, 4, [4 * 64 - 1, 64], SHAPE), (2, 4, [64, 64], SHAPE),
    (2, 4, [-4 * 64, 64], SHAPE), (2, 4, [1 << 62, 64], SHAPE)])
def test_rows(built_lib, batch, heads, stride, rc):
    p = 1 << 20
    a = _lib.PagedDecodeArgs(q=p, o=p, k=p, v=p, pages=_lib.PageTable(table=p, table_stride=4, max_pages=4, n_pages=8, page_size=16), kv_lens=p,
                             batch=batch, n_head=heads, n_kv_head=1, max_kv_seq=64, head_dim=64, weights=p + 2)
    a.k_stride[:] = a.v_stride[:] = [16 * 64, 16 * 64, 64]
    a.q_stride[:], a.o_stride[:], a.weights_stride[:] = [heads * 64, 64], stride, [64, 64]
    assert built_lib.tyr_b200_attn_paged_decode(ctypes.byref(a), None) == rc
