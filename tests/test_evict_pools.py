"""An eviction whose K and V pools share memory is refused before any launch (no GPU): different thread blocks move the two in place.
An apart pair goes on to the next check, the sums' alignment, which every call here fails."""
import ctypes
import itertools
import random

import pytest

from tyr_b200 import _lib

SHAPE, ALIGN = -2, -4
BASE = 1 << 30
D = 64


@pytest.fixture(scope="module")
def evict(built_lib):
    def call(k, v, k_stride, v_stride, counts):
        pages, heads, rows = counts
        a = _lib.EvictArgs(k=BASE + 2 * k, v=BASE + 2 * v, pages=_lib.PageTable(table=64, table_stride=4, max_pages=4, n_pages=pages, page_size=rows),
                           kv_lens=64, weights=66, new_lens=128, kept=64, batch=1, n_kv_head=heads, max_kv_seq=rows, head_dim=D, n_keep=1)
        a.k_stride[:], a.v_stride[:], a.weights_stride[:] = k_stride, v_stride, [1 << 20, 1 << 10]
        rc = built_lib.tyr_b200_attn_paged_evict(ctypes.byref(a), None)
        assert rc in (SHAPE, ALIGN)
        return rc
    return call


def packed(counts, order, row=D):
    """Strides {page, head, row} of a pool whose axes lie in `order`, outermost first."""
    stride, step = [0, 0, 0], row
    for x in reversed(order):
        stride[x] = step
        step *= counts[x]
    return stride, step


@pytest.mark.parametrize("order", list(itertools.permutations(range(3))))
def test_usual_layouts(evict, order):
    counts = (4, 3, 16)
    st, size = packed(counts, order)
    assert evict(0, 0, st, st, counts) == SHAPE                    # V is K
    assert evict(0, size, st, st, counts) == ALIGN                 # one behind the other
    assert evict(size, 0, st, st, counts) == ALIGN
    assert evict(0, size - 8, st, st, counts) == SHAPE             # by the last eight elements
    assert evict(size - 8, 0, st, st, counts) == SHAPE
    wide, _ = packed(counts, order, row=2 * D)
    assert evict(0, D, wide, wide, counts) == ALIGN                # a row of K, a row of V
    assert evict(0, D - 8, wide, wide, counts) == SHAPE
    # K and V interleaved over each of the axes: [.., 2, ..]
    for at in range(1, 3):
        four, step, v_at = [0, 0, 0], D, 0
        for n, x in reversed(list(enumerate(order))):
            four[x] = step
            step *= counts[x]
            if n == at:
                v_at, step = step, 2 * step
        assert evict(0, v_at, four, four, counts) == ALIGN
        assert evict(v_at, 0, four, four, counts) == ALIGN
        assert evict(0, v_at - 8, four, four, counts) == SHAPE
        assert evict(0, four[order[0]], four, four, counts) == SHAPE   # K of the next block


def test_blocks_of_a_page_laid_out_differently(evict):
    """[page][K as heads x rows, V as rows x heads]: the blocks do not meet."""
    counts = (4, 3, 16)
    block = 3 * 16 * D
    k, v = [2 * block, 16 * D, D], [2 * block, D, 3 * D]
    assert evict(0, block, k, v, counts) == ALIGN and evict(block, 0, v, k, counts) == ALIGN
    assert evict(0, block - 8, k, v, counts) == SHAPE and evict(0, 0, k, v, counts) == SHAPE


def rows_of(at, stride, counts):
    return {at + sum(i * s for i, s in zip(x, stride)) for x in itertools.product(*(range(n) for n in counts))}


def test_random_pools_against_all_their_rows(evict):
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        counts = [rng.choice([1, 2, 3, 5]) for _ in range(3)]

        def strides():
            order, st, step = rng.sample(range(3), 3), [0, 0, 0], D + 8 * rng.choice([0, 0, 1, 8, 9, 16])
            for x in order:
                st[x] = step
                step = step * counts[x] + 8 * rng.choice([0, 0, 0, 8, 16, 50, 200])
            return st, step
        st, size = strides()
        same = rng.random() < 0.8
        st2 = st if same else strides()[0]
        k, v = 0, 8 * rng.randint(-size // 8 - 2, size // 8 + 2)
        a, b = rows_of(k, st, counts), rows_of(v, st2, counts)
        meet = any(x + d in b for x in a for d in range(-D + 8, D, 8))
        rc = evict(k, v, st, st2, counts)
        assert not (meet and rc == ALIGN), (counts, st, st2, v)
        if same:
            assert (rc == SHAPE) == meet, (counts, st, v)
            seen[meet] += 1
    assert min(seen.values()) > 500


def test_far_apart_and_large(evict):
    counts = (1 << 20, 8, 64)
    st, size = packed(counts, (0, 1, 2))
    assert evict(0, size, st, st, counts) == ALIGN and evict(0, size - 64, st, st, counts) == SHAPE
    st = [1 << 39, 1 << 37, 64]
    assert evict(0, 1 << 30, st, st, (1 << 20, 4, 64)) == ALIGN
    assert evict(0, (1 << 37) * 3, st, st, (1 << 20, 4, 64)) == SHAPE
