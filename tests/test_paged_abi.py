"""What the paged-cache calls refuse before any launch (no GPU)."""
import ctypes

import pytest

from tyr_b200 import _lib


@pytest.fixture
def mem():
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    return buf, p + (-p) % 16


def table(p, **kw):
    t = dict(table=p, table_stride=4, max_pages=4, n_pages=8, page_size=16)
    t.update(kw)
    return _lib.PageTable(**t)


def test_struct_sizes_match_the_c_layout():
    assert ctypes.sizeof(_lib.PageTable) == 2 * 8 + 3 * 4 + 4
    assert ctypes.sizeof(_lib.PagedDecodeArgs) == 5 * 8 + 32 + 2 * 8 + 2 * 8 + 7 * 4 + 4 + 10 * 8 + 2 * 4 + 3 * 8
    assert ctypes.sizeof(_lib.EvictArgs) == 2 * 8 + 32 + 2 * 8 + 2 * 8 + 2 * 8 + 7 * 4 + 4 + 6 * 8


def test_decode(built_lib, mem):
    _, p = mem
    f = built_lib.tyr_b200_attn_paged_decode
    assert f(None, None) == -1

    def call(**kw):
        a = _lib.PagedDecodeArgs(q=p, o=p, k=p, v=p, pages=table(p), kv_lens=p, batch=2, n_head=4, n_kv_head=2, max_kv_seq=64, head_dim=64)
        for s in ("k_stride", "v_stride"):
            getattr(a, s)[:] = [2 * 16 * 64, 16 * 64, 64]
        a.q_stride[:] = a.o_stride[:] = [4 * 64, 64]
        for k, v in kw.items():
            if isinstance(v, list):
                getattr(a, k)[:] = v
            else:
                setattr(a, k, v)
        return f(ctypes.byref(a), None)

    for name in ("q", "o", "k", "v", "kv_lens"):
        assert call(**{name: None}) == -1, name
    assert call(pages=table(None)) == -1
    assert call(batch=0) == 0                                        # no sequence: nothing to do
    for bad in (dict(batch=-1), dict(n_head=0), dict(n_kv_head=0), dict(n_head=5), dict(max_kv_seq=0), dict(window_size=-1),
                dict(n_sink=-1), dict(n_sink=4), dict(pages=table(p, max_pages=0)), dict(pages=table(p, n_pages=0)),
                dict(pages=table(p, page_size=0)), dict(pages=table(p, table_stride=-1))):
        assert call(**bad) == -2, bad
    assert call(head_dim=96) == -3 and call(head_dim=256) == -3
    assert call(max_kv_seq=65) == -11                                # more than four pages of 16 rows
    assert call(pages=table(p, page_size=1 << 30)) == -10            # rows past 32 bits
    assert call(pages=table(p, max_pages=2, page_size=(1 << 30) - 1), max_kv_seq=(1 << 30) + 1) == -10
    assert call(batch=65536) == -10 and call(n_kv_head=65537, n_head=65537) == -10
    for bad in (dict(k=p + 8), dict(v=p + 2), dict(k_stride=[2048, 1024, 60]), dict(v_stride=[2047, 1024, 64]), dict(k_stride=[2048, 1024, 0]),
                dict(q=p + 2), dict(q_stride=[255, 64]), dict(o=p + 1), dict(weights=p + 2, weights_stride=[128, 64])):
        assert call(**bad) == -4, bad
    assert call(weights=p, weights_stride=[128, 32]) == -2           # rows of two heads overlap
    assert call(weights=p, weights_stride=[32, 64]) == -2
    assert call(weights=p, weights_stride=[64, 64]) == -2            # the second head of one sequence is the first of the next
    assert call(weights=p, weights_stride=[64, 127]) == -2 and call(weights=p, weights_stride=[64, 128]) == -7   # heads outermost: fine
    assert call(weights=p, weights_stride=[128, 64]) == -7           # the scores' workspace is missing
    assert call(weights=p, weights_stride=[128, 64], workspace=p + 8, workspace_bytes=1 << 20) == -7
    assert call(weights=p, weights_stride=[128, 64], workspace=p, workspace_bytes=2 * 4 * 65 * 4 - 1) == -7


def test_decode_workspace(built_lib, mem):
    f = built_lib.tyr_b200_attn_paged_decode_workspace_bytes
    a = _lib.PagedDecodeArgs(batch=2, n_head=4, n_kv_head=2, max_kv_seq=64, head_dim=64)
    assert f(ctypes.byref(a)) == 0
    a.weights = mem[1]
    assert f(ctypes.byref(a)) == 2 * 4 * (64 + 1) * 4                # every score and each row's LSE
    a.max_kv_seq = 100000
    part = built_lib.tyr_b200_attn_decode_workspace_bytes(2, 4, 64, 100000, 64)
    assert f(ctypes.byref(a)) == (part + 255) // 256 * 256 + 2 * 4 * 100001 * 4
    a.window_size, a.n_sink = 50, 6                                  # what is out of sight needs no room
    assert f(ctypes.byref(a)) == 2 * 4 * (56 + 1) * 4
    a.window_size = a.n_sink = 2 ** 31 - 1
    assert f(ctypes.byref(a)) == (part + 255) // 256 * 256 + 2 * 4 * 100001 * 4
    a.head_dim = 80
    assert f(ctypes.byref(a)) == -3 and f(None) == -1


def test_evict(built_lib, mem):
    _, p = mem
    f = built_lib.tyr_b200_attn_paged_evict
    assert f(None, None) == -1

    def call(**kw):
        a = _lib.EvictArgs(k=p, v=p, pages=table(p), kv_lens=p, weights=p, new_lens=p + 64, kept=p, batch=2, n_kv_head=2, max_kv_seq=64,
                           head_dim=64, n_keep=8, n_recent=2, n_sink=1)
        for s in ("k_stride", "v_stride"):
            getattr(a, s)[:] = [2 * 16 * 64, 16 * 64, 64]
        a.weights_stride[:] = [128, 64]
        for k, v in kw.items():
            if isinstance(v, list):
                getattr(a, k)[:] = v
            else:
                setattr(a, k, v)
        return f(ctypes.byref(a), None)

    for name in ("k", "v", "kv_lens", "weights", "new_lens", "kept"):
        assert call(**{name: None}) == -1, name
    assert call(batch=0) == 0
    for bad in (dict(batch=-1), dict(n_kv_head=0), dict(max_kv_seq=0), dict(n_keep=0), dict(n_recent=-1), dict(n_sink=-1),
                dict(n_recent=8), dict(n_recent=2 ** 31 - 1, n_sink=2 ** 31 - 1), dict(new_lens=p), dict(weights_stride=[128, 63]),
                dict(weights_stride=[0, 64]), dict(weights_stride=[64, 64]), dict(pages=table(p, table_stride=0)),
                dict(k_stride=[0, 1024, 64]), dict(v_stride=[2048, 0, 64]), dict(k_stride=[2048, 1024, 56])):
        assert call(**bad) == -2, bad
    assert call(head_dim=96) == -3
    assert call(max_kv_seq=65, weights_stride=[256, 128]) == -11
    assert call(k=p + 8) == -4 and call(v_stride=[2048, 1024, 4]) == -4
    assert call(n_kv_head=70000) == -10
    # (the list of the kept keys is walked in steps of up to 2048 in 32 bits)
    assert call(n_keep=(1 << 30) + 1) == -10 and call(n_keep=2 ** 31 - 1) == -10
    assert call(new_lens=p + 4) == -2 and call(kv_lens=p + 4, new_lens=p) == -2         # overlapping lengths
    # two heads of a page of 16 rows, and two pages, on one another
    assert call(k_stride=[2048, 64, 64]) == -2 and call(v_stride=[2048, 512, 64]) == -2 and call(k_stride=[1024, 1024, 64]) == -2
    assert call(v_stride=[1 << 62, 1024, 64]) == -2
    assert call(pages=table(p, max_pages=2, page_size=(1 << 30) - 1), max_kv_seq=(1 << 30) + 1) == -10


def test_append(built_lib, mem):
    _, p = mem
    f = built_lib.tyr_b200_attn_qk_prologue_paged

    def call(pages=None, **kw):
        a = _lib.PrologueArgs(x=p, out=p, batch=2, seq=3, n_head=2, head_dim=64)
        a.x_stride[:] = [3 * 2 * 64, 2 * 64, 64]
        a.out_stride[:] = [2 * 16 * 64, 16 * 64, 64]
        for k, v in kw.items():
            if isinstance(v, list):
                getattr(a, k)[:] = v
            else:
                setattr(a, k, v)
        return f(ctypes.byref(a), ctypes.byref(pages if pages is not None else table(p)), None, None)

    assert f(None, ctypes.byref(table(p)), None, None) == -1 and call(pages=table(None)) == -1 and call(x=None) == -1
    assert call(out_at_row0=1) == -2 and call(pages=table(p, page_size=0)) == -2
    assert call(position0=62) == -11                                 # rows 62..64 of 64
    assert call(pages=table(p, page_size=1 << 29)) == -10
    assert call(out=p + 8) == -4 and call(head_dim=96) == -3
    assert call(out_stride=[2048, 0, 64]) == -2 and call(out_stride=[0, 1024, 64]) == -2      # heads or pages on one another
    assert call(out_stride=[2048, 64, 64]) == -2 and call(out_stride=[1024, 1024, 64]) == -2
    assert call(cos=p, sin=p) == -2                                  # a rotary table without rows
    assert call(cos=p, sin=p, max_pos=2) == -11


def test_python_calls_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from tyr_b200 import nn
    q, pool = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        nn.flashDecodePaged(q, pool, pool, t, n)
    with pytest.raises(ValueError):
        nn.evictPaged(pool, pool, t, n, torch.zeros(1, 2, 64), 4, 1)
    with pytest.raises(ValueError):
        nn.qkPrologue(torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), pool, page_table=t)
