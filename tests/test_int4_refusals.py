"""Argument checks of 4-bit pools, block summaries, block choice and row
reading, and the planner on host-only pools. CPU only."""
import ctypes as C

import pytest

import krill_b200 as kb
from krill_b200 import _lib as L


def pool(**kw):
    args = dict(num_layers=2, num_kv_heads=8, num_q_heads=32, head_dim=128, num_blocks=64, device=-1,
                kv_format=kb.KV_INT4, block_summaries=True)
    args.update(kw)
    return kb.KVPool(**args)


def seq_of(p, n):
    s = p.create_sequence()
    arr = (C.c_uint64 * 1)(s.handle)
    if n:
        L.check(L.lib.krill_append_quantize(p.handle, 1, arr, 0, p.num_layers, n, None, None, L.DTYPE_BF16, None))
    return s, arr


@pytest.mark.parametrize("kw,msg", [
    (dict(attn_impl=kb.ATTN_CUDA_CORE), "TENSOR_CORE"),
    (dict(attn_impl=kb.ATTN_TENSOR_CORE_PAIR), "TENSOR_CORE"),
    (dict(attn_impl=kb.ATTN_TENSOR_CORE_SYNC), "TENSOR_CORE"),
    (dict(quant_variant=kb.QUANT_INPUT_DTYPE), "QUANT_F32"),
    (dict(kv_format=3), "kv_format"),
    (dict(window=512), "full-history"),
    (dict(kv_format=kb.KV_BF16), "block_summaries"),
    (dict(kv_format=kb.KV_INT8, attn_impl=kb.ATTN_CUDA_CORE), "tensor-core"),
    (dict(group_size=32), "group_size"),
])
def test_pool_refusals(kw, msg):
    with pytest.raises(kb.KrillError) as e:
        pool(**kw)
    assert e.value.status == L.KRILL_ERR_INVALID and msg in str(e.value)


def test_geometry():
    for D, G in ((64, 64), (128, 64), (128, 128), (256, 64), (256, 256)):
        row = D + 8 * D // G  # bytes of one token of one head
        p = pool(head_dim=D, group_size=G, block_summaries=False)
        assert p.block_bytes == 2 * 8 * 256 * row and p.select_tokens == 64
        p = pool(head_dim=D, group_size=G)
        assert p.block_bytes == 2 * 8 * (256 * row + 4 * (2 * D + 4))
        assert p.block_bytes % 16 == 0
    p = pool(kv_format=kb.KV_INT8, head_dim=256)
    assert p.select_tokens == 32
    assert p.block_bytes == 2 * 8 * (256 * (512 + 32) + 8 * (512 + 4))


def select(p, arr, n=1, budget=8, first=1, last=1, lb=0, lc=2, dtype=L.DTYPE_BF16, q=None, sel=None):
    return L.lib.krill_select_blocks(p.handle, n, arr, lb, lc, q, dtype, budget, first, last, sel, None)


def sparse(p, arr, n=1, budget=8, first=1, last=1, scale=0.1, out_dtype=L.DTYPE_BF16, sel=None, q=None):
    return L.lib.krill_sparse_decode_attention(p.handle, n, arr, 0, 2, q, L.DTYPE_BF16, None, out_dtype, scale,
                                               budget, first, last, sel, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(budget=1), "max_blocks"),
    (dict(budget=0, first=0), "max_blocks"),
    (dict(first=-1), "first_blocks"),
    (dict(last=0), "last_blocks"),
    (dict(first=2**31 - 1, last=2**31 - 1, budget=2**31 - 1), "max_blocks"),
    (dict(n=-1), "n_seqs"),
])
def test_choice_refusals(kw, msg):
    p = pool()
    _, arr = seq_of(p, 1000)
    for call in (select, sparse):
        assert call(p, arr, **kw) == L.KRILL_ERR_INVALID and msg in L.last_error()
    assert select(p, arr) == L.KRILL_OK and sparse(p, arr) == L.KRILL_OK


def test_more_choice_refusals():
    p = pool()
    _, arr = seq_of(p, 1000)
    assert select(p, arr, dtype=L.DTYPE_F32) == L.KRILL_ERR_INVALID and "dtype" in L.last_error()
    assert select(p, arr, lb=1) == L.KRILL_ERR_INVALID and "layer range" in L.last_error()
    assert select(p, arr, sel=C.c_void_p(6)) == L.KRILL_ERR_INVALID and "4-byte" in L.last_error()
    assert sparse(p, arr, sel=C.c_void_p(6)) == L.KRILL_ERR_INVALID and "4-byte" in L.last_error()
    assert select(p, arr, q=C.c_void_p(8)) == L.KRILL_ERR_INVALID and "16-byte" in L.last_error()
    assert sparse(p, arr, q=C.c_void_p(8)) == L.KRILL_ERR_INVALID and "16-byte" in L.last_error()
    for scale in (0.0, -1.0, float("nan")):
        assert sparse(p, arr, scale=scale) == L.KRILL_ERR_INVALID and "scale" in L.last_error()
    _, empty = seq_of(p, 0)
    assert select(p, empty) == L.KRILL_ERR_INVALID and "empty" in L.last_error()
    assert sparse(p, empty) == L.KRILL_ERR_INVALID and "empty" in L.last_error()
    stale = (C.c_uint64 * 1)(77 << 32)
    assert select(p, stale) == L.KRILL_ERR_INVALID
    plain = pool(block_summaries=False)
    _, arr = seq_of(plain, 1000)
    for call in (select, sparse):
        assert call(plain, arr) == L.KRILL_ERR_INVALID and "block_summaries" in L.last_error()
    assert select(p, None, n=0) == L.KRILL_OK


def test_read_rows_refusals():
    p = pool()
    _, arr = seq_of(p, 300)

    def read(starts, n, dtype=L.DTYPE_F16, keys=None, lb=0, lc=2, pl=p, a=arr):
        st = None if starts is None else (C.c_int64 * 1)(starts)
        return L.lib.krill_read_rows(pl.handle, 1, a, lb, lc, st, n, keys, None, dtype, None)

    assert read(0, 300) == L.KRILL_ERR_NO_DEVICE and read(None, 300) == L.KRILL_ERR_NO_DEVICE
    for starts, n in ((1, 300), (0, 301), (-1, 1), (300, 1), (0, 2**62), (2**62, 1)):
        assert read(starts, n) == L.KRILL_ERR_INVALID and "not cached" in L.last_error()
    assert read(0, 0) == L.KRILL_OK
    assert read(0, -1) == L.KRILL_ERR_INVALID
    assert read(0, 1, dtype=L.DTYPE_U8) == L.KRILL_ERR_INVALID and "dtype" in L.last_error()
    assert read(0, 1, keys=C.c_void_p(4)) == L.KRILL_ERR_INVALID and "16-byte" in L.last_error()
    assert read(0, 1, lb=1) == L.KRILL_ERR_INVALID
    raw = pool(kv_format=kb.KV_BF16, block_summaries=False)
    _, a = seq_of(raw, 10)
    assert read(0, 1, pl=raw, a=a) == L.KRILL_ERR_INVALID
    win = pool(window=64, block_summaries=False)
    _, a = seq_of(win, 256)
    _, a2 = seq_of(win, 256)
    L.check(L.lib.krill_append_quantize(win.handle, 1, a2, 0, 2, 200, None, None, L.DTYPE_BF16, None))
    assert read(0, 1, pl=win, a=a2) == L.KRILL_ERR_INVALID and "not cached" in L.last_error()


def test_append_alignment():
    p = pool()
    s, arr = seq_of(p, 0)
    st = L.lib.krill_append_quantize(p.handle, 1, arr, 0, 1, 1, C.c_void_p(24), C.c_void_p(32), L.DTYPE_F16, None)
    assert st == L.KRILL_ERR_INVALID and "16-byte" in L.last_error() and s.length(0) == 0
    raw = kb.KVPool(2, 8, 32, 128, num_blocks=8, kv_format=kb.KV_BF16, device=-1)
    _, arr = seq_of(raw, 0)
    st = L.lib.krill_append_quantize_rope(raw.handle, 1, arr, 0, 1, 1, None, None, L.DTYPE_BF16,
                                          C.cast(C.c_void_p(64), C.c_void_p), C.c_void_p(64), 10, None)
    assert st == L.KRILL_ERR_INVALID and "RoPE" in L.last_error()


def test_disk_tier_refused():
    pc = kb.PrefixCache(pool())
    with pytest.raises(kb.KrillError):
        pc.set_disk("/tmp/never", 1)


def test_planned_kernels():
    p = pool()
    s, arr = seq_of(p, 5000)
    assert sparse(p, arr, budget=16) == L.KRILL_OK
    assert "attn_tc_kernel<128,2," in p.last_kernels() and "picked" in p.last_kernels()
    c, hg, items, ctas = p.last_plan()
    assert items >= 1 and ctas >= 1
    L.check(L.lib.krill_decode_attention(p.handle, 1, arr, 0, 2, None, 1, None, 1, 0.1, None))
    assert ",2>" in p.last_kernels().split("+")[0].split("[")[0] and "picked" not in p.last_kernels()
    L.check(L.lib.krill_prefill_attention(p.handle, 1, arr, 0, 2, 300, None, 1, None, 1, 0.1, None))
    assert "attn_shared_umma_kernel" in p.last_kernels()
