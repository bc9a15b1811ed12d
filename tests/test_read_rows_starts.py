"""Where krill_read_rows begins: checked and read rows are the same ones. CPU
only (host-only pools: a call that passes the checks reports no device)."""
import ctypes as C

import pytest

import krill_b200 as kb
from krill_b200 import _lib as L


def make(fmt, lens, window=100):
    """A sequence whose layers were appended one at a time, to `lens` tokens."""
    p = kb.KVPool(len(lens), 2, 4, 64, num_blocks=16, window=window, max_append=64, device=-1, kv_format=fmt)
    s = p.create_sequence()
    arr = (C.c_uint64 * 1)(s.handle)
    for layer, n in enumerate(lens):
        while s.length(layer) < n:
            step = min(64, n - s.length(layer))
            L.check(L.lib.krill_append_quantize(p.handle, 1, arr, layer, 1, step, None, None, L.DTYPE_BF16, None))
    return p, s, arr


@pytest.mark.parametrize("fmt", [kb.KV_INT4, kb.KV_INT8])
@pytest.mark.parametrize("lens", [[211, 178], [178, 211], [400, 256, 301], [128, 127]])
def test_default_start_is_retained_by_every_layer(fmt, lens):
    p, s, arr = make(fmt, lens)
    firsts = [s.length(i) - s.retained(i) for i in range(len(lens))]

    def read(starts, n):
        st = None if starts is None else (C.c_int64 * 1)(starts)
        return L.lib.krill_read_rows(p.handle, 1, arr, 0, len(lens), st, n, None, None, L.DTYPE_F16, None)

    most = max(0, min(lens) - max(firsts))  # (0: no row is in every layer)
    for n in {1, most} if most else ():
        assert read(None, n) == L.KRILL_ERR_NO_DEVICE
    assert read(None, most + 1) == L.KRILL_ERR_INVALID and "not cached" in L.last_error()
    # as the call with that start
    assert read(max(firsts), most) == (L.KRILL_ERR_NO_DEVICE if most else L.KRILL_OK)
    assert read(max(firsts), most + 1) == L.KRILL_ERR_INVALID


def test_no_common_row():
    """Layers so far apart that no row is in both."""
    p, s, arr = make(kb.KV_INT4, [64, 600])
    assert L.lib.krill_read_rows(p.handle, 1, arr, 0, 2, None, 1, None, None, L.DTYPE_F16, None) == L.KRILL_ERR_INVALID
    assert "not cached" in L.last_error()


@pytest.mark.parametrize("starts", [[5], [], [1, 2, 3]])
def test_one_start_for_each_sequence(starts):
    """Too few starts are refused, not filled up with zeros."""
    p, s, _ = make(kb.KV_INT4, [128, 128])
    with pytest.raises(ValueError, match="starts"):
        kb.read_rows(p, [s, s], 0, 2, 1, starts=starts)
