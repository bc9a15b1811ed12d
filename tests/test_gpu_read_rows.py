"""Reading rows back from windowed pools whose layers have different lengths."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402
from tests.test_gpu_int4 import gen, rows  # noqa: E402


def test_read_rows_of_unequal_layers():
    """Windowed layers of different lengths, no starts given: the rows begin at
    the first one that every layer of the call retains."""
    D, G, hkv, W = 64, 64, 2, 100
    g = gen(53)
    for fmt in (kb.KV_INT4, kb.KV_INT8):
        pool = kb.KVPool(2, hkv, 4, D, num_blocks=8, group_size=G, window=W, max_append=64, kv_format=fmt)
        seq = pool.create_sequence()
        hist = [[], []]
        for layer, n in [(0, 64), (1, 64), (0, 64), (1, 64), (0, 50), (1, 50), (0, 33)]:
            k = rows(g, (1, 1, hkv, n, D), torch.float16)
            kb.append_quantize(pool, [seq], layer, k, k)
            hist[layer].append(k[0, 0])
        full = [torch.cat(h, 1) for h in hist]
        first = [seq.length(layer) - seq.retained(layer) for layer in range(2)]
        assert first[0] != first[1]
        start, n = max(first), min(seq.length(0), seq.length(1)) - max(first)
        got, _ = kb.read_rows(pool, [seq], 0, 2, n)
        for layer in range(2):
            x = full[layer][:, start:start + n]
            want = ref.value4(*ref.quantize4(x, G)) if fmt == kb.KV_INT4 else ref.value8(*ref.quantize8(x, G))
            assert torch.equal(got[layer, 0], want.half())
        with pytest.raises(kb.KrillError):
            kb.read_rows(pool, [seq], 0, 2, n + 1)
        pool.close()
