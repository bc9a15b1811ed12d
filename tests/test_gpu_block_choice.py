"""Block choice over clusters of every size."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests.test_gpu_int4 import gen  # noqa: E402
from tests.test_gpu_sparse import INT4, check_pick, make  # noqa: E402


@pytest.mark.parametrize("layers,hkv,lens", [
    (1, 1, [8192]),                    # 128 blocks, one pair: two CTAs a choice
    (1, 2, [16500, 100]),              # four; a sequence that is picked whole
    (1, 1, [32768 + 7]),               # eight
    (2, 2, [66000, 65, 40000]),        # eight, over 256 blocks and shorter beside
    (2, 16, [9000, 17000, 3000, 640]), # 128 pairs: two or four
    (4, 16, [8300, 4000, 100]),        # 192 pairs: two
])
def test_choice_over_clusters(layers, hkv, lens):
    """Consecutive choices for different queries, none waited for."""
    g = gen(len(lens) + hkv)
    pool, seqs, kv = make(INT4, layers, hkv, hkv, 64, 64, lens, torch.float16, g, chunk=20000)
    qs = [torch.randn(layers, len(lens), hkv, 64, device="cuda", generator=g).half() for _ in range(4)]
    torch.cuda.synchronize()
    got = [kb.select_blocks(pool, seqs, 0, q, 11, 1, 2) for q in qs]
    for q, picked in zip(qs, got):
        check_pick(picked, q, kv, lens, 64, 11, 1, 2)
    pool.close()
