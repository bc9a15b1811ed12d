"""Block choice over clusters of every size, and picked blocks of consecutive
calls and of several streams."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402
from tests.test_gpu_int4 import gen  # noqa: E402
from tests.test_gpu_sparse import INT4, INT8, check_pick, check_sparse, make  # noqa: E402


def check_step(out, q, kv, lens, scale, budget, first, last, pool):
    """A sparse step's output against attention over the blocks that the plain
    restatement picks for its query."""
    L, S, H = out.shape[0], out.shape[1], pool.num_kv_heads
    want = torch.full((L, S, H, budget), -1, dtype=torch.int32)
    for layer in range(L):
        for i in range(S):
            for h, blocks in enumerate(ref.pick(q[layer, i], kv[i][0][layer], lens[i], 64, budget, first, last)):
                want[layer, i, h, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
    check_sparse(out, want, q, kv, lens, 64, scale, pool)


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


@pytest.mark.parametrize("fmt", [INT4, INT8])
def test_consecutive_choices_into_one_buffer(fmt):
    """Sparse steps back to back whose choices differ and go to the same
    scratch: each attends its own blocks, none the step's before it."""
    g = gen(41)
    lens, D, H = [4000, 3300, 4031], 64, 4
    pool, seqs, kv = make(fmt, 2, H, H, D, 64, lens, torch.float16, g)
    n = 24
    qs = [(3 * torch.randn(2, 3, H, D, device="cuda", generator=g)).half() for _ in range(n)]
    outs = [torch.empty(2, 3, H, D, device="cuda") for _ in range(n)]
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        kb.sparse_decode_attention(pool, seqs, 0, q, o, 0.125, 6, 1, 1)
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        check_step(o, q, kv, lens, 0.125, 6, 1, 1, pool)
    pool.close()


def test_streams_with_work_of_their_own():
    """Sparse steps of different queries, budgets and sequences and split dense
    decodes, interleaved over four streams: the pool's scratch (picked blocks,
    partial records) is one buffer, laid out anew by each call."""
    g = gen(42)
    lens, D, H, hq = [20001, 9000, 12345], 64, 2, 8
    pool, seqs, kv = make(INT4, 1, H, hq, D, 64, lens, torch.float16, g)
    groups = [[0, 1, 2], [2, 0], [1], [0]]
    budgets = [40, 7, 90, 21]
    streams = [torch.cuda.Stream() for _ in groups]
    steps = []  # (stream, sequences, budget or None, q, out)
    for _ in range(6):
        for s, who, budget in zip(streams, groups, budgets):
            for b in (budget, None):
                q = (2 * torch.randn(1, len(who), hq, D, device="cuda", generator=g)).half()
                steps.append((s, who, b, q, torch.empty(1, len(who), hq, D, device="cuda")))
    # the scratch has its final size before the streams start: growing it waits for the device
    for s, who, b, q, o in steps[:8]:
        if b:
            kb.sparse_decode_attention(pool, [seqs[i] for i in who], 0, q, o, 0.125, b, 1, 2)
        else:
            kb.decode_attention(pool, [seqs[i] for i in who], 0, q, o, 0.125)
    for step in steps:
        step[4].fill_(math.nan)
    torch.cuda.synchronize()
    for s, who, b, q, o in steps:
        if b:
            kb.sparse_decode_attention(pool, [seqs[i] for i in who], 0, q, o, 0.125, b, 1, 2, stream=s)
        else:
            kb.decode_attention(pool, [seqs[i] for i in who], 0, q, o, 0.125, stream=s)
    torch.cuda.synchronize()
    for s, who, b, q, o in steps:
        mine, n = [kv[i] for i in who], [lens[i] for i in who]
        if b:
            check_step(o, q, mine, n, 0.125, b, 1, 2, pool)
            continue
        for j in range(len(who)):
            want = ref.attend(q[0, j][None], mine[j][0][0], mine[j][1][0], 0.125)[0]
            err = (o[0, j].double() - want).abs()
            assert (err <= ref.tolerance(mine[j][1][0], o.dtype, want)).all(), f"{err.max().item():.3e}"
    pool.close()


@pytest.mark.parametrize("blocks", [8193, 12289, 49152])
def test_many_keys_in_shared_memory(blocks):
    """Sequences whose keys take more than 32 KB, more than 48 KB and all of the
    shared memory that a choice may use."""
    n = 64 * blocks - 5
    g = gen(blocks)
    pool, seqs, kv = make(INT4, 1, 1, 2, 64, 64, [n], torch.float16, g, chunk=400000)
    q = torch.randn(1, 1, 2, 64, device="cuda", generator=g).half()
    picked = kb.select_blocks(pool, seqs, 0, q, 33, 1, 2)
    check_pick(picked, q, kv, [n], 64, 33, 1, 2)
    assert pool.device_error() == 0
    pool.close()
