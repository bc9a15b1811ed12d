"""Block choice and block-sparse decode on the GPU: picked indices equal those
of the plain restatement (tests/_int4.py), and the attention over them equals
softmax attention in 64 bits over the picked tokens."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402
from tests.test_gpu_int4 import gen  # noqa: E402

INT8, INT4 = kb.KV_INT8, kb.KV_INT4


def topic_rows(g, shape, dtype):
    """Rows that drift along the text, so that blocks differ."""
    lead, t, D = shape[:-2], shape[-2], shape[-1]
    topics = torch.randn(*lead, t // 50 + 1, D, device="cuda", generator=g).repeat_interleave(50, -2)[..., :t, :]
    return (torch.randn(*shape, device="cuda", generator=g) + 0.7 * topics).to(dtype)


def values(fmt, x, G):
    return ref.value4(*ref.quantize4(x, G)) if fmt == INT4 else ref.value8(*ref.quantize8(x, G))


def make(fmt, layers, hkv, hq, D, G, lens, dtype, g, blocks=0, chunk=0):
    pool = kb.KVPool(layers, hkv, hq, D, num_blocks=blocks or sum(n // 256 + 2 for n in lens), group_size=G,
                     kv_format=fmt, block_summaries=True)
    seqs, kv = [], []
    for n in lens:
        s = pool.create_sequence()
        k, v = (topic_rows(g, (layers, 1, hkv, n, D), dtype) for _ in range(2))
        step = chunk or n
        for t in range(0, n, step):
            kb.append_quantize(pool, [s], 0, k[:, :, :, t:t + step].contiguous(), v[:, :, :, t:t + step].contiguous())
        seqs.append(s)
        kv.append((values(fmt, k[:, 0], G), values(fmt, v[:, 0], G)))
    return pool, seqs, kv


def check_pick(got, q, kv, lens, T, budget, first, last):
    L, S, H, B = got.shape
    for layer in range(L):
        for i in range(S):
            want = ref.pick(q[layer, i], kv[i][0][layer], lens[i], T, budget, first, last)
            for h in range(H):
                w = want[h] + [-1] * (B - len(want[h]))
                assert got[layer, i, h].tolist() == w, (layer, i, h)


def check_sparse(out, picked, q, kv, lens, T, scale, pool):
    for layer in range(out.shape[0]):
        for i, n in enumerate(lens):
            k, v = kv[i][0][layer], kv[i][1][layer]
            H = k.shape[0]
            seen = torch.zeros(1, H, n, dtype=torch.bool, device="cuda")
            for h in range(H):
                for b in picked[layer, i, h].tolist():
                    if b >= 0:
                        seen[0, h, b * T:(b + 1) * T] = True
            want = ref.attend(q[layer, i][None], k, v, scale, seen)[0]
            # int8 rounds the weights against values, not against half a range
            tol = ref.tolerance(v if pool.kv_format == INT4 else 2 * v, out.dtype, want)
            err = (out[layer, i].double() - want).abs()
            assert (err <= tol).all(), f"{err.max().item():.3e}"
    assert pool.device_error() == 0


@pytest.mark.parametrize("fmt,D,G,hq,hkv,dtype,lens,budget,first,last", [
    (INT4, 128, 64, 32, 8, torch.bfloat16, [1, 64, 65, 1000, 4097, 2048], 8, 1, 2),
    (INT4, 64, 64, 32, 8, torch.float16, [5000, 129], 5, 0, 1),
    (INT4, 256, 256, 8, 4, torch.bfloat16, [3000], 12, 1, 1),
    (INT4, 256, 64, 7, 1, torch.float16, [4000, 777], 9, 2, 3),
    (INT4, 128, 128, 16, 16, torch.float16, [1500, 63], 3, 1, 1),
    (INT8, 128, 64, 32, 4, torch.bfloat16, [3000, 64, 700], 8, 1, 2),
    (INT8, 64, 64, 4, 2, torch.float16, [2500], 6, 0, 4),
    (INT8, 256, 64, 8, 4, torch.bfloat16, [1000, 31, 2049], 7, 1, 1),
    (INT8, 256, 256, 8, 8, torch.float16, [1300], 10, 2, 2),
    (INT8, 128, 128, 8, 2, torch.bfloat16, [64 * 20], 4, 1, 1),
])
def test_select_and_sparse(fmt, D, G, hq, hkv, dtype, lens, budget, first, last):
    layers = 2
    g = gen(D + hq + budget)
    pool, seqs, kv = make(fmt, layers, hkv, hq, D, G, lens, dtype, g)
    T = pool.select_tokens
    assert T == (32 if fmt == INT8 and D == 256 else 64)
    q = (1.5 * torch.randn(layers, len(lens), hq, D, device="cuda", generator=g)).to(dtype)
    got = kb.select_blocks(pool, seqs, 0, q, budget, first, last)
    check_pick(got, q, kv, lens, T, budget, first, last)
    out = torch.empty(layers, len(lens), hq, D, dtype=torch.float32, device="cuda")
    scale = 1 / math.sqrt(D)
    out2, picked = kb.sparse_decode_attention(pool, seqs, 0, q, out, scale, budget, first, last, return_blocks=True)
    assert torch.equal(picked, got) and "picked" in pool.last_kernels()
    check_sparse(out, picked, q, kv, lens, T, scale, pool)
    again = torch.empty_like(out)  # without a buffer for the indices, layer by layer
    for layer in range(layers):
        kb.sparse_decode_attention(pool, seqs, layer, q[layer:layer + 1].contiguous(), again[layer:layer + 1], scale,
                                   budget, first, last)
    check_sparse(again, picked, q, kv, lens, T, scale, pool)
    pool.close()


def test_budget_covers_everything():
    """With a budget of every block the result is decode_attention's."""
    g = gen(30)
    pool, seqs, kv = make(INT4, 1, 8, 32, 128, 64, [777, 3, 1024], torch.bfloat16, g)
    q = torch.randn(1, 3, 32, 128, device="cuda", generator=g).to(torch.bfloat16)
    a, b = (torch.empty(1, 3, 32, 128, device="cuda") for _ in range(2))
    kb.decode_attention(pool, seqs, 0, q, a, 0.09)
    _, picked = kb.sparse_decode_attention(pool, seqs, 0, q, b, 0.09, 100, return_blocks=True)
    assert picked[0, 0, 0].tolist() == list(range(13)) + [-1] * 87
    check_sparse(b, picked, q, kv, [777, 3, 1024], 64, 0.09, pool)
    assert (a - b).abs().max() <= 4e-3
    pool.close()


def test_ties_go_to_the_lowest_index():
    """Equal blocks score alike; so do all blocks for a query of zeros."""
    g = gen(31)
    D, n = 64, 40
    pool = kb.KVPool(1, 2, 4, D, num_blocks=16, kv_format=INT4, block_summaries=True)
    seq = pool.create_sequence()
    one = torch.randn(1, 1, 2, 64, D, device="cuda", generator=g).half()
    kb.append_quantize(pool, [seq], 0, one.repeat(1, 1, 1, n, 1), one.repeat(1, 1, 1, n, 1))
    q = torch.randn(1, 1, 4, D, device="cuda", generator=g).half()
    for x in (q, torch.zeros_like(q), torch.full_like(q, math.nan), torch.full_like(q, math.inf)):
        got = kb.select_blocks(pool, [seq], 0, x, 7, 0, 2)
        assert got[0, 0].tolist() == [[0, 1, 2, 3, 4, 38, 39]] * 2
    pool.close()


@pytest.mark.parametrize("fmt", [INT4, INT8])
def test_summaries_follow_every_way_of_writing(fmt):
    """Single tokens, decode steps, prompts cut anywhere, truncation and
    rewriting, copy-on-write forks and restored snapshots leave the summaries
    of the full blocks equal to those of the cached values."""
    D, G, hkv, hq, layers, dtype = 128, 64, 2, 8, 2, torch.bfloat16
    g = gen(32)
    pool = kb.KVPool(layers, hkv, hq, D, num_blocks=64, group_size=G, kv_format=fmt, block_summaries=True)
    seq = pool.create_sequence()
    hist = [[], []]

    def add(n, step=False, s=None, h=None):
        s, h = s or seq, h or hist
        k, v = (topic_rows(g, (layers, 1, hkv, n, D), dtype) for _ in range(2))
        if step:
            q = torch.randn(layers, 1, hq, D, device="cuda", generator=g).to(dtype)
            kb.decode_step(pool, [s], 0, k, v, q, torch.empty_like(q), 0.1)
        else:
            kb.append_quantize(pool, [s], 0, k, v)
        h[0].append(values(fmt, k[:, 0], G))
        h[1].append(values(fmt, v[:, 0], G))

    def verify(s, h):
        kk = torch.cat(h[0], 2)
        n = kk.shape[2]
        assert s.length(0) == n
        q = torch.randn(layers, 1, hq, D, device="cuda", generator=g).to(dtype)
        got = kb.select_blocks(pool, [s], 0, q, 4, 0, 1)
        check_pick(got, q, [(kk, None)], [n], 64, 4, 0, 1)

    add(500)
    for _ in range(12):
        add(1)
    add(70)
    verify(seq, hist)
    for _ in range(70):
        add(1, step=True)
    verify(seq, hist)
    seq.truncate(300)
    hist = [[torch.cat(x, 2)[:, :, :300]] for x in hist]
    for n in (3, 15, 40, 1, 200):
        add(n)
    verify(seq, hist)
    n = seq.length(0)
    pc = kb.PrefixCache(pool)
    pc.store_quantized(list(range(n)), "m", seq)
    hit = pc.lookup_quantized(list(range(n)), "m")
    fork = hit.fork(400)
    forked = [[torch.cat(x, 2)[:, :, :400]] for x in hist]
    add(333, s=fork, h=forked)
    verify(fork, forked)
    verify(seq, hist)
    new = pool.create_sequence()
    for layer in range(layers):
        new.restore_quantized(layer, fork.quantized_snapshot(layer))
    verify(new, forked)
    pool.close()


def test_long_sequence_clusters_and_other_stream():
    """Many blocks of few (sequence, head) pairs (several CTAs share a choice),
    on a stream of its own, with the pool's scratch in use on two streams."""
    g = gen(33)
    lens = [70001, 40000]
    pool, seqs, kv = make(INT4, 1, 2, 16, 64, 64, lens, torch.float16, g, chunk=20000)
    q = torch.randn(1, 2, 16, 64, device="cuda", generator=g).half()
    outs = [torch.empty(1, 2, 16, 64, device="cuda") for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in outs]
    torch.cuda.synchronize()
    for o, s in zip(outs, streams):
        kb.sparse_decode_attention(pool, seqs, 0, q, o, 0.125, 40, 1, 2, stream=s)
    torch.cuda.synchronize()
    picked = kb.select_blocks(pool, seqs, 0, q, 40, 1, 2)
    check_pick(picked, q, kv, lens, 64, 40, 1, 2)
    for o in outs:
        check_sparse(o, picked, q, kv, lens, 64, 0.125, pool)
    pool.close()


def test_very_long_sequence_uses_scratch_keys():
    """More blocks than a CTA's shared memory holds keys for."""
    D, n = 64, 64 * 49152 + 1000
    g = gen(34)
    pool = kb.KVPool(1, 1, 1, D, num_blocks=n // 256 + 1, kv_format=INT4, block_summaries=True)
    seq = pool.create_sequence()
    kept = []
    for t in range(0, n, 400000):
        m = min(400000, n - t)
        k = topic_rows(g, (1, 1, 1, m, D), torch.float16)
        kb.append_quantize(pool, [seq], 0, k, k)
        kept.append(ref.value4(*ref.quantize4(k[0, 0], 64)).float())
    k = torch.cat(kept, 1)
    q = torch.randn(1, 1, 1, D, device="cuda", generator=g).half()
    got = kb.select_blocks(pool, [seq], 0, q, 25, 1, 1)
    check_pick(got, q, [(k[None], None)], [n], 64, 25, 1, 1)
    out = torch.empty(1, 1, 1, D, device="cuda")
    _, picked = kb.sparse_decode_attention(pool, [seq], 0, q, out, 0.125, 25, 1, 1, return_blocks=True)
    assert torch.equal(picked, got)
    at = torch.cat([torch.arange(b * 64, min(n, b * 64 + 64), device="cuda") for b in got[0, 0, 0].tolist()])
    kk = k[:, at].double()
    want = ref.attend(q[0], kk, kk, 0.125)[0]
    assert ((out[0, 0].double() - want).abs() <= ref.tolerance(kk, out.dtype, want)).all()
    pool.close()
