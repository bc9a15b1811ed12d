"""4-bit pools on the GPU: codes, scales and read-back bit for bit against the
plain restatement (tests/_int4.py), and every attention entry point against
softmax attention in 64 bits over the cached values."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402

SHAPES = [(64, 64), (128, 64), (128, 128), (256, 64), (256, 256)]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, shape, dtype, odd=False, strong=False):
    """K/V rows: normal values, for keys (`strong`) with a few strong channels;
    `odd` adds groups that are constant, empty, tiny, huge, infinite or NaN."""
    x = torch.randn(*shape, device="cuda", generator=g)
    if strong:
        x = x * (1.0 + 7.0 * (torch.rand(shape[-1], device="cuda", generator=g) > 0.95)) + 0.25
    x = x.to(dtype)
    if odd:
        flat = x.view(-1, shape[-1])
        n = flat.shape[0]
        flat[0 % n] = 0
        flat[1 % n] = 3.140625
        flat[2 % n] *= 1e-6 if dtype == torch.float16 else 1e-20
        flat[3 % n] *= 8000
        flat[4 % n, 5] = math.inf
        flat[5 % n, 7] = -math.inf
        flat[6 % n, 9] = math.nan
        flat[7 % n] = math.nan
        flat[8 % n, ::2] = -0.0
    return x


def pool4(layers, hkv, hq, D, G, blocks=64, **kw):
    return kb.KVPool(layers, hkv, hq, D, num_blocks=blocks, group_size=G, kv_format=kb.KV_INT4, **kw)


def fill(pool, lens, dtype, g, layers, chunk=0):
    """Sequences of the given lengths and their cached values [layer][seq] (k, v) in f64."""
    seqs, kv = [], []
    for n in lens:
        s = pool.create_sequence()
        k = rows(g, (layers, 1, pool.num_kv_heads, n, pool.head_dim), dtype, strong=True)
        v = rows(g, (layers, 1, pool.num_kv_heads, n, pool.head_dim), dtype)
        step = chunk or n
        for t in range(0, n, step):
            kb.append_quantize(pool, [s], 0, k[:, :, :, t:t + step].contiguous(), v[:, :, :, t:t + step].contiguous())
        seqs.append(s)
        kv.append((ref.value4(*ref.quantize4(k[:, 0], pool.group_size)),
                   ref.value4(*ref.quantize4(v[:, 0], pool.group_size))))
    return seqs, kv


def check(out, want, v, pool, out_dtype=None):
    tol = ref.tolerance(v, out_dtype or out.dtype, want)
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"max error {err.max().item():.3e}, bound there {tol.flatten()[err.argmax()].item():.3e}"
    assert pool.device_error() == 0


# ---------------------------------------------------------------- append and read back
@pytest.mark.parametrize("D,G", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("start,n", [(0, 1), (5, 3), (63, 2), (0, 16), (60, 15), (7, 130), (64, 64), (255, 257)])
def test_append_bits(D, G, dtype, start, n):
    layers, hkv = 2, 2
    g = gen(1000 * D + 10 * n + start)
    pool = pool4(layers, hkv, 4, D, G, blocks=16)
    seqs = [pool.create_sequence() for _ in range(3)]
    old = [rows(g, (layers, 3, hkv, start, D), dtype) for _ in range(2)] if start else None
    if start:
        kb.append_quantize(pool, seqs, 0, *old)
    k, v = rows(g, (layers, 3, hkv, n, D), dtype, odd=True), rows(g, (layers, 3, hkv, n, D), dtype, odd=True)
    kb.append_quantize(pool, seqs, 0, k, v)
    for x, name in ((k, "k"), (v, "v")):
        whole = torch.cat([old[name == "v"], x], 3) if start else x
        codes, s, z = ref.quantize4(whole, G)
        for layer in range(layers):
            for i, seq in enumerate(seqs):
                snap = seq.quantized_snapshot(layer)
                got = (snap.keys, snap.key_scales, snap.key_zeros) if name == "k" else \
                    (snap.values, snap.value_scales, snap.value_zeros)
                for a, b in zip(got, (codes, s, z)):
                    assert torch.equal(a, b[layer, i])
    for out_dtype in (torch.float16, torch.bfloat16, torch.float32):
        kk, vv = kb.read_rows(pool, seqs, 0, layers, n, starts=[start] * 3, dtype=out_dtype)
        for x, got in ((k, kk), (v, vv)):
            codes, s, z = ref.quantize4(x, G)
            c = codes.float().unflatten(-1, (D // G, G))
            want = (c * s[..., None].float() + z[..., None].float()).flatten(-2).to(out_dtype)
            assert torch.equal(got, want) and torch.isfinite(got).all()
    kk, vv = seqs[1].snapshot(1)
    k16, v16 = kb.read_rows(pool, [seqs[1]], 1, 1, start + n)
    assert torch.equal(kk, k16[0, 0]) and torch.equal(vv, v16[0, 0])
    pool.close()


def test_quantizer_ties_and_division():
    """Codes equal those of the correctly rounded quotient, ties to even: rows
    of small whole numbers and halves, whose quotients tie often, and a wide
    sweep of scales."""
    D, G = 128, 64
    g = gen(3)
    pool = pool4(1, 8, 8, D, G, blocks=64)
    for dtype in (torch.float16, torch.bfloat16):
        seq = pool.create_sequence()
        a = torch.randint(-64, 65, (8, 700, D), device="cuda", generator=g).float() / 2
        b = torch.randn(8, 700, D, device="cuda", generator=g) * torch.exp2(
            torch.randint(-12, 12, (8, 700, 1), device="cuda", generator=g).float())
        x = torch.cat([a, b], 1).to(dtype)[None, None].contiguous()
        kb.append_quantize(pool, [seq], 0, x, x)
        snap = seq.quantized_snapshot(0)
        codes, s, z = ref.quantize4(x[0, 0], G)
        assert torch.equal(snap.keys, codes) and torch.equal(snap.values, codes)
        assert torch.equal(snap.key_scales, s) and torch.equal(snap.value_zeros, z)
        seq.release()
    pool.close()


def test_append_rope():
    hkv, rows_n = 2, 400
    g = gen(4)
    for D, dtype in ((64, torch.float16), (128, torch.bfloat16), (256, torch.float16)):
        p = torch.arange(rows_n, device="cuda").float()[:, None] * torch.pow(
            10000.0, -torch.arange(0, D, 2, device="cuda").float() / D)
        cos, sin = p.cos().contiguous(), p.sin().contiguous()
        pool = pool4(1, hkv, 4, D, 64, blocks=8)
        seq = pool.create_sequence()
        start, seen = 0, []
        for n in (3, 200, 1):
            k, v = rows(g, (1, 1, hkv, n, D), dtype), rows(g, (1, 1, hkv, n, D), dtype)
            kb.append_quantize(pool, [seq], 0, k, v, rope=(cos, sin))
            x = k[0, 0].float()
            lo, hi = x[..., : D // 2], x[..., D // 2:]
            c, s = cos[start:start + n], sin[start:start + n]
            seen.append(torch.cat([lo * c - hi * s, lo * s + hi * c], -1).to(dtype))
            start += n
        codes, s, z = ref.quantize4(torch.cat(seen, 1), 64)
        snap = seq.quantized_snapshot(0)
        assert torch.equal(snap.keys, codes) and torch.equal(snap.key_scales, s) and torch.equal(snap.key_zeros, z)
        pool.close()


def test_windowed_append_wraps_one_subblock():
    """A call whose first and last tokens fall into one sub-block of the ring."""
    D, G, hkv, W, M = 64, 64, 2, 2, 255
    g = gen(5)
    pool = pool4(1, hkv, 4, D, G, blocks=4, window=W, max_append=M)
    seq = pool.create_sequence()
    hist = []
    for n in (100, 255, 255, 40, 255):
        k = rows(g, (1, 1, hkv, n, D), torch.float16)
        v = rows(g, (1, 1, hkv, n, D), torch.float16)
        kb.append_quantize(pool, [seq], 0, k, v)
        hist.append((k, v))
        # the call's own rows are all retained
        total = seq.length(0)
        kk, vv = kb.read_rows(pool, [seq], 0, 1, n, starts=[total - n])
        for x, got in ((k, kk), (v, vv)):
            assert torch.equal(got[0, 0], ref.value4(*ref.quantize4(x[0, 0], G)).half())
    pool.close()


def test_snapshot_restore_stack_scatter():
    D, G, hkv = 128, 64, 2
    g = gen(6)
    pool = pool4(2, hkv, 4, D, G, blocks=32)
    seqs, kv = fill(pool, [70, 300], torch.bfloat16, g, 2)
    new = pool.create_sequence()
    for layer in range(2):
        new.restore_quantized(layer, seqs[1].quantized_snapshot(layer))
    for layer in range(2):
        a, b = seqs[1].quantized_snapshot(layer), new.quantized_snapshot(layer)
        for name in ("keys", "values", "key_scales", "key_zeros", "value_scales", "value_zeros"):
            assert torch.equal(getattr(a, name), getattr(b, name))
    q = torch.randn(2, 2, 4, D, device="cuda", generator=g).to(torch.bfloat16)
    x, y = torch.empty_like(q), torch.empty_like(q)
    kb.decode_attention(pool, [seqs[0], seqs[1]], 0, q, x, 0.1)
    kb.decode_attention(pool, [seqs[0], new], 0, q, y, 0.1)
    assert torch.equal(x, y)
    st = kb.stack_caches_left_padded_quantized(pool, seqs, 0)
    assert st.keys.shape == (2, hkv, 300, D) and int(st.keys[0, :, :230].max()) == 0
    assert torch.equal(st.keys[0, :, 230:], seqs[0].quantized_snapshot(0).keys)
    assert seqs[0].memory_size_bytes(0) == 70 * hkv * (D + 8 * D // G)
    pool.close()


# ---------------------------------------------------------------- decode
@pytest.mark.parametrize("D,G,hq,hkv,dtype,out_dtype", [
    (64, 64, 32, 8, torch.float16, torch.float32),
    (128, 64, 32, 8, torch.bfloat16, torch.float32),
    (128, 64, 32, 4, torch.bfloat16, torch.bfloat16),
    (128, 128, 7, 1, torch.float16, torch.float32),
    (128, 64, 16, 16, torch.float16, torch.float16),
    (256, 64, 8, 4, torch.bfloat16, torch.float32),
    (256, 256, 16, 2, torch.float16, torch.float32),
])
@pytest.mark.parametrize("lens", [[1], [63, 64, 65, 1], [257, 3000, 128], [5000]])
def test_decode(D, G, hq, hkv, dtype, out_dtype, lens):
    layers = 2
    g = gen(D + hq + len(lens))
    pool = pool4(layers, hkv, hq, D, G)
    seqs, kv = fill(pool, lens, dtype, g, layers)
    q = (torch.randn(layers, len(lens), hq, D, device="cuda", generator=g) * 2).to(dtype)
    out = torch.empty(layers, len(lens), hq, D, dtype=out_dtype, device="cuda")
    scale = 1 / math.sqrt(D)
    kb.decode_attention(pool, seqs, 0, q, out, scale)
    for layer in range(layers):
        for i in range(len(lens)):
            want = ref.attend(q[layer, i][None], kv[i][0][layer], kv[i][1][layer], scale)[0]
            check(out[layer, i], want, kv[i][1][layer], pool)
    pool.close()


@pytest.mark.parametrize("kw", [dict(), dict(split_tokens=256), dict(split_tokens=64)])
def test_decode_many_and_noalloc(kw):
    """A batch that splits long sequences over CTAs, the allocation-free entry
    point, and another stream than the one that appended."""
    D, G, hq, hkv, layers = 128, 64, 32, 8, 2
    g = gen(8)
    lens = [9000, 17, 640, 4097, 2500, 333, 64, 6000]
    pool = pool4(layers, hkv, hq, D, G, blocks=128, **kw)
    seqs, kv = fill(pool, lens, torch.bfloat16, g, layers, chunk=1000)
    q = torch.randn(layers, len(lens), hq, D, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.empty(layers, len(lens), hq, D, dtype=torch.float32, device="cuda")
    other = torch.empty_like(out)
    alt = torch.empty_like(out)
    kb.decode_attention(pool, seqs, 0, q, out, 0.09)
    from krill_b200 import _lib as L
    from krill_b200.cache import _ptr, _seq_array, _stream
    L.check(L.lib.krill_decode_attention_noalloc(pool.handle, len(lens), _seq_array(seqs), 0, layers, _ptr(q), 1,
                                                 _ptr(other), 2, 0.09, _stream(None)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kb.decode_attention(pool, seqs, 0, q, alt, 0.09, stream=side)
    torch.cuda.synchronize()
    for layer in range(layers):
        for i in range(len(lens)):
            want = ref.attend(q[layer, i][None], kv[i][0][layer], kv[i][1][layer], 0.09)[0]
            for o in (out, other, alt):
                check(o[layer, i], want, kv[i][1][layer], pool)
    pool.close()


def test_decode_windowed():
    D, G, hq, hkv, W = 64, 64, 8, 4, 300
    g = gen(9)
    pool = pool4(1, hkv, hq, D, G, blocks=16, window=W, max_append=200)
    seq = pool.create_sequence()
    ks, vs = [], []
    for n in (200, 200, 1, 150, 1, 77):
        k, v = rows(g, (1, 1, hkv, n, D), torch.float16), rows(g, (1, 1, hkv, n, D), torch.float16)
        kb.append_quantize(pool, [seq], 0, k, v)
        ks.append(k[0, 0])
        vs.append(v[0, 0])
    total = sum(k.shape[1] for k in ks)
    keep = min(seq.retained(0), W)
    kk = ref.value4(*ref.quantize4(torch.cat(ks, 1), G))[:, total - keep:]
    vv = ref.value4(*ref.quantize4(torch.cat(vs, 1), G))[:, total - keep:]
    q = torch.randn(1, 1, hq, D, device="cuda", generator=g).half()
    out = torch.empty(1, 1, hq, D, device="cuda")
    kb.decode_attention(pool, [seq], 0, q, out, 0.125)
    check(out[0, 0], ref.attend(q[0], kk, vv, 0.125)[0], vv, pool)
    pool.close()


@pytest.mark.parametrize("size", [1e-4, 1.0, 900.0, 30000.0])
def test_decode_value_range(size):
    """Values from tiny (scales near the f16 subnormals) to near the format's
    end (scales of 64 and more change the weights' exponent bias), and queries
    far from one."""
    D, G, hq, hkv = 128, 64, 8, 2
    g = gen(10)
    pool = pool4(1, hkv, hq, D, G, blocks=8)
    seq = pool.create_sequence()
    k = rows(g, (1, 1, hkv, 700, D), torch.bfloat16)
    v = (torch.randn(1, 1, hkv, 700, D, device="cuda", generator=g) * size / 4).clamp(-size, size).to(torch.bfloat16)
    kb.append_quantize(pool, [seq], 0, k, v)
    kk, vv = (ref.value4(*ref.quantize4(x[0, 0], G)) for x in (k, v))
    for qs in (1e-3, 1.0, 300.0):
        q = (torch.randn(1, 1, hq, D, device="cuda", generator=g) * qs).to(torch.bfloat16)
        out = torch.empty(1, 1, hq, D, device="cuda")
        kb.decode_attention(pool, [seq], 0, q, out, 0.1 / qs)
        check(out[0, 0], ref.attend(q[0], kk, vv, 0.1 / qs)[0], vv, pool)
    pool.close()


def test_stale_infinities_do_not_leak():
    """Blocks that held infinite and NaN scales (restored from a snapshot) are
    reused by a shorter sequence: nothing past its end may reach the result,
    on the decode, the multi-query and the prompt path."""
    D, G, hq, hkv = 128, 64, 32, 8
    g = gen(11)
    pool = pool4(1, hkv, hq, D, G, blocks=2)
    bad = pool.create_sequence()
    n = 512
    codes = torch.full((hkv, n, D), 15, dtype=torch.uint8, device="cuda")
    meta = torch.full((hkv, n, D // G), math.inf, dtype=torch.float16, device="cuda")
    nan = torch.full_like(meta, math.nan)
    bad.restore_quantized(0, kb.QuantizedKVSnapshot(codes, codes, meta, nan, nan, meta))
    torch.cuda.synchronize()
    bad.release()
    seqs, kv = fill(pool, [300], torch.bfloat16, g, 1, chunk=10)
    for nq in (1, 3, 5, 40):
        q = torch.randn(1, 1, nq, hq, D, device="cuda", generator=g).to(torch.bfloat16)
        out = torch.empty(1, 1, nq, hq, D, dtype=torch.float32, device="cuda")
        kb.verify_attention(pool, seqs, 0, q, out, 0.09)
        pos = torch.arange(300, device="cuda")
        seen = (pos[None] <= (300 - nq + torch.arange(nq, device="cuda"))[:, None])[:, None]
        vv = kv[0][1][0]
        kk = kv[0][0][0]
        if nq >= 16:  # the prompt path rounds K and V to f16
            kk, vv = kk.half().double(), vv.half().double()
        check(out[0, 0], ref.attend(q[0, 0], kk, vv, 0.09, seen), vv * (2 if nq >= 16 else 1), pool)
    pool.close()


# ---------------------------------------------------------------- several queries
@pytest.mark.parametrize("D,G,hq,hkv,dtype,nq", [
    (128, 64, 32, 8, torch.bfloat16, 4),   # two query tiles
    (128, 128, 32, 8, torch.float16, 3),
    (64, 64, 32, 8, torch.float16, 5),
    (128, 64, 32, 4, torch.bfloat16, 2),
    (256, 64, 8, 4, torch.float16, 3),
    (256, 256, 8, 8, torch.bfloat16, 9),
    (128, 64, 14, 2, torch.bfloat16, 2),   # 7 heads to a kv head
])
def test_verify(D, G, hq, hkv, dtype, nq):
    layers, lens = 2, [nq, 63 + nq, 65, 700, 2049]
    lens = [max(x, nq) for x in lens]
    g = gen(D + nq)
    pool = pool4(layers, hkv, hq, D, G)
    seqs, kv = fill(pool, lens, dtype, g, layers)
    q = torch.randn(layers, len(lens), nq, hq, D, device="cuda", generator=g).to(dtype)
    out = torch.empty(layers, len(lens), nq, hq, D, dtype=torch.float32, device="cuda")
    scale = 1 / math.sqrt(D)
    kb.verify_attention(pool, seqs, 0, q, out, scale)
    for layer in range(layers):
        for i, n in enumerate(lens):
            seen = (torch.arange(n, device="cuda")[None] <= (n - nq + torch.arange(nq, device="cuda"))[:, None])[:, None]
            check(out[layer, i], ref.attend(q[layer, i], kv[i][0][layer], kv[i][1][layer], scale, seen),
                  kv[i][1][layer], pool)
    pool.close()


@pytest.mark.parametrize("D,G,hq,hkv,dtype,nq,lens", [
    (128, 64, 32, 8, torch.bfloat16, 300, [300, 1300, 301]),
    (64, 64, 32, 8, torch.float16, 130, [207, 130]),
    (128, 128, 16, 16, torch.float16, 64, [564, 64]),
    (256, 64, 8, 4, torch.bfloat16, 70, [70, 500]),  # head_dim 256: the decode kernel's units
])
def test_prefill(D, G, hq, hkv, dtype, nq, lens):
    """Prompt chunks. On tcgen05 (head_dim <= 128) K and V enter as f16, so the
    reference uses the values rounded to f16; the softmax weights are rounded
    to f16 as well, which bounds the error by 2^-11 of the largest |v| (not of
    half a range: hence the doubled span)."""
    layers = 1
    g = gen(D + nq)
    pool = pool4(layers, hkv, hq, D, G)
    seqs, kv = fill(pool, lens, dtype, g, layers)
    q = torch.randn(layers, len(lens), nq, hq, D, device="cuda", generator=g).to(dtype)
    out = torch.empty(layers, len(lens), nq, hq, D, dtype=torch.float32, device="cuda")
    scale = 1 / math.sqrt(D)
    kb.prefill_attention(pool, seqs, 0, q, out, scale)
    assert ("umma" in pool.last_kernels()) == (D <= 128)
    for i, n in enumerate(lens):
        seen = (torch.arange(n, device="cuda")[None] <= (n - nq + torch.arange(nq, device="cuda"))[:, None])[:, None]
        kk, vv = kv[i][0][0], kv[i][1][0]
        if D <= 128:
            kk, vv = kk.half().double(), vv.half().double()
        check(out[0, i], ref.attend(q[0, i], kk, vv, scale, seen), 2 * vv, pool)
    pool.close()


def test_prefix_cascade_and_copy_on_write():
    """Forks of one prefix attend its blocks together on tcgen05 (K and V as
    f16 there); the fork that writes into a shared block gets its own copy."""
    D, G, hq, hkv, layers = 128, 64, 32, 8, 2
    g = gen(12)
    pool = pool4(layers, hkv, hq, D, G, blocks=64)
    seqs, kv = fill(pool, [700], torch.bfloat16, g, layers)
    pc = kb.PrefixCache(pool)
    tokens = list(range(700))
    pc.store_quantized(tokens, "m", seqs[0])
    hit = pc.lookup_quantized(tokens, "m")
    forks = [hit.fork(700 - i) for i in range(6)]
    k, v = (rows(g, (layers, 6, hkv, 1, D), torch.bfloat16) for _ in range(2))
    q = torch.randn(layers, 6, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.empty(layers, 6, hq, D, device="cuda")
    kb.decode_step(pool, forks, 0, k, v, q, out, 0.09)
    assert pool.last_cascade()[0] == 1
    for layer in range(layers):
        for i in range(6):
            new = [ref.value4(*ref.quantize4(x[layer, i], G)) for x in (k, v)]
            kk, vv = (torch.cat([kv[0][j][layer][:, :700 - i], new[j]], 1) for j in range(2))
            want = ref.attend(q[layer, i][None], kk.half().double(), vv.half().double(), 0.09)[0]
            check(out[layer, i], want, 2 * vv, pool)
    pool.close()


def test_decode_step_host():
    D, G, hq, hkv, layers = 64, 64, 8, 2, 3
    g = gen(13)
    pool = pool4(layers, hkv, hq, D, G, blocks=16)
    seqs, kv = fill(pool, [63, 200], torch.float16, g, layers)
    k, v = (rows(g, (layers, 2, hkv, 1, D), torch.float16) for _ in range(2))
    q = torch.randn(layers, 2, hq, D, device="cuda", generator=g).half()
    out = torch.empty(layers, 2, hq, D, dtype=torch.float32).pin_memory()
    kb.decode_step_host(pool, seqs, 0, *[x.cpu().pin_memory() for x in (k, v, q)], out, 0.125, layer_chunk=2)
    torch.cuda.synchronize()
    for layer in range(layers):
        for i in range(2):
            new = [ref.value4(*ref.quantize4(x[layer, i], G)) for x in (k, v)]
            kk, vv = (torch.cat([kv[i][j][layer], new[j]], 1) for j in range(2))
            check(out[layer, i].cuda(), ref.attend(q[layer, i][None], kk, vv, 0.125)[0], vv, pool)
    pool.close()


@pytest.mark.parametrize("n_seqs", [128, 129, 1024, 1025])
def test_metadata_packets_of_every_route(n_seqs):
    """Appends and reads whose metadata packet is the largest or the first past
    each route's limit (1 KB and 8 KB; an append destination has 8 bytes)."""
    D = 64
    pool = pool4(1, 1, 1, D, 64, blocks=n_seqs + 1)
    seqs = [pool.create_sequence() for _ in range(n_seqs)]
    g = gen(n_seqs)
    k, v = (rows(g, (1, n_seqs, 1, 1, D), torch.float16) for _ in range(2))
    kb.append_quantize(pool, seqs, 0, k, v)
    got_k, got_v = kb.read_rows(pool, seqs, 0, 1, 1)
    assert torch.equal(got_k, ref.value4(*ref.quantize4(k, 64)).half())
    assert torch.equal(got_v, ref.value4(*ref.quantize4(v, 64)).half())
    pool.close()
