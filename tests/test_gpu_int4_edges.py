"""4-bit pools at the edges of the format: restored metadata that no append
would store, and what the prompt path's f16 values cost against the format's."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402
from tests.test_gpu_int4 import check, fill, gen, pool4, rows  # noqa: E402

BAD = [math.inf, -math.inf, math.nan, 65504.0, -65504.0]


def snapshot(g, hkv, n, D, G, dtype):
    """Codes and metadata of normal rows, as an append would store them."""
    k, v = (ref.quantize4(rows(g, (hkv, n, D), dtype), G) for _ in range(2))
    return kb.QuantizedKVSnapshot(k[0], v[0], k[1], k[2], v[1], v[2])


def test_restored_metadata_is_kept_in_range():
    """Restored zeros end in +-61440, scales where every code's value is within
    f16's range, NaN as 0; what an append stores comes back bit for bit."""
    D, G, hkv = 64, 64, 1
    grid = [(s, z) for s in BAD + [0.0, 1.0, -3.0, 8192.0, 30000.0] for z in BAD + [0.0, 61440.0, -61440.0, 5.0]]
    n = len(grid)
    codes = torch.full((hkv, n, D), 15, dtype=torch.uint8, device="cuda")
    s = torch.tensor([x[0] for x in grid], device="cuda").half().reshape(hkv, n, 1)
    z = torch.tensor([x[1] for x in grid], device="cuda").half().reshape(hkv, n, 1)
    pool = pool4(1, hkv, hkv, D, G, blocks=4)
    seq = pool.create_sequence()
    seq.restore_quantized(0, kb.QuantizedKVSnapshot(codes, codes, s, z, s, z))
    got = seq.quantized_snapshot(0)
    for gs, gz in ((got.key_scales, got.key_zeros), (got.value_scales, got.value_zeros)):
        wz = torch.where(z.isnan(), torch.zeros_like(z), z).clamp(-61440, 61440)
        ws = torch.where(s.isnan(), torch.zeros_like(s), s).double()
        assert torch.equal(gz, wz)
        hi, lo = (65504.0 - wz.double()) / 15, (-65504.0 - wz.double()) / 15
        inside = (ws <= hi) & (ws >= lo)
        assert torch.equal(gs[inside].double(), ws[inside])
        assert ((gs.double() <= hi) & (gs.double() >= lo)).all()
        # what is clamped ends within one f16 step of the bound
        bound = torch.where(ws > hi, hi, lo)[~inside]
        assert ((gs[~inside].double() - bound).abs() <= bound.abs() * 2.0 ** -10).all()
    kk, vv = kb.read_rows(pool, [seq], 0, 1, n, dtype=torch.float16)
    assert torch.isfinite(kk).all() and torch.isfinite(vv).all()
    new = pool.create_sequence()
    g = gen(51)
    x = rows(g, (1, 1, hkv, 90, D), torch.bfloat16, odd=True)
    kb.append_quantize(pool, [new], 0, x, x)
    a = new.quantized_snapshot(0)
    seq.restore_quantized(0, a)
    b = seq.quantized_snapshot(0)
    assert torch.equal(a.key_scales, b.key_scales) and torch.equal(a.value_zeros, b.value_zeros)
    pool.close()


@pytest.mark.parametrize("D,G,hq,hkv,nq", [
    (128, 64, 32, 8, 1),    # one query: the bad token is the last
    (128, 64, 32, 8, 4),    # two query tiles
    (64, 64, 8, 2, 3),
    (256, 64, 8, 4, 5),
    (128, 64, 32, 8, 40),   # the prompt path
])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_masked_token_with_bad_metadata(D, G, hq, hkv, nq, bad):
    """A token restored with infinite or NaN scales and zeros in the middle of
    the queries' bounds: the queries before it are exact, the others finite."""
    n, scale = 200, 0.1
    g = gen(D + nq)
    snap = snapshot(g, hkv, n, D, G, torch.bfloat16)
    at = n - (nq + 1) // 2  # seen by the last queries only
    kk = ref.value4(snap.keys, snap.key_scales, snap.key_zeros)
    vv = ref.value4(snap.values, snap.value_scales, snap.value_zeros)
    for m in (snap.key_scales, snap.key_zeros, snap.value_scales, snap.value_zeros):
        m[:, at] = bad
    pool = pool4(1, hkv, hq, D, G, blocks=4)
    seq = pool.create_sequence()
    seq.restore_quantized(0, snap)
    q = torch.randn(1, 1, nq, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.empty(1, 1, nq, hq, D, device="cuda")
    kb.verify_attention(pool, [seq], 0, q, out, scale)
    assert torch.isfinite(out).all()
    before = at - (n - nq)  # queries whose own token comes before it
    if before > 0:
        seen = (torch.arange(n, device="cuda")[None] <= (n - nq + torch.arange(nq, device="cuda"))[:, None])[:, None]
        if nq * hq // hkv >= 64:  # the prompt path rounds K and V to f16
            kk, vv = kk.half().double(), vv.half().double()
        want = ref.attend(q[0, 0], kk, vv, scale, seen)[:before]
        check(out[0, 0, :before], want, vv * 2, pool)
    pool.close()


def test_scatter_back():
    """Stacked sequences grown by new rows and written back."""
    D, G, hkv, steps = 128, 64, 2, 5
    g = gen(52)
    pool = pool4(2, hkv, 4, D, G, blocks=32)
    lens = [70, 300, 1]
    seqs, kv = fill(pool, lens, torch.bfloat16, g, 2)
    for layer in range(2):
        st = kb.stack_caches_left_padded_quantized(pool, seqs, layer)
        s_max = st.keys.shape[2]
        new = snapshot(g, 3 * hkv, steps, D, G, torch.bfloat16)
        grown = kb.QuantizedKVSnapshot(*[
            torch.cat([getattr(st, name), getattr(new, name).reshape(3, hkv, steps, -1)], 2).contiguous()
            for name in ("keys", "values", "key_scales", "key_zeros", "value_scales", "value_zeros")])
        kb.scatter_back(pool, seqs, layer, grown, lens, s_max, steps)
        for i, n in enumerate(lens):
            got = seqs[i].quantized_snapshot(layer)
            for name in ("keys", "values", "key_scales", "key_zeros", "value_scales", "value_zeros"):
                assert torch.equal(getattr(got, name), getattr(grown, name)[i, :, s_max - n:])
    q = torch.randn(2, 3, 4, D, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.empty(2, 3, 4, D, device="cuda")
    kb.decode_attention(pool, seqs, 0, q, out, 0.09)
    for layer in range(2):
        for i in range(3):
            x = seqs[i].quantized_snapshot(layer)
            k, v = ref.value4(x.keys, x.key_scales, x.key_zeros), ref.value4(x.values, x.value_scales, x.value_zeros)
            check(out[layer, i], ref.attend(q[layer, i][None], k, v, 0.09)[0], v, pool)
    pool.close()


@pytest.mark.parametrize("D,G", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_read_rows_int8(D, G, dtype):
    """Rows of an int8 pool read back: the format's two f16 roundings, then one
    to the output's type."""
    layers, hkv, lens = 2, 2, [300, 77, 513]
    g = gen(D + G)
    pool = kb.KVPool(layers, hkv, 4, D, num_blocks=16, group_size=G)
    seqs, kept = [], []
    for n in lens:
        seqs.append(pool.create_sequence())
        k, v = (rows(g, (layers, 1, hkv, n, D), dtype) for _ in range(2))
        kb.append_quantize(pool, [seqs[-1]], 0, k, v)
        kept.append([ref.value8(*ref.quantize8(x[:, 0], G)) for x in (k, v)])
    for starts, n in (([0, 0, 0], 77), ([63, 1, 255], 65), ([299, 76, 512], 1), ([10, 5, 500], 13)):
        for out_dtype in (torch.float16, torch.bfloat16, torch.float32):
            got = kb.read_rows(pool, seqs, 0, layers, n, starts=starts, dtype=out_dtype)
            for i, at in enumerate(starts):
                for x, y in zip(got, kept[i]):
                    assert torch.equal(x[:, i], y[:, :, at:at + n].to(out_dtype))
    win = kb.KVPool(1, hkv, 4, D, num_blocks=16, group_size=G, window=100, max_append=200)
    seq = win.create_sequence()
    for n in (200, 200, 130, 200):
        k, v = (rows(g, (1, 1, hkv, n, D), dtype) for _ in range(2))
        kb.append_quantize(win, [seq], 0, k, v)
    got = kb.read_rows(win, [seq], 0, 1, 200, starts=[530])
    for x, y in zip(got, (k, v)):
        assert torch.equal(x[0, 0], ref.value8(*ref.quantize8(y[0, 0], G)).half())
    pool.close()
    win.close()


@pytest.mark.parametrize("D,G,hq,hkv,nq,n", [(128, 64, 32, 8, 64, 700), (64, 64, 8, 2, 130, 207), (128, 128, 16, 16, 64, 64)])
def test_prompt_path_against_the_format(D, G, hq, hkv, nq, n):
    """Prompt chunks on tcgen05 take K and V rounded to f16, against the values
    of the format. With |k| and |v| each off by 2^-11 at most, a query's scores
    move by e = scale * max_t sum_d |q_d k_td| * 2^-11, its weights by a factor
    exp(+-2e), its output by (exp(2e) - 1) spans of v; v itself adds 2^-11 of
    its largest magnitude, and the f16 weights what tests/_int4.py bounds."""
    scale = 1 / math.sqrt(D)
    g = gen(n)
    pool = pool4(1, hkv, hq, D, G)
    seqs, kv = fill(pool, [n], torch.bfloat16, g, 1)
    q = torch.randn(1, 1, nq, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.empty(1, 1, nq, hq, D, device="cuda")
    kb.prefill_attention(pool, seqs, 0, q, out, scale)
    assert "umma" in pool.last_kernels()
    k, v = kv[0][0][0], kv[0][1][0]
    seen = (torch.arange(n, device="cuda")[None] <= (n - nq + torch.arange(nq, device="cuda"))[:, None])[:, None]
    want = ref.attend(q[0, 0], k, v, scale, seen)
    reach = torch.einsum("nhgd,htd->nhgt", q[0, 0].double().abs().reshape(nq, hkv, hq // hkv, D), k.abs()).amax(-1)
    e = scale * reach.reshape(nq, hq, 1) * 2.0 ** -11
    span = (v.amax() - v.amin()).item()
    bound = torch.expm1(2 * e) * span + v.abs().max().item() * 2.0 ** -11 + ref.tolerance(2 * v, out.dtype, want)
    err = (out[0, 0].double() - want).abs()
    assert (err <= bound).all(), f"{err.max().item():.3e}"
    pool.close()


@pytest.mark.parametrize("D,hq,hkv,split", [(128, 32, 8, 256), (64, 4, 2, 64), (256, 4, 2, 128)])
def test_fixed_pieces_do_not_depend_on_the_batch(D, hq, hkv, split):
    """With a fixed split_tokens a sequence's output is the same alone and in
    a batch, bit for bit."""
    lens, layers = [300, 900, 4000, 65], 2
    g = gen(D + split)
    pool = pool4(layers, hkv, hq, D, 64, split_tokens=split)
    seqs, _ = fill(pool, lens, torch.bfloat16, g, layers)
    q = torch.randn(layers, 4, hq, D, device="cuda", generator=g).to(torch.bfloat16)
    out, one = torch.empty(layers, 4, hq, D, device="cuda"), torch.empty(layers, 1, hq, D, device="cuda")
    kb.decode_attention(pool, seqs, 0, q, out, 0.09)
    for i in range(4):
        kb.decode_attention(pool, [seqs[i]], 0, q[:, i:i + 1].contiguous(), one, 0.09)
        assert torch.equal(one[:, 0], out[:, i])
    pool.close()
