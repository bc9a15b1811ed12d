"""4-bit pools at the edges of the format: restored metadata that no append
would store."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

import krill_b200 as kb  # noqa: E402
from tests import _int4 as ref  # noqa: E402
from tests.test_gpu_int4 import check, gen, pool4, rows  # noqa: E402

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
