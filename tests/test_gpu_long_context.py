"""The long-conversation example: 4-bit append, chunked prefill, block choice,
sparse and dense decode, read-back, verify and rollback in one run."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("needs a CUDA device", allow_module_level=True)

_path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "long_context_int4.py")
_spec = importlib.util.spec_from_file_location("long_context_int4", _path)
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


@pytest.mark.parametrize("kw", [
    dict(prompt=5000, chunk=512, steps=6, layers=2, kv_heads=2, q_heads=8, head_dim=128, max_blocks=16),
    dict(prompt=2047, chunk=300, steps=6, layers=3, kv_heads=1, q_heads=8, head_dim=64, max_blocks=12, dtype=torch.float16),
    dict(prompt=1500, chunk=1500, steps=4, layers=1, kv_heads=4, q_heads=4, head_dim=256, max_blocks=10),
])
def test_every_needle_is_found(kw):
    """A query of 4 times a key (2 * topic + noise / 2, unit normals) has 16 D with
    the middle of its own block and N(0, 16 sqrt(D)) with the others' middles,
    the blocks' extents adding nearly the same to all: of at most 80 blocks the
    needle's comes first by 16 D - 16 sqrt(D) * 2.5 > 9 sigma at D = 64. So far
    below, the others weigh under e^-40 in the dense softmax, and both outputs
    are sums over the same tokens: they differ by their roundings to 16 bits
    (2^-8 at the most) and by half-precision weights, together below 1e-2. An
    unpicked block leaves an unrelated output (difference above 1)."""
    r = example.run(**kw)
    assert r["found"] == r["searched"] == kw["steps"] * kw["layers"] * kw["kv_heads"]
    assert r["error"] < 1e-2
    assert r["length"] == kw["prompt"] + kw["steps"]
