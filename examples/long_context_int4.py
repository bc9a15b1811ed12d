"""A long conversation on a 4-bit pool: the prompt is appended and attended in
chunks, then tokens are decoded over the picked blocks only, with a dense step
beside each for comparison, and a few drafted tokens are verified and rolled
back.

    python examples/long_context_int4.py [--prompt 32768] [--layers 8] ...

Keys are a topic, which a run of tokens shares as neighbouring tokens of a text
do, plus noise. Every query looks for one cached token (the needle of its
step), so that what the attention should find is known: the block of the
needle's topic has to be among the picked ones, and the output close to the
dense one. (Keys without anything in common in a block bound every block alike:
no choice by bounds could tell them apart.)
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import krill_b200 as kb  # noqa: E402


def timed(f):
    """(result, device milliseconds) of one call."""
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    y = f()
    b.record()
    b.synchronize()
    return y, a.elapsed_time(b)


def run(prompt=32768, chunk=512, steps=16, drafts=4, layers=8, kv_heads=8, q_heads=32, head_dim=128, max_blocks=32,
        dtype=torch.bfloat16, seed=0):
    """Runs the conversation; returns what it measured."""
    dev, g = torch.device("cuda"), torch.Generator(device="cuda")
    g.manual_seed(seed)
    scale = head_dim**-0.5
    group = min(64, head_dim)

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=g).to(dtype)

    pool = kb.KVPool(layers, kv_heads, q_heads, head_dim, num_blocks=(prompt + steps + drafts) // 256 + 2,
                     group_size=group, kv_format=kb.KV_INT4, block_summaries=True)
    seq = pool.create_sequence()
    T, ratio = pool.select_tokens, q_heads // kv_heads
    topics = 2.0 * torch.randn(layers, 1, kv_heads, (prompt + steps + drafts) // T + 1, head_dim, device=dev, generator=g)

    def keys(n):
        """Keys of the next n tokens."""
        at = torch.arange(seq.length(0), seq.length(0) + n, device=dev) // T
        noise = torch.randn(layers, 1, kv_heads, n, head_dim, device=dev, generator=g)
        return (topics[:, :, :, at] + 0.5 * noise).to(dtype)

    out = {"bytes_per_token": 2 * layers * kv_heads * (head_dim // 2 + 4 * head_dim // group),
           "f16_bytes_per_token": 4 * layers * kv_heads * head_dim, "prefill_ms": 0.0, "sparse_ms": 0.0, "dense_ms": 0.0,
           "found": 0, "searched": 0, "error": 0.0}

    # the prompt, chunk by chunk: quantize and append, then attend
    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        k, v, q = keys(n), rand(layers, 1, kv_heads, n, head_dim), rand(layers, 1, n, q_heads, head_dim)

        def step():
            kb.append_quantize(pool, [seq], 0, k, v)
            return kb.prefill_attention(pool, [seq], 0, q, torch.empty_like(q), scale)

        out["prefill_ms"] += timed(step)[1]

    # decoding: one token a step, looking for a token somewhere in the prompt
    for i in range(steps):
        kb.append_quantize(pool, [seq], 0, keys(1), rand(layers, 1, kv_heads, 1, head_dim))
        needle = (i * 7919 + 11) % prompt
        key, _ = kb.read_rows(pool, [seq], 0, layers, 1, starts=[needle], dtype=dtype)
        q = (4.0 * key[:, :, :, 0]).repeat_interleave(ratio, 2).contiguous()  # [layers, 1, q_heads, head_dim]
        (sparse, picked), ms = timed(lambda: kb.sparse_decode_attention(
            pool, [seq], 0, q, torch.empty_like(q), scale, max_blocks, return_blocks=True))
        dense, dense_ms = timed(lambda: kb.decode_attention(pool, [seq], 0, q, torch.empty_like(q), scale))
        out["sparse_ms"] += ms / steps
        out["dense_ms"] += dense_ms / steps
        out["found"] += int((picked == needle // T).any(-1).sum())
        out["searched"] += layers * kv_heads
        out["error"] = max(out["error"], float((sparse.float() - dense.float()).norm() / dense.float().norm()))

    # drafted tokens: appended, verified in one call, rolled back
    kb.append_quantize(pool, [seq], 0, keys(drafts), rand(layers, 1, kv_heads, drafts, head_dim))
    q = rand(layers, 1, drafts, q_heads, head_dim)
    _, out["verify_ms"] = timed(lambda: kb.verify_attention(pool, [seq], 0, q, torch.empty_like(q), scale))
    seq.truncate(prompt + steps)
    out["length"] = seq.length(0)
    pool.close()
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("prompt", 32768), ("chunk", 512), ("steps", 16), ("drafts", 4), ("layers", 8),
                          ("kv-heads", 8), ("q-heads", 32), ("head-dim", 128), ("max-blocks", 32)):
        ap.add_argument("--" + name, type=int, default=default)
    a = vars(ap.parse_args())
    run(**a)  # kernels loaded, memory reserved
    r = run(**a)
    print("cache     %d bytes a token (16 bits: %d)" % (r["bytes_per_token"], r["f16_bytes_per_token"]))
    print("prefill   %.2f ms for %d tokens" % (r["prefill_ms"], a["prompt"]))
    print("decode    %.3f ms a step over picked blocks, %.3f ms dense" % (r["sparse_ms"], r["dense_ms"]))
    print("verify    %.3f ms for %d drafted tokens" % (r["verify_ms"], a["drafts"]))
    print("needles   %d of %d found, outputs within %.3g of the dense ones" % (r["found"], r["searched"], r["error"]))


if __name__ == "__main__":
    main()
