"""Cases of the 4-bit KV cache and of block-sparse decode attention.

Five operators over a paged KV cache of 256-token blocks:

  append   K/V rows quantized to 4 bits as they are written, and read back
  decode   attention of one query token per sequence over the 4-bit cache
  causal   attention of the last n_query cached tokens of each sequence
           (draft verification, prompt chunks) over the 4-bit cache
  select   the blocks of the cache that a cheap score picks for each query
  sparse   select, then decode attention over the picked blocks alone

``run`` has each of them twice: in elementary torch operations (``own`` false)
and as calls of krill_b200 (``own`` true).

Formats. A row of K or V is cut into groups of G elements.
  4 bits: s = f16(f32(max - min) / 15), z = f16(min), code =
          clip(round((x - z) / s), 0, 15), value = code * s + z, every step
          in f32 (s = 0: every code 0). Values beyond +-61440 saturate and
          NaN counts as 0 before anything else.
  8 bits: the cache's int8 format (code = trunc(clip(x - min, in the input
          type) / scale, 0, 255), value in two f16 roundings).
Summary of a full block of T tokens, per channel: mid and half-range of its K
values, in units of sigma = max |k| / 127 rounded to whole numbers. A query
head rounds to whole numbers a of tau = max |q| / 127; its score of a block is
(sum_d a_d mid_d + |a_d| half_d) * sigma * tau, the sum a whole number, and a
kv head's score the largest of its query heads'. The first and the last blocks
are always picked, and of the others the best, the lowest index among equals.
"""
import math

import torch

own = False

T = 64          # tokens of a selectable block (32 for 8 bits at head_dim 256)
SATURATE = 61440.0


def _case(name, op, **kw):
    base = dict(name=name, op=op, bits=4, dtype="bf16", layers=1, seqs=1, hq=32, hkv=8, head_dim=128, group=64,
                len_lo=2048, len_hi=2048, n=1, budget=0, first=0, last=0)
    base.update(kw)
    return base


def listed():
    return [
        # one new token for each of 4 short chats, all 16 layers of a 1B model: launch latency
        _case("append_step", "append", dtype="f16", layers=16, seqs=4, head_dim=64, len_lo=301, len_hi=777, n=1),
        # two prompts of odd length behind a short cached prefix, 8 layers: bandwidth
        _case("append_prompt", "append", layers=8, seqs=2, len_lo=77, len_hi=77, n=2039),
        # one sequence of a 1B model at 2048 tokens, every layer in one call
        _case("decode_single", "decode", dtype="f16", layers=16, seqs=1, head_dim=64, len_lo=2048, len_hi=2048),
        # a continuous batch of 32 ragged sequences of an 8B model, 8 layers
        _case("decode_batch", "decode", layers=8, seqs=32, len_lo=512, len_hi=8192),
        # two long documents, 8 query heads to a kv head, 12 layers
        _case("decode_long", "decode", layers=12, seqs=2, hkv=4, len_lo=32701, len_hi=32768),
        # four drafted tokens of 16 sequences verified at once
        _case("verify_drafts", "causal", layers=8, seqs=16, len_lo=512, len_hi=4096, n=4),
        # a prompt chunk of 512 tokens of 8 sequences behind 4096 cached tokens
        _case("prefill_chunk", "causal", layers=2, seqs=8, len_lo=4608, len_hi=4608, n=512),
        # block choice for the batch above: 1024 of up to 8192 tokens
        _case("select_batch", "select", layers=8, seqs=32, len_lo=512, len_hi=8192, budget=16, first=1, last=2),
        # block choice in two very long documents: 2048 blocks a head
        _case("select_long", "select", layers=4, seqs=2, hkv=4, len_lo=130001, len_hi=131072, budget=64, first=1, last=4),
        # one chat over a long document, two layers: latency of the whole chain
        _case("sparse_single", "sparse", dtype="f16", layers=2, seqs=1, hq=8, hkv=4, head_dim=256, group=256,
              len_lo=16400, len_hi=16400, budget=32, first=1, last=1),
        # 16 long documents, 2048 tokens of each attended
        _case("sparse_batch", "sparse", layers=4, seqs=16, len_lo=8193, len_hi=32768, budget=32, first=1, last=2),
        # the same choice over the 8-bit cache
        _case("sparse_int8", "sparse", bits=8, layers=4, seqs=8, len_lo=4000, len_hi=16384, budget=48, first=1, last=2),
    ]


def draw(rng):
    def spread(lo, hi):  # over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "decode", "decode", "causal", "causal", "select", "sparse", "sparse"])
    head_dim = rng.choice([64, 64, 128, 128, 128, 256])
    bits = rng.choice([4, 4, 8]) if op in ("select", "sparse") else 4
    hkv = rng.choice([1, 2, 4, 8, 16])
    c = dict(op=op, bits=bits, dtype=rng.choice(["f16", "bf16"]), layers=rng.choice([1, 2, 3, 4, 8, 16]), seqs=spread(1, 40),
             hkv=hkv, hq=hkv * rng.choice([1, 2, 3, 4, 7, 8]), head_dim=head_dim, group=rng.choice([64, head_dim]),
             n=1, budget=0, first=0, last=0)
    longest = {"append": 4096, "decode": 40000, "causal": 6000, "select": 131072, "sparse": 65536}[op]
    hi = spread({"append": 1, "decode": 1, "select": 3000}.get(op, 70), longest)
    if op == "append":
        c["n"] = rng.choice([1, 1, 2, spread(3, 2500)])
    if op == "causal":
        c["n"] = min(hi, rng.choice([2, 3, 4, 5, spread(6, 700)]))
    if op in ("select", "sparse"):
        c["first"], c["last"] = rng.choice([0, 1, 2]), rng.choice([1, 1, 2, 4])
        most = max(5, (hi // T - c["first"] - c["last"]) // 2) if op == "select" else 100  # a choice that leaves something out
        c["budget"] = c["first"] + c["last"] + min(most, spread(4 if op == "select" else 1, 100))
    lo = max(c["n"] if op == "causal" else 1, spread(max(1, hi // 16), hi))
    c.update(len_lo=min(lo, hi), len_hi=hi)
    while True:  # never above the largest listed case
        rows = c["layers"] * c["seqs"] * c["hkv"] * (c["n"] if op == "append" else c["len_hi"])
        pairs = c["layers"] * c["seqs"] * c["hq"] * c["n"] * c["len_hi"] if op == "causal" else 0
        if rows * head_dim <= 4.5e8 and pairs * head_dim <= 1.4e11 and pairs <= 1.0e9:
            return c
        if c["layers"] > 1:
            c["layers"] = (c["layers"] + 1) // 2
        elif c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        else:
            c["hkv"], c["hq"] = max(1, c["hkv"] // 2), c["hq"] // c["hkv"] * max(1, c["hkv"] // 2)
            if c["hkv"] == 1 and op != "select":
                c["len_hi"] = max(70, c["len_hi"] // 2)
                c["len_lo"] = min(c["len_lo"], c["len_hi"])
                c["n"] = min(c["n"], c["len_lo"]) if op == "causal" else c["n"]


def _lengths(case):
    """Cached tokens of each sequence, spread over the case's range."""
    lo, hi, n = case["len_lo"], case["len_hi"], case["seqs"]
    at = [(0.31 + 0.6180339887 * i) % 1.0 for i in range(n)]
    got = [int(round(lo * (hi / lo) ** a)) for a in at]
    got[-1] = hi
    return got


def _block(case):
    return 32 if case["bits"] == 8 and case["head_dim"] == 256 else T


def work(case):
    L, H, D, Hq = case["layers"], case["hkv"], case["head_dim"], case["hq"]
    NG = D // case["group"]
    lens = _lengths(case)
    row = D * case["bits"] // 4 + 8 * NG  # cached bytes of one token of one kv head, K and V
    qo = L * case["seqs"] * case["n"] * Hq * D * 4
    if case["op"] == "append":
        rows = L * case["seqs"] * H * case["n"]
        return {"bytes": rows * (4 * D + row + 4 * D), "flops": rows * 2 * D * 8}
    if case["op"] == "decode":
        return {"bytes": L * H * sum(lens) * row + qo, "flops": 4 * L * Hq * D * sum(lens)}
    if case["op"] == "causal":
        n = case["n"]
        pairs = sum(n * (s - n) + n * (n + 1) // 2 for s in lens)
        return {"bytes": L * H * sum(lens) * row + qo, "flops": 4 * L * Hq * D * pairs}
    B = _block(case)
    blocks = sum(-(-s // B) for s in lens)
    picked = sum(min(case["budget"], -(-s // B)) for s in lens)
    choice = {"bytes": L * H * (blocks * (2 * D + 4) + 4 * case["seqs"] * case["budget"]) + qo // 2, "flops": 4 * L * Hq * D * blocks}
    if case["op"] == "select":
        return choice
    return {"bytes": choice["bytes"] + L * H * picked * B * row + qo // 2, "flops": choice["flops"] + 4 * L * Hq * D * picked * B}


# ---------------------------------------------------------------- inputs
def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(case, gen, tokens, is_key):
    """One layer's new K or V rows of every sequence, [seqs, hkv, tokens, D]. Keys have a few strong channels and drift along the text."""
    S, H, D = case["seqs"], case["hkv"], case["head_dim"]
    x = torch.randn(S, H, tokens, D, device="cuda", generator=gen)
    if is_key:
        gain = 1.0 + 2.0 * (torch.rand(1, H, 1, D, device="cuda", generator=gen) > 0.97)
        topics = torch.randn(S, H, tokens // 96 + 1, D, device="cuda", generator=gen)
        x += 0.6 * topics.repeat_interleave(96, dim=2)[:, :, :tokens]
        x *= gain
    return x.to(_dtype(case))


def _inputs(case, seed):
    """(k, v, q): new rows, one [seqs, hkv, tokens, D] for each layer, and the queries [layers, seqs, (n,) hq, D]."""
    gen = _generator(seed)
    tokens = case["n"] if case["op"] == "append" else case["len_hi"]
    k, v = [], []
    for _ in range(case["layers"]):
        k.append(_rows(case, gen, tokens, True))
        v.append(_rows(case, gen, tokens, False))
    shape = [case["layers"], case["seqs"], case["n"], case["hq"], case["head_dim"]]
    q = 1.5 * torch.randn(*(shape if case["op"] == "causal" else shape[:2] + shape[3:]), device="cuda", generator=gen)
    return k, v, q.to(_dtype(case))


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def prepare(case, seed):
    """The queries (or new rows) of the call, and the cache that earlier steps of the program have filled: with ``own`` the framework's
    block pool and its sequences, otherwise the same cache as plain tensors of codes, scales and zeros, padded to the longest sequence."""
    lens = _lengths(case)
    state = {"case": case, "lens": lens, "lens_t": torch.tensor(lens, device="cuda")}
    k, v, state["q"] = _inputs(case, seed)
    append = case["op"] == "append"
    if append:
        state["k"], state["v"] = torch.stack(k), torch.stack(v)
    if own:
        import krill_b200 as kb
        state["kb"] = kb
        pool = kb.KVPool(case["layers"], case["hkv"], case["hq"], case["head_dim"],
                         num_blocks=sum((s + (case["n"] if append else 0) + 255) // 256 for s in lens), group_size=case["group"],
                         kv_format=kb.KV_INT4 if case["bits"] == 4 else kb.KV_INT8,
                         block_summaries=case["op"] in ("select", "sparse"))
        state["pool"], state["seqs"] = pool, [pool.create_sequence() for _ in lens]
        for i, s in enumerate(lens):
            for layer in range(case["layers"]):
                if append:  # what is cached already does not enter the new rows
                    old = torch.zeros(1, 1, case["hkv"], s, case["head_dim"], dtype=_dtype(case), device="cuda")
                    kb.append_quantize(pool, [state["seqs"][i]], layer, old, old)
                else:
                    kb.append_quantize(pool, [state["seqs"][i]], layer, k[layer][i, :, :s].contiguous()[None, None],
                                       v[layer][i, :, :s].contiguous()[None, None])
        state["out"] = torch.empty_like(state["q"])
        return state
    if not append:
        tail = -case["len_hi"] % _block(case)  # the cache ends in a whole block; rows past a sequence's length hold zeros
        live = (torch.arange(case["len_hi"], device="cuda") < state["lens_t"][:, None])[:, None, :, None]
        for name, rows in (("k", k), ("v", v)):
            got = []
            for layer in range(case["layers"]):
                x = torch.nn.functional.pad(torch.where(live, rows[layer], 0), (0, 0, 0, tail))
                rows[layer] = None
                got.append(_quantize(case, x))
            state[name] = [torch.stack([g[j] for g in got]) for j in range(3)]
        if case["op"] in ("select", "sparse"):
            got = [_summary(case, _values(case, [t[layer] for t in state["k"]])) for layer in range(case["layers"])]
            state["summary"] = [torch.stack([g[j] for g in got]) for j in range(3)]
            if case["op"] == "select":
                del state["k"]
        if case["op"] == "select":
            del state["v"]
    return state


# ---------------------------------------------------------------- the plain forms
def _over(x, n):
    """x / n, correctly rounded (a Python number as divisor becomes a product with its reciprocal on the GPU)."""
    return x / torch.full((), n, dtype=x.dtype, device=x.device)


def _groups(case, x):
    return x.reshape(*x.shape[:-1], case["head_dim"] // case["group"], case["group"])


def _quantize(case, x):
    """(codes u8, scale f16, zero f16) of rows [..., D]."""
    if case["bits"] == 8:
        g = _groups(case, x)
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        scale = _over((hi.float() - lo.float()).to(x.dtype).float(), 255.0).clamp_min(1e-8)
        codes = ((g.float() - lo.float()).to(x.dtype).float() / scale).clamp(0.0, 255.0).trunc()
        return codes.to(torch.uint8).reshape(x.shape), scale[..., 0].half(), lo[..., 0].half()
    g = _groups(case, torch.nan_to_num(x.float(), nan=0.0, posinf=SATURATE, neginf=-SATURATE).clamp(-SATURATE, SATURATE))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale, zero = _over(hi - lo, 15.0).half(), lo.half()
    codes = torch.where(scale > 0, (g - zero.float()) / scale.float(), 0.0).round().clamp(0.0, 15.0)
    return codes.to(torch.uint8).reshape(x.shape), scale[..., 0], zero[..., 0]


def _values(case, cached):
    """What the codes stand for, in f32."""
    codes, scale, zero = cached
    g = _groups(case, codes)
    if case["bits"] == 8:  # the format's two f16 roundings
        return ((g.half() * scale[..., None]) + zero[..., None]).reshape(codes.shape).float()
    return (g.float() * scale[..., None].float() + zero[..., None].float()).reshape(codes.shape)


def _summary(case, k):
    """(mid, half-range, sigma) of every whole block of k [..., tokens, D]."""
    b = k.reshape(*k.shape[:-2], k.shape[-2] // _block(case), _block(case), k.shape[-1])
    lo, hi = b.amin(-2), b.amax(-2)
    sigma = _over(torch.maximum(lo.abs(), hi.abs()).amax(-1, keepdim=True), 127.0)
    inverse = torch.where(sigma > 0, 1.0 / sigma, 0.0)
    return (((hi + lo) * 0.5) * inverse).round(), (((hi - lo) * 0.5) * inverse).round(), sigma[..., 0]


def _blocks_of(state):
    B = _block(state["case"])
    return (state["lens_t"] + B - 1) // B


def _pick(state):
    """Picked block indices [layers, seqs, hkv, budget], ascending, -1 past the last."""
    case, (mid, half, sigma) = state["case"], state["summary"]
    L, S, H, g = case["layers"], case["seqs"], case["hkv"], case["hq"] // case["hkv"]
    q = state["q"].float().reshape(L, S, H, g, case["head_dim"])
    q = torch.where(q.isfinite(), q, 0.0)
    tau = _over(q.abs().amax(-1, keepdim=True), 127.0)
    a = (q * torch.where(tau > 0, 1.0 / tau, 0.0)).round().clamp(-127.0, 127.0)
    whole = torch.matmul(a, mid.mT) + torch.matmul(a.abs(), half.mT)  # whole numbers below 2^24
    score = ((whole * sigma[..., None, :]) * tau).amax(-2)  # [L, S, H, blocks]
    index = torch.arange(score.shape[-1], device="cuda")
    n = _blocks_of(state)[:, None]
    forced = (index < case["first"]) | (index >= n - case["last"])
    score = torch.where(forced[:, None], math.inf, score)
    score = torch.where((index < n)[:, None], score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    order = torch.nn.functional.pad(order, (0, max(0, case["budget"] - order.shape[-1])), value=0)[..., : case["budget"]]
    rank = torch.arange(case["budget"], device="cuda")
    count = torch.clamp(n, max=case["budget"])[:, None]
    order = torch.where(rank < count, order, 1 << 30).sort(dim=-1).values
    return torch.where(rank < count, order, -1).to(torch.int32)


def _attend(case, q, k, v, seen):
    """Softmax attention: q [L, S, n, hq, D], k/v [L, S, hkv, t, D], seen broadcastable to [L, S, hkv, n, 1, t]."""
    L, S, n, hq, D = q.shape
    H = case["hkv"]
    qg = q.float().reshape(L, S, n, H, hq // H, D).permute(0, 1, 3, 2, 4, 5)  # [L, S, H, n, g, D]
    score = torch.matmul(qg.reshape(L, S, H, -1, D), k.mT).reshape(L, S, H, n, hq // H, -1) * _scale(case)
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(L, S, H, n * (hq // H), -1), v).reshape(L, S, H, n, hq // H, D)
    return out.permute(0, 1, 3, 2, 4, 5).reshape(L, S, n, hq, D).to(q.dtype)


def _plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "append":
        return tuple(_values(case, _quantize(case, state[x])).half() for x in ("k", "v"))
    if op == "select":
        return _pick(state)
    lens = state["lens_t"][:, None, None, None, None]
    if op == "sparse":
        picked, B, D = _pick(state), _block(case), case["head_dim"]
        at = picked.clamp_min(0).long()
        pos = at[..., None] * B + torch.arange(B, device="cuda")  # [L, S, H, budget, B]
        seen = ((pos < state["lens_t"][:, None, None, None]) & (picked >= 0)[..., None]).flatten(-2)[..., None, None, :]
        flat = pos.flatten(-2)[..., None]
        k, v = (_values(case, [torch.gather(t, 3, flat.expand(*flat.shape[:-1], t.shape[-1])) for t in state[x]]) for x in ("k", "v"))
        return _attend(case, state["q"].unsqueeze(2), k, v, seen).squeeze(2), picked
    index = torch.arange(state["k"][0].shape[3], device="cuda")
    if op == "decode":
        return _attend(case, state["q"].unsqueeze(2), _values(case, state["k"]), _values(case, state["v"]), index < lens).squeeze(2)
    n = case["n"]
    own_pos = lens - n + torch.arange(n, device="cuda")[:, None, None]
    return _attend(case, state["q"], _values(case, state["k"]), _values(case, state["v"]), index <= own_pos)


def _calls(state):
    case, kb, pool, seqs = state["case"], state["kb"], state["pool"], state["seqs"]
    op = case["op"]
    if op == "append":
        [s.truncate(n) for s, n in zip(seqs, state["lens"])]  # the rows of the pass before are dropped
        kb.append_quantize(pool, seqs, 0, state["k"], state["v"])
        return kb.read_rows(pool, seqs, 0, case["layers"], case["n"], starts=state["lens"])
    if op == "decode":
        return kb.decode_attention(pool, seqs, 0, state["q"], state["out"], _scale(case))
    if op == "causal":
        return kb.prefill_attention(pool, seqs, 0, state["q"], state["out"], _scale(case))
    if op == "select":
        return kb.select_blocks(pool, seqs, 0, state["q"], case["budget"], first_blocks=case["first"], last_blocks=case["last"])
    return kb.sparse_decode_attention(pool, seqs, 0, state["q"], state["out"], _scale(case), case["budget"],
                                      first_blocks=case["first"], last_blocks=case["last"], return_blocks=True)


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------- in 64 bits
def _exact_values(case, x):
    """Rows [..., D] through the format, in 64 bits (8 bits: with the format's own roundings)."""
    D, G = case["head_dim"], case["group"]
    d = x.double().unflatten(-1, (D // G, G))
    if case["bits"] == 8:
        lo, hi = d.amin(-1, keepdim=True), d.amax(-1, keepdim=True)
        scale = ((hi - lo).to(x.dtype).double() / 255.0).float().clamp_min(1e-8)
        code = ((d - lo).to(x.dtype).float() / scale).clamp(0, 255).floor().half()
        return ((code * scale.half()) + lo.half()).flatten(-2).double()
    d = torch.nan_to_num(d, nan=0.0).clamp(-SATURATE, SATURATE)
    lo = d.amin(-1, keepdim=True)
    s, z = ((d.amax(-1, keepdim=True) - lo).float().double() / 15.0).float().half().double(), lo.half().double()
    code = torch.where(s > 0, (d - z) / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15)
    return (code * s + z).flatten(-2)


def _exact_pick(case, q, k, length):
    """Picked blocks of one layer of one sequence: q [hq, D], k [hkv, tokens, D] in 64 bits. The roundings to whole numbers and of the scores are the definition's."""
    B, H, D = _block(case), case["hkv"], case["head_dim"]
    n, whole = -(-length // B), length // B
    b = k[:, : whole * B].reshape(H, whole, B, D)
    lo, hi = b.amin(2), b.amax(2)
    lo, hi = lo.float(), hi.float()  # a block's bounds are kept in f32
    sigma = (torch.maximum(lo.abs(), hi.abs()).amax(-1).double() / 127.0).float()
    inv = torch.where(sigma > 0, 1.0 / sigma, 0.0)[..., None]
    mid, half = ((0.5 * (hi + lo)) * inv).round().double(), ((0.5 * (hi - lo)) * inv).round().double()
    q = torch.nan_to_num(q.float(), nan=0.0, posinf=0.0, neginf=0.0).reshape(H, -1, D)
    tau = (q.abs().amax(-1).double() / 127.0).float()
    a = (q * torch.where(tau > 0, 1.0 / tau, 0.0)[..., None]).round().clamp(-127, 127).double()
    total = torch.einsum("hgd,hbd->hgb", a, mid) + torch.einsum("hgd,hbd->hgb", a.abs(), half)
    score = ((total.float() * sigma[:, None, :]) * tau[..., None]).amax(1)
    picked = []
    for h in range(H):
        always = set(range(min(case["first"], n))) | set(range(max(0, n - case["last"]), n))
        rest = [i for i in range(whole) if i not in always]
        s = score[h].tolist()
        rest.sort(key=lambda i: (-s[i], i))
        got = sorted(list(always) + rest[: max(0, case["budget"] - len(always))])[: case["budget"]]
        picked.append(got + [-1] * (case["budget"] - len(got)))
    return torch.tensor(picked, dtype=torch.int32, device="cuda")


def exact(case, seed):
    L, H, D = case["layers"], case["hkv"], case["head_dim"]
    k, v, q = _inputs(case, seed)
    if case["op"] == "append":
        return tuple(torch.stack([_exact_values(case, r) for r in rows]) for rows in (k, v))
    g, n, B = case["hq"] // H, case["n"], _block(case)
    outs, picks = [], []
    for layer in range(L):
        for i, length in enumerate(_lengths(case)):
            kk = _exact_values(case, k[layer][i, :, :length])
            ql = q[layer, i]
            if case["op"] in ("select", "sparse"):
                picks.append(_exact_pick(case, ql, kk, length))
                if case["op"] == "select":
                    continue
            vv = _exact_values(case, v[layer][i, :, :length])
            qq = ql.double().reshape(n, H, g, D)
            score = torch.einsum("nhgd,htd->hngt", qq, kk) / math.sqrt(D)
            pos = torch.arange(length, device="cuda")
            if case["op"] == "sparse":
                hit = torch.zeros(H, -(-length // B) + 1, dtype=torch.bool, device="cuda")
                hit.scatter_(1, torch.where(picks[-1] >= 0, picks[-1], hit.shape[1] - 1).long(), True)
                score.masked_fill_(~hit[:, pos // B][:, None, None, :], -math.inf)
            else:
                late = pos > (length - n + torch.arange(n, device="cuda"))[:, None]
                score.masked_fill_(late[None, :, None, :], -math.inf)
            out = torch.einsum("hngt,htd->nhgd", torch.softmax(score, -1), vv)
            outs.append(out.reshape(n, case["hq"], D))
    picks = torch.stack(picks).reshape(L, case["seqs"], H, case["budget"]) if picks else None
    if case["op"] == "select":
        return picks
    out = torch.stack(outs).reshape(L, case["seqs"], n, case["hq"], D)
    if case["op"] == "decode":
        return out.squeeze(2)
    return out if case["op"] == "causal" else (out.squeeze(2), picks)
