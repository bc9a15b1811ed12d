"""Plain restatement of the 4-bit cache format, of softmax attention and of the
block choice, in 64 bits (the format's own f32 / f16 steps where it defines
them). Test infrastructure; torch on whatever device the inputs are on."""
import math

import torch

SAT = 61440.0


def over(x, n):
    """x / n, correctly rounded: a tensor divided by a Python number becomes a
    product with the number's reciprocal on the GPU."""
    return x / torch.full((), n, dtype=x.dtype, device=x.device)


def quantize4(x, G):
    """x [..., D] f16/bf16 -> (codes u8, scale f16, zero f16)."""
    g = x.float().unflatten(-1, (x.shape[-1] // G, G))
    g = torch.where(g.isnan(), torch.zeros_like(g), g).clamp(-SAT, SAT)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    s, z = over(hi - lo, 15.0).half(), lo.half()
    q = ((g - z.float()) / torch.where(s > 0, s, torch.ones_like(s)).float()).round().clamp(0, 15)
    q = torch.where(s > 0, q, torch.zeros_like(q))
    return q.to(torch.uint8).flatten(-2), s[..., 0], z[..., 0]


def value4(codes, s, z):
    """Values in f64 (a 4-bit code times an 11-bit scale plus a zero: exact)."""
    G = codes.shape[-1] // s.shape[-1]
    return (codes.double().unflatten(-1, (s.shape[-1], G)) * s[..., None].double() + z[..., None].double()).flatten(-2)


def quantize8(x, G):
    """The int8 format (f32 quantizer): (codes u8, scale f16, zero f16)."""
    g = x.float().unflatten(-1, (x.shape[-1] // G, G))
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    s = over((hi - lo).to(x.dtype).float(), 255.0).clamp_min(1e-8)
    q = ((g - lo).to(x.dtype).float() / s).clamp(0, 255).floor()
    return q.to(torch.uint8).flatten(-2), s[..., 0].half(), lo[..., 0].half()


def value8(codes, s, z):
    G = codes.shape[-1] // s.shape[-1]
    c = codes.half().unflatten(-1, (s.shape[-1], G))
    return ((c * s[..., None]) + z[..., None]).flatten(-2).double()


def attend(q, k, v, scale, seen=None):
    """q [n, hq, D], k/v [hkv, t, D] f64 -> [n, hq, D]; seen [n or 1, hkv or 1, t] bool."""
    n, hq, D = q.shape
    H = k.shape[0]
    s = torch.einsum("nhgd,htd->nhgt", q.double().reshape(n, H, hq // H, D), k) * scale
    if seen is not None:
        s = s.masked_fill(~seen[:, :, None, :], -math.inf)
    return torch.einsum("nhgt,htd->nhgd", torch.softmax(s, -1), v).reshape(n, hq, D)


def summary(k, T):
    """k [hkv, tokens, D] f64, whole blocks -> (mid, half, sigma) per block, f32."""
    b = k.float().unflatten(1, (k.shape[1] // T, T))
    lo, hi = b.min(2).values, b.max(2).values
    sigma = over(torch.maximum(lo.abs(), hi.abs()).max(-1).values, 127.0)
    inv = torch.where(sigma > 0, 1.0 / sigma, torch.zeros_like(sigma))[..., None]
    return (((hi + lo) * 0.5) * inv).round(), (((hi - lo) * 0.5) * inv).round(), sigma


def pick(q, k, length, T, budget, first, last):
    """Picked blocks of one sequence: q [hq, D] 16-bit, k [hkv, >= length, D] f64 -> list of hkv lists."""
    H, D = k.shape[0], k.shape[2]
    n, full = -(-length // T), length // T
    if n <= budget:
        return [list(range(n))] * H
    mid, half, sigma = summary(k[:, : full * T], T)
    x = q.float()
    x = torch.where(x.isfinite(), x, torch.zeros_like(x)).reshape(H, -1, D)
    tau = over(x.abs().max(-1).values, 127.0)
    a = (x * torch.where(tau > 0, 1.0 / tau, torch.zeros_like(tau))[..., None]).round().clamp(-127, 127).double()
    total = torch.einsum("hgd,hbd->hgb", a, mid.double()) + torch.einsum("hgd,hbd->hgb", a.abs(), half.double())
    score = ((total.float() * sigma[:, None, :]) * tau[..., None]).max(1).values.tolist()
    got = []
    for h in range(H):
        always = sorted(set(range(first)) | set(range(n - last, n)))
        rest = sorted((i for i in range(first, n - last)), key=lambda i: (-score[h][i], i))
        got.append(sorted(always + rest[: budget - len(always)]))
    return got


def tolerance(v, out_dtype, ref):
    """Bound of |out - ref| for decode over values v: the softmax weights times
    the scale are rounded to f16 (2^-11 relative) while they multiply values at
    most half a group's range from its middle; f32 steps (scores up to 2^6 in
    the exponent, sums) stay below 2^-16 of the range; then the output type."""
    span = float((v.amax() - v.amin()).item())
    t = span / 2 * 2.0 ** -11 + span * 2.0 ** -16
    half_ulp = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[out_dtype]
    return t + half_ulp * ref.abs() + (2.0 ** -25 if out_dtype == torch.float16 else 0.0)
