// kv_int4.cu — 4-bit pools: quantize + append, reading rows back, snapshots
// and restores.
//
// A row of K or V is cut into groups of G elements; per group
//   s = f16(f32(max - min) / 15), z = f16(min)
//   code = clip(rint((x - z) / s), 0, 15), every step in f32 (s = 0: code 0)
//   value = c * s + z in f32, rounded once to the type it is read in.
// Inputs beyond +-61440 saturate and NaN counts as 0, so that no stored scale
// or zero is infinite or NaN and every value is within f16's range
// (15 * f16(122880 / 15) - 61440 = 61440); restored scales and zeros are kept
// there too (sane_meta4). A masked token can then never contribute more than
// its weight of zero.
// The quotient (x - z) / s is the correctly rounded one: q = t * RN(1/s) is
// corrected by its residual, q + (t - q s) RN(1/s), one fma each (P. Markstein,
// IBM J. Res. Dev. 34(1), 1990, theorem on division with a correctly rounded
// reciprocal), which settles the ties that 16-bit inputs often hit.
#include "kv_device.cuh"

namespace krill {
namespace {

constexpr float kSat4 = 61440.0f;

template <int DT>
struct Pk;  // two packed 16-bit values of the input dtype (0 f16, 1 bf16)
template <>
struct Pk<0> {
  static __device__ __forceinline__ uint32_t mn(uint32_t a, uint32_t b) { return h2u(__hmin2(u2h(a), u2h(b))); }
  static __device__ __forceinline__ uint32_t mx_nan(uint32_t a, uint32_t b) { return h2u(__hmax2_nan(u2h(a), u2h(b))); }
  static __device__ __forceinline__ float2 f(uint32_t w) { return __half22float2(u2h(w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return f2h2(a, b); }
};
template <>
struct Pk<1> {
  static __device__ __forceinline__ __nv_bfloat162 v(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ uint32_t u(__nv_bfloat162 x) { return *reinterpret_cast<uint32_t*>(&x); }
  static __device__ __forceinline__ uint32_t mn(uint32_t a, uint32_t b) { return u(__hmin2(v(a), v(b))); }
  static __device__ __forceinline__ uint32_t mx_nan(uint32_t a, uint32_t b) { return u(__hmax2_nan(v(a), v(b))); }
  static __device__ __forceinline__ float2 f(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return u(__floats2bfloat162_rn(a, b)); }
};

__device__ __forceinline__ float sane4(float x) {
  return isnan(x) ? 0.0f : fminf(fmaxf(x, -kSat4), kSat4);
}

// Quantizes this lane's 16 elements (8 packed words); the LPG lanes of a group
// are consecutive and aligned. Element e's code is the low nibble of codes[e],
// whose other bits are those of 1.5 * 2^23 (see chunk_byte). Every lane of the
// warp calls it. The quotients stay in [0, 15] by themselves unless z or s was
// rounded far from the group's minimum and range (tiny values), which the
// group's own extremes tell; only then are they clamped.
template <int LPG, int DT>
__device__ __forceinline__ void quant16(uint32_t (&w)[8], uint32_t (&codes)[16], uint16_t& s16, uint16_t& z16) {
  using P = Pk<DT>;
  uint32_t mn2 = w[0], mx2 = w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mn2 = P::mn(mn2, w[i]);
    mx2 = P::mx_nan(mx2, w[i]);
  }
#pragma unroll
  for (int off = 1; off < LPG; off <<= 1) {
    mn2 = P::mn(mn2, __shfl_xor_sync(0xffffffffu, mn2, off));
    mx2 = P::mx_nan(mx2, __shfl_xor_sync(0xffffffffu, mx2, off));
  }
  float2 lo = P::f(mn2), hi = P::f(mx2);
  float mn = fminf(lo.x, lo.y), mx = fmaxf(hi.x, hi.y);
  // group-uniform: a NaN (kept by mx_nan in one of the halves) or a value out
  // of range
  const bool odd = !(hi.x <= kSat4 && hi.y <= kSat4 && mn >= -kSat4);
  if (__any_sync(0xffffffffu, odd)) {
    if (odd) {
      mn = kSat4;
      mx = -kSat4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float2 x = P::f(w[i]);
        x = make_float2(sane4(x.x), sane4(x.y));
        w[i] = P::pack(x.x, x.y);  // exact: values of the input type, 0 or +-61440
        mn = fminf(mn, fminf(x.x, x.y));
        mx = fmaxf(mx, fmaxf(x.x, x.y));
      }
    }
#pragma unroll
    for (int off = 1; off < LPG; off <<= 1) {
      const float a = __shfl_xor_sync(0xffffffffu, mn, off), b = __shfl_xor_sync(0xffffffffu, mx, off);
      mn = odd ? fminf(mn, a) : mn;
      mx = odd ? fmaxf(mx, b) : mx;
    }
  }
  const __half hs = __float2half_rn(__fdiv_rn(mx - mn, 15.0f)), hz = __float2half_rn(mn);
  const float s = __half2float(hs), z = __half2float(hz);
  const float r = s > 0.0f ? __frcp_rn(s) : 0.0f;
  const float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to nearest even
  const F2 s2 = f2(-s, -s), r2 = f2(r, r), z2 = f2(-z, -z), round2 = f2(kRound, kRound);
  auto quotient = [&](float a, float b) {
    const F2 t = f2_add(f2(a, b), z2);
    const F2 q = f2_mul(t, r2);
    return f2_fma(f2_fma(q, s2, t), r2, q);
  };
  const F2 ends = quotient(mn, mx);
  const bool inside = f2_lo(ends) > -0.5f && f2_hi(ends) < 15.5f;
  if (__all_sync(0xffffffffu, inside)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = P::f(w[i]);
      const F2 k = f2_add(quotient(x.x, x.y), round2);
      codes[2 * i] = __float_as_uint(f2_lo(k));
      codes[2 * i + 1] = __float_as_uint(f2_hi(k));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = P::f(w[i]);
      const F2 q = quotient(x.x, x.y);
      codes[2 * i] = __float_as_uint(fminf(fmaxf(f2_lo(q), 0.0f), 15.0f) + kRound);
      codes[2 * i + 1] = __float_as_uint(fminf(fmaxf(f2_hi(q), 0.0f), 15.0f) + kRound);
    }
  }
  s16 = __half_as_ushort(hs);
  z16 = __half_as_ushort(hz);
}

// Byte j of this lane's chunk (see q4_kbyte / q4_vbyte), from codes whose bits
// 4 to 7 are zero.
__device__ __forceinline__ uint8_t chunk_byte(const uint32_t (&codes)[16], bool is_k, int j) {
  return is_k ? (uint8_t)(codes[q4_elem(true, j)] + 16u * codes[q4_elem(true, j) + q4_step(true)])
              : (uint8_t)(codes[q4_elem(false, j)] + 16u * codes[q4_elem(false, j) + q4_step(false)]);
}

__device__ __forceinline__ void load16(const void* src, int64_t elem, uint32_t (&w)[8]) {
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + elem);
  const uint4 a = __ldg(p), b = __ldg(p + 1);
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
}

// Rotate-half RoPE of a lane's 16 elements of K (chunk c of D/16): element d <
// D/2 pairs with d + D/2, held D/32 lanes away. Unfused f32 products and sum,
// rounded to the input dtype, as on the int8 path. Every lane of the warp
// calls it; lanes with live = false keep their words.
template <int D, int DT>
__device__ __forceinline__ void rope16(uint32_t (&w)[8], int c, int64_t pos, const RopeTable& rope, bool live) {
  using P = Pk<DT>;
  constexpr int LPT = D / 16, H = D / 2;
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __shfl_xor_sync(0xffffffffu, w[i], LPT / 2);
  if (!live) return;
  const bool upper = c >= LPT / 2;
  const float* cr = rope.cos + pos * H + 16 * (c % (LPT / 2));
  const float* sr = rope.sin + pos * H + 16 * (c % (LPT / 2));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = P::f(w[i]), y = P::f(o[i]);
    const float c0 = __ldg(cr + 2 * i), c1 = __ldg(cr + 2 * i + 1);
    const float s0 = __ldg(sr + 2 * i), s1 = __ldg(sr + 2 * i + 1);
    const float a = upper ? __fadd_rn(__fmul_rn(y.x, s0), __fmul_rn(x.x, c0))
                          : __fsub_rn(__fmul_rn(x.x, c0), __fmul_rn(y.x, s0));
    const float b = upper ? __fadd_rn(__fmul_rn(y.y, s1), __fmul_rn(x.y, c1))
                          : __fsub_rn(__fmul_rn(x.y, c1), __fmul_rn(y.y, s1));
    w[i] = P::pack(a, b);
  }
}

// Appends of a few tokens (decode steps): one lane per 16 elements of a row,
// D/16 lanes a row, K and V rows of a token side by side. Each lane's 8 code
// bytes go straight to the pool (a byte belongs to one token). Launch latency
// bounds it: 4.1 us for one token of 4 sequences, 16 layers, 8 heads of 64.
template <int D, int G, int DT>
__global__ void __launch_bounds__(256) append4_kernel(uint8_t* __restrict__ pool, Geom geom,
                                                      const AppendDst* __restrict__ dst,
                                                      const __grid_constant__ InlinePacket inl, int layer_begin,
                                                      int layer_count, int n_seqs, int n_new,
                                                      const void* __restrict__ k, const void* __restrict__ v,
                                                      int* __restrict__ large_scale, RopeTable rope) {
  asm volatile("griddepcontrol.launch_dependents;");  // as in append_quantize_kernel
  constexpr int LPT = D / 16, LPG = G / 16, NG = D / G;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int c = (int)(idx % LPT);
  const bool is_k = (idx / LPT) % 2 == 0;
  const int64_t row = idx / (2 * LPT);
  const int64_t total = (int64_t)layer_count * n_seqs * geom.Hkv * n_new;
  const bool live = row < total;
  uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
  AppendDst d{0, 0};
  int h = 0, li = 0;
  if (live) {
    const int64_t rest = row / n_new;
    h = (int)(rest % geom.Hkv);
    const int64_t ls = rest / geom.Hkv;
    li = (int)(ls / n_seqs);
    const int64_t i = ls * n_new + row % n_new;
    if (dst) {
      d = dst[i];
    } else {
      d.block = (int32_t)inl.w[2 * i];
      d.pos = (int32_t)inl.w[2 * i + 1];
    }
    load16(is_k ? k : v, row * D + 16 * c, w);
  }
  if (rope.cos) rope16<D, DT>(w, c, d.pos, rope, live && is_k);
  uint32_t codes[16];
  uint16_t s16, z16;
  quant16<LPG, DT>(w, codes, s16, z16);
  if (!live) return;
  const int slot = d.pos & (kBlockTokens - 1), t = slot % kSub4;
  uint8_t* sb = pool + (((int64_t)d.block * geom.L + (layer_begin + li)) * geom.Hkv + h) * geom.page_bytes +
                (int64_t)(slot / kSub4) * geom.sb_bytes;
#pragma unroll
  for (int j = 0; j < 8; ++j) sb[is_k ? q4_kbyte(D, t, c, j) : q4_vbyte(D, NG, t, c, j)] = chunk_byte(codes, is_k, j);
  if (c % LPG == 0) {
    const int gi = c / LPG, a = is_k ? 0 : 2;
    *reinterpret_cast<uint16_t*>(sb + q4_meta(D, NG, a, gi, t)) = s16;
    *reinterpret_cast<uint16_t*>(sb + q4_meta(D, NG, a + 1, gi, t)) = z16;
    if (s16 >= 0x5400u) atomicOr(large_scale, 1);
  }
}

// One thread's rows of a sub-block's K or V: chunk c of the tokens t0, t0 +
// 4096 / D, ... (PER of them), those outside [t_lo, t_hi) as zeros.
template <int D, int PER>
__device__ __forceinline__ void tile_fetch(const void* src, int64_t row0, int c, int t0, int t_lo, int t_hi,
                                           uint32_t (&w)[PER][8]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = t0 + i * (4096 / D);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = 0u;
    if (t >= t_lo && t < t_hi) load16(src, (row0 + t) * D + 16 * c, w[i]);
  }
}
// Quantizes them into the sub-block at `to` (shared or global); true when a
// scale is 64 or more.
template <int D, int G, int DT, int PER, bool K>
__device__ __forceinline__ bool tile_quantize(uint32_t (&w)[PER][8], int64_t cs, int c, int t0, int t_lo, int t_hi,
                                              const RopeTable& rope, uint8_t* to) {
  constexpr int LPG = G / 16, NG = D / G, a = K ? 0 : 2;
  bool large = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = t0 + i * (4096 / D);
    const bool live = t >= t_lo && t < t_hi;
    if (K && rope.cos) rope16<D, DT>(w[i], c, cs + t, rope, live);
    uint32_t codes[16];
    uint16_t s16, z16;
    quant16<LPG, DT>(w[i], codes, s16, z16);
    if (!live) continue;
    uint8_t* at = to + (K ? q4_kbyte(D, t, c, 0) : q4_vbyte(D, NG, t, c, 0));
#pragma unroll
    for (int j = 0; j < 8; ++j) at[K ? (j >> 1) * 4 + (j & 1) * 2 : j * 64] = chunk_byte(codes, K, j);
    if (c % LPG == 0) {
      const int gi = c / LPG;
      *reinterpret_cast<uint16_t*>(to + q4_meta(D, NG, a, gi, t)) = s16;
      *reinterpret_cast<uint16_t*>(to + q4_meta(D, NG, a + 1, gi, t)) = z16;
      large |= s16 >= 0x5400u;
    }
  }
  return large;
}

// Appends of many tokens (prompts): one CTA per (layer, sequence, kv head,
// touched sub-block). A sub-block that the call covers whole is built in shared
// memory and leaves with 16-byte stores; one that it covers in part gets byte
// stores (on a windowed pool the call's first and last chunk can be parts of
// one sub-block, so neither may write the other's bytes). 49 us for 2 x 2039
// tokens, 8 layers, 8 heads of 128, whose 171 MB take 26 us at copy bandwidth.
// It runs 15.6 instructions a code, the quotients about five of them; the rest
// unpacks words, finds extremes, packs and stores single bytes. Issue slots are
// 62 % busy, the L1 72 %, and warps wait for loads first of all.
template <int D, int G, int DT>
__global__ void __launch_bounds__(256) append4_tile_kernel(uint8_t* __restrict__ pool, Geom geom,
                                                           const AppendDst* __restrict__ dst, int layer_begin,
                                                           int n_seqs, int n_new, int n_chunks,
                                                           const void* __restrict__ k,
                                                           const void* __restrict__ v,
                                                           int* __restrict__ large_scale, RopeTable rope) {
  asm volatile("griddepcontrol.launch_dependents;");  // as in append_quantize_kernel
  constexpr int LPT = D / 16, NG = D / G, T = kSub4;
  constexpr int SB = T * (D + 8 * NG);
  __shared__ __align__(16) uint8_t img[SB];
  uint32_t b = blockIdx.x;
  const int ch = (int)(b % (uint32_t)n_chunks);
  b /= (uint32_t)n_chunks;
  const int h = (int)(b % (uint32_t)geom.Hkv);
  const int64_t ls = b / (uint32_t)geom.Hkv;  // li * n_seqs + si
  const int64_t p0 = dst[ls * n_chunks].pos;
  const int64_t cs = p0 - p0 % T + (int64_t)ch * T;  // first position of the sub-block
  const int t_lo = (int)max((int64_t)0, p0 - cs), t_hi = (int)min((int64_t)T, p0 + n_new - cs);
  if (t_lo >= t_hi) return;
  const AppendDst d0 = dst[ls * n_chunks + ch];
  const int slot0 = d0.pos & (kBlockTokens - 1);
  uint8_t* sb = pool +
                (((int64_t)d0.block * geom.L + (layer_begin + (int)(ls / n_seqs))) * geom.Hkv + h) * geom.page_bytes +
                (int64_t)(slot0 / T) * geom.sb_bytes;
  const int64_t row0 = (ls * geom.Hkv + h) * n_new + (cs - p0);  // input row of token t: row0 + t
  const bool whole = t_lo == 0 && t_hi == T;
  bool large = false;
  // all of K's loads, then V's while K is quantized
  constexpr int PER = T * LPT / 256;  // rounds of K (and of V) items
  uint32_t wk[PER][8], wv[PER][8];
  const int c = threadIdx.x % LPT, t0 = threadIdx.x / LPT;
  tile_fetch<D, PER>(k, row0, c, t0, t_lo, t_hi, wk);
  tile_fetch<D, PER>(v, row0, c, t0, t_lo, t_hi, wv);
  uint8_t* to = whole ? img : sb;
  large |= tile_quantize<D, G, DT, PER, true>(wk, cs, c, t0, t_lo, t_hi, rope, to);
  large |= tile_quantize<D, G, DT, PER, false>(wv, cs, c, t0, t_lo, t_hi, rope, to);
  if (large) atomicOr(large_scale, 1);
  if (!whole) return;
  __syncthreads();
  for (int i = threadIdx.x; i < SB / 16; i += 256)
    reinterpret_cast<uint4*>(sb)[i] = reinterpret_cast<const uint4*>(img)[i];
}

// The 16 codes of chunk c of token t of a 4-bit sub-block.
__device__ __forceinline__ void unpack_chunk(const uint8_t* sb, int D, int NG, int t, int c, bool is_k,
                                             uint8_t (&codes)[16]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint8_t x = sb[is_k ? q4_kbyte(D, t, c, j) : q4_vbyte(D, NG, t, c, j)];
    if (is_k) {
      codes[q4_elem(true, j)] = x & 15;
      codes[q4_elem(true, j) + q4_step(true)] = x >> 4;
    } else {
      codes[q4_elem(false, j)] = x & 15;
      codes[q4_elem(false, j) + q4_step(false)] = x >> 4;
    }
  }
}

// Stores 16 f32 values as 16-byte words of the output type.
__device__ __forceinline__ void store16(void* out, int dtype, int64_t elem, const float (&v)[16]) {
  if (dtype == KRILL_DTYPE_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + elem);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = dtype == KRILL_DTYPE_F16 ? Pk<0>::pack(v[2 * i], v[2 * i + 1]) : Pk<1>::pack(v[2 * i], v[2 * i + 1]);
  uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + elem);
  p[0] = make_uint4(w[0], w[1], w[2], w[3]);
  p[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// Where the rows [starts[si], + n) of a read lie: sub-block ch of those that
// row range touches in (layer, sequence, kv head) of CTA b; false: none.
struct ReadAt {
  const uint8_t* sb;
  int64_t row0;  // output row of the sub-block's token 0
  int t_lo, t_hi;
};
__device__ __forceinline__ bool read_at(const uint8_t* pool, const Geom& geom, const uint32_t* meta,
                                        const InlinePacket& inl, int bt_stride, int layer_begin, int n_seqs, int64_t n,
                                        int n_chunks, uint32_t b, ReadAt& at) {
  auto word = [&](int64_t i) { return meta ? meta[i] : inl.w[i]; };
  const int T = geom.subt;
  const int ch = (int)(b % (uint32_t)n_chunks);
  b /= (uint32_t)n_chunks;
  const int h = (int)(b % (uint32_t)geom.Hkv);
  const int64_t ls = b / (uint32_t)geom.Hkv;
  const int si = (int)(ls % n_seqs), layer = layer_begin + (int)(ls / n_seqs);
  const int64_t p0 = (int64_t)((uint64_t)word(2 * si + 1) << 32 | word(2 * si));
  const int64_t cs = p0 - p0 % T + (int64_t)ch * T;
  at.t_lo = (int)max((int64_t)0, p0 - cs);
  at.t_hi = (int)min((int64_t)T, p0 + n - cs);
  if (at.t_lo >= at.t_hi) return false;
  int64_t bi = cs / kBlockTokens;
  if (geom.ring > 0) bi %= geom.ring;
  const int32_t block = (int32_t)word((n_seqs + 1) / 2 * 4 + (int64_t)si * bt_stride + bi);
  at.sb = pool + (((int64_t)block * geom.L + layer) * geom.Hkv + h) * geom.page_bytes +
          (cs % kBlockTokens) / T * geom.sb_bytes;
  at.row0 = (ls * geom.Hkv + h) * n + (cs - p0);
  return true;
}

// Rows of a 4-bit pool, dequantized, in the layout that an append takes:
// [layers][seqs][Hkv][n][D]. One CTA per (layer, sequence, kv head, touched
// sub-block). A thread takes four consecutive tokens (one tile row pair's) of
// 16 elements: of K two 16-byte words, of V eight 4-byte words of the image in
// shared memory, whose V codes are spread by 16 bytes per 512 against bank
// conflicts. Its eight (K) lanes along D write 256 consecutive bytes a row.
// 41 us for the rows of the append above (the same bytes, 26 us), 4.9 us for
// the one-token one.
template <int D, int G>
__global__ void __launch_bounds__(256) read_rows4_kernel(const uint8_t* __restrict__ pool, Geom geom,
                                                         const uint32_t* __restrict__ meta,
                                                         const __grid_constant__ InlinePacket inl, int bt_stride,
                                                         int layer_begin, int n_seqs, int64_t n, int n_chunks, void* keys,
                                                         void* values, int dtype) {
  constexpr int LPT = D / 16, NG = D / G, HALF = q4_half(D, NG), CODES = 32 * D;
  __shared__ __align__(16) uint8_t img[2 * HALF + CODES / 32];
  ReadAt at;
  if (!read_at(pool, geom, meta, inl, bt_stride, layer_begin, n_seqs, n, n_chunks, blockIdx.x, at)) return;
  // image: K half, V scales and zeros, V codes (spread)
  constexpr int VMETA = HALF, VCODES = HALF + 256 * NG;
  for (int i = threadIdx.x; i < 2 * HALF / 16; i += 256) {
    const int off = 16 * i;
    int to = off;
    if (off >= HALF + CODES) to = VMETA + off - HALF - CODES;
    else if (off >= HALF) to = VCODES + (off - HALF) + ((off - HALF) >> 9) * 16;
    *reinterpret_cast<uint4*>(img + to) = __ldg(reinterpret_cast<const uint4*>(at.sb) + i);
  }
  __syncthreads();
  // 16 items of four tokens: tile u, rows 2 tig and 2 tig + 1 (both halves)
  for (int i = threadIdx.x; i < 2 * 16 * LPT; i += 256) {
    const bool is_k = i < 16 * LPT;
    const int c = i % LPT, u = i / LPT % 4, tig = i / (4 * LPT) % 4, gi = 16 * c / G;
    const int t = 16 * tig + 4 * u;  // tokens t + 2 hi + h
    if (t + 4 <= at.t_lo || t >= at.t_hi) continue;
    void* out = is_k ? keys : values;
    if (!out) continue;
    const uint8_t* meta = is_k ? img + CODES : img + VMETA;
    float s[2][2], z[2][2];  // [h][hi]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 ss = __half22float2(u2h(*reinterpret_cast<const uint32_t*>(meta + gi * 128 + (2 * tig + h) * 16 + 4 * u)));
      const float2 zz =
          __half22float2(u2h(*reinterpret_cast<const uint32_t*>(meta + (NG + gi) * 128 + (2 * tig + h) * 16 + 4 * u)));
      s[h][0] = ss.x; s[h][1] = ss.y;
      z[h][0] = zz.x; z[h][1] = zz.y;
    }
    // code words: of V word j holds the codes of elements j, j + 8 of the four
    // tokens; of K the words of row h hold those of its two tokens
    uint32_t w[2][4];
    if (is_k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(img + ((u * (D / 64) + (c >> 2)) * 32 + (2 * tig + h) * 4 + (c & 3)) * 16);
        w[h][0] = x.x; w[h][1] = x.y; w[h][2] = x.z; w[h][3] = x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        w[j >> 2][j & 3] = *reinterpret_cast<const uint32_t*>(img + VCODES + c * 528 + (j * 4 + tig) * 16 + 4 * u);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int tok = t + 2 * hi + h;
        if (tok < at.t_lo || tok >= at.t_hi) continue;
        float x[16];
        if (is_k) {  // row h: word k, halves d = 4k, 4k + 1 (low nibbles), + 2, + 3 (high)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int nib = 0; nib < 2; ++nib) {
              const uint32_t v = ((w[h][k] >> (8 * hi + 4 * nib)) & 0x000f000fu) | 0x64006400u;
              const float2 f = __half22float2(__hsub2_rn(u2h(v), u2h(0x64006400u)));
              x[4 * k + 2 * nib] = f.x;
              x[4 * k + 2 * nib + 1] = f.y;
            }
        } else {  // half h of word j: byte hi, element j (low nibble) and j + 8
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t b = w[j >> 2][j & 3] >> (16 * h + 8 * hi);
            const uint32_t v = (b & 0xfu) | ((b & 0xf0u) << 12) | 0x64006400u;
            const float2 f = __half22float2(__hsub2_rn(u2h(v), u2h(0x64006400u)));
            x[j] = f.x;
            x[j + 8] = f.y;
          }
        }
        const F2 s2 = f2(s[h][hi], s[h][hi]), z2 = f2(z[h][hi], z[h][hi]);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const F2 y = f2_fma(f2(x[e], x[e + 1]), s2, z2);
          x[e] = f2_lo(y);
          x[e + 1] = f2_hi(y);
        }
        store16(out, dtype, (at.row0 + tok) * D + 16 * c, x);
      }
  }
}

// The same of an int8 pool.
__global__ void __launch_bounds__(256) read_rows8_kernel(const uint8_t* __restrict__ pool, Geom geom,
                                                         const uint32_t* __restrict__ meta,
                                                         const __grid_constant__ InlinePacket inl, int bt_stride,
                                                         int layer_begin, int n_seqs, int64_t n, int n_chunks, void* keys,
                                                         void* values, int dtype) {
  extern __shared__ __align__(16) uint8_t img8[];
  const int D = geom.D, NG = geom.NG, LPT = D / 16;
  ReadAt at;
  if (!read_at(pool, geom, meta, inl, bt_stride, layer_begin, n_seqs, n, n_chunks, blockIdx.x, at)) return;
  for (int i = threadIdx.x; i < (int)(geom.sb_bytes / 16); i += 256)
    reinterpret_cast<uint4*>(img8)[i] = reinterpret_cast<const uint4*>(at.sb)[i];
  __syncthreads();
  const int span = (at.t_hi - at.t_lo) * LPT;
  for (int i = threadIdx.x; i < 2 * span; i += 256) {
    const bool is_k = i < span;
    const int j = is_k ? i : i - span;
    const int c = j % LPT, t = at.t_lo + j / LPT, gi = 16 * c / geom.G, a = is_k ? 0 : 2;
    void* out = is_k ? keys : values;
    if (!out) continue;
    const __half s = *reinterpret_cast<const __half*>(img8 + sb_meta(D, NG, a, gi, t));
    const __half z = *reinterpret_cast<const __half*>(img8 + sb_meta(D, NG, a + 1, gi, t));
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint8_t code = img8[is_k ? sb_kcode(D, t, 16 * c + e) : sb_vcode(D, t, 16 * c + e)];
      x[e] = __half2float(__hadd_rn(__hmul_rn(__ushort2half_rn(code), s), z));
    }
    store16(out, dtype, (at.row0 + t) * D + 16 * c, x);
  }
}

// Snapshot rows [p0, p0 + S) of one (sequence, layer), one thread per 16
// elements of a row: unpacked codes + meta (mode 0) or f16 values (mode 1).
__global__ void gather4_kernel(const uint8_t* __restrict__ pool, Geom geom, int layer,
                               const int32_t* __restrict__ bt, int64_t p0, int64_t S, GatherOut out) {
  const int D = geom.D, NG = geom.NG, LPT = D / 16;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= (int64_t)geom.Hkv * S * LPT * 2) return;
  const bool is_k = idx % 2 == 0;
  const int c = (int)(idx / 2 % LPT);
  const int64_t hr = idx / 2 / LPT, i = hr % S, pos = p0 + i;
  const int h = (int)(hr / S);
  int64_t bidx = pos / kBlockTokens;
  if (geom.ring > 0) bidx %= geom.ring;
  const int slot = (int)(pos % kBlockTokens), t = slot % kSub4, gi = 16 * c / geom.G, a = is_k ? 0 : 2;
  const uint8_t* sb = pool + (((int64_t)bt[bidx] * geom.L + layer) * geom.Hkv + h) * geom.page_bytes +
                      (int64_t)(slot / kSub4) * geom.sb_bytes;
  const int64_t orow = (int64_t)h * out.rows_total + out.row_off + i;
  uint8_t* dst = is_k ? out.keys : out.values;
  const uint16_t s16 = *reinterpret_cast<const uint16_t*>(sb + q4_meta(D, NG, a, gi, t));
  const uint16_t z16 = *reinterpret_cast<const uint16_t*>(sb + q4_meta(D, NG, a + 1, gi, t));
  if (dst) {
    uint8_t codes[16];
    unpack_chunk(sb, D, NG, t, c, is_k, codes);
    if (out.mode == 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) dst[orow * D + 16 * c + e] = codes[e];
    } else {
      const float s = __half2float(__ushort_as_half(s16)), z = __half2float(__ushort_as_half(z16));
#pragma unroll
      for (int e = 0; e < 16; ++e)
        reinterpret_cast<__half*>(dst)[orow * D + 16 * c + e] = __float2half_rn(fmaf((float)codes[e], s, z));
    }
  }
  if (out.mode == 0 && (16 * c) % geom.G == 0) {
    uint16_t* so = is_k ? out.key_scales : out.value_scales;
    uint16_t* zo = is_k ? out.key_zeros : out.value_zeros;
    if (so) so[orow * NG + gi] = s16;
    if (zo) zo[orow * NG + gi] = z16;
  }
}

// A restored group's scale and zero, which may be any f16: the zero is kept
// within +-61440 and the scale where all sixteen values are finite in f16, NaN
// as 0. What an append stores passes unchanged (its values end below 61440 + 16
// + 15 * 2, the roundings of z and s).
__device__ __forceinline__ void sane_meta4(uint16_t& s16, uint16_t& z16) {
  float z = __half2float(__ushort_as_half(z16));
  if (!(fabsf(z) <= kSat4)) {
    z = sane4(z);
    z16 = __half_as_ushort(__float2half_rn(z));
  }
  const float s = __half2float(__ushort_as_half(s16));
  const float hi = __fdiv_rz(65504.0f - z, 15.0f), lo = __fdiv_rz(-65504.0f - z, 15.0f);
  if (!(s >= lo && s <= hi)) s16 = isnan(s) ? 0 : __half_as_ushort(__float2half_rz(s > hi ? hi : lo));
}

// Snapshot layout -> pages (restore, scatter-back); codes are taken modulo 16.
__global__ void scatter4_kernel(uint8_t* __restrict__ pool, Geom geom, int layer, const int32_t* __restrict__ bt,
                                int64_t p0, int64_t S, ScatterIn in, int* __restrict__ large_scale) {
  const int D = geom.D, NG = geom.NG, LPT = D / 16;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= (int64_t)geom.Hkv * S * LPT * 2) return;
  const bool is_k = idx % 2 == 0;
  const int c = (int)(idx / 2 % LPT);
  const int64_t hr = idx / 2 / LPT, i = hr % S, pos = p0 + i;
  const int h = (int)(hr / S);
  int64_t bidx = pos / kBlockTokens;
  if (geom.ring > 0) bidx %= geom.ring;
  const int slot = (int)(pos % kBlockTokens), t = slot % kSub4, gi = 16 * c / geom.G, a = is_k ? 0 : 2;
  uint8_t* sb = pool + (((int64_t)bt[bidx] * geom.L + layer) * geom.Hkv + h) * geom.page_bytes +
                (int64_t)(slot / kSub4) * geom.sb_bytes;
  const int64_t irow = (int64_t)h * in.rows_total + in.row_off + i;
  const uint8_t* src = (is_k ? in.keys : in.values) + irow * D + 16 * c;
  uint32_t codes[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) codes[e] = src[e] & 15u;
#pragma unroll
  for (int j = 0; j < 8; ++j) sb[is_k ? q4_kbyte(D, t, c, j) : q4_vbyte(D, NG, t, c, j)] = chunk_byte(codes, is_k, j);
  if ((16 * c) % geom.G == 0) {
    uint16_t s16 = (is_k ? in.key_scales : in.value_scales)[irow * NG + gi];
    uint16_t z16 = (is_k ? in.key_zeros : in.value_zeros)[irow * NG + gi];
    sane_meta4(s16, z16);
    *reinterpret_cast<uint16_t*>(sb + q4_meta(D, NG, a, gi, t)) = s16;
    *reinterpret_cast<uint16_t*>(sb + q4_meta(D, NG, a + 1, gi, t)) = z16;
    if ((s16 & 0x7fffu) >= 0x5400u) atomicOr(large_scale, 1);
  }
}

template <int D, int G, int DT>
cudaError_t append4(const Geom& g, uint8_t* pool, const AppendDst* d_dst, const InlinePacket& inl, int layer_begin,
                    int layer_count, int n_seqs, int n_new, const void* k, const void* v, int* large_scale, RopeTable rope,
                    cudaStream_t stream) {
  if (append_uses_tiles(n_new)) {
    const int n_chunks = append_tile_chunks(n_new, g.subt);
    const int64_t tiles = (int64_t)layer_count * n_seqs * g.Hkv * n_chunks;
    if (tiles > INT32_MAX) return cudaErrorInvalidValue;
    append4_tile_kernel<D, G, DT><<<(unsigned)tiles, 256, 0, stream>>>(pool, g, d_dst, layer_begin, n_seqs, n_new,
                                                                       n_chunks, k, v, large_scale, rope);
    return cudaGetLastError();
  }
  const int64_t threads = (int64_t)layer_count * n_seqs * g.Hkv * n_new * (D / 8);
  append4_kernel<D, G, DT><<<(unsigned)((threads + 255) / 256), 256, 0, stream>>>(
      pool, g, d_dst, inl, layer_begin, layer_count, n_seqs, n_new, k, v, large_scale, rope);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append4(const Geom& g, uint8_t* pool, const AppendDst* d_dst, const void* h, int layer_begin,
                           int layer_count, int n_seqs, int n_new, const void* k, const void* v, int dtype,
                           int* large_scale, RopeTable rope, cudaStream_t stream) {
  static const InlinePacket none{};
  const InlinePacket& inl = d_dst ? none : *static_cast<const InlinePacket*>(h);
#define KRILL_APPEND4(DD, GG)                                                                               \
  if (g.D == DD && g.G == GG)                                                                               \
    return dtype == 0 ? append4<DD, GG, 0>(g, pool, d_dst, inl, layer_begin, layer_count, n_seqs, n_new, k, v, \
                                           large_scale, rope, stream)                                       \
                      : append4<DD, GG, 1>(g, pool, d_dst, inl, layer_begin, layer_count, n_seqs, n_new, k, v, \
                                           large_scale, rope, stream);
  KRILL_APPEND4(64, 64)
  KRILL_APPEND4(128, 64)
  KRILL_APPEND4(128, 128)
  KRILL_APPEND4(256, 64)
  KRILL_APPEND4(256, 256)
#undef KRILL_APPEND4
  return cudaErrorInvalidValue;
}

cudaError_t launch_gather4(const Geom& g, const uint8_t* pool, int layer, const int32_t* d_bt, int64_t p0,
                           int64_t S, const GatherOut& out, cudaStream_t stream) {
  const int64_t total = (int64_t)g.Hkv * S * (g.D / 8);
  gather4_kernel<<<(unsigned)((total + 255) / 256), 256, 0, stream>>>(pool, g, layer, d_bt, p0, S, out);
  return cudaGetLastError();
}

cudaError_t launch_scatter4(const Geom& g, uint8_t* pool, int layer, const int32_t* d_bt, int64_t p0, int64_t S,
                            const ScatterIn& in, int* large_scale, cudaStream_t stream) {
  const int64_t total = (int64_t)g.Hkv * S * (g.D / 8);
  scatter4_kernel<<<(unsigned)((total + 255) / 256), 256, 0, stream>>>(pool, g, layer, d_bt, p0, S, in, large_scale);
  return cudaGetLastError();
}

cudaError_t launch_read_rows(const Geom& g, const uint8_t* pool, const void* meta, const void* h, int bt_stride,
                             int layer_begin, int layer_count, int n_seqs, int64_t n, void* keys, void* values,
                             int dtype, cudaStream_t stream) {
  static const InlinePacket none{};
  const InlinePacket& inl = meta ? none : *static_cast<const InlinePacket*>(h);
  const uint32_t* words = static_cast<const uint32_t*>(meta);
  const int64_t n_chunks = (n + g.subt - 1) / g.subt + 1;
  const int64_t blocks = (int64_t)layer_count * n_seqs * g.Hkv * n_chunks;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
#define KRILL_READ4(DD, GG)                                                                                \
  if (g.fmt == kFmtInt4 && g.D == DD && g.G == GG)                                                         \
    read_rows4_kernel<DD, GG><<<(unsigned)blocks, 256, 0, stream>>>(pool, g, words, inl, bt_stride,        \
                                                                    layer_begin, n_seqs, n, (int)n_chunks, \
                                                                    keys, values, dtype);
  KRILL_READ4(64, 64)
  KRILL_READ4(128, 64)
  KRILL_READ4(128, 128)
  KRILL_READ4(256, 64)
  KRILL_READ4(256, 256)
#undef KRILL_READ4
  if (g.fmt != kFmtInt4)
    read_rows8_kernel<<<(unsigned)blocks, 256, (size_t)g.sb_bytes, stream>>>(
        pool, g, words, inl, bt_stride, layer_begin, n_seqs, n, (int)n_chunks, keys, values, dtype);
  return cudaGetLastError();
}

}  // namespace krill
