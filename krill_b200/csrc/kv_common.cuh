// kv_common.cuh — page geometry and device helpers shared by the kernels.
//
// HBM layout of one pool (one layer group on one GPU):
//   pool = blocks[num_blocks]; block = pages[num_layers][num_kv_heads];
//   page = 256 tokens = sub-blocks of T tokens (T = 64, or 32 for D = 256 so
//   that every sub-block is about 17 KB); each sub-block is one contiguous run
//   of SB = T * (2*D + 8*NG) bytes:
//     [0, T*D)             K codes, token-major rows of D bytes; for D >= 128
//                          the 16-byte chunks of odd rows are XOR-swizzled by 4
//                          so the decode kernel's shared-memory reads are
//                          bank-conflict free
//     [T*D, 2*T*D)         V codes transposed: D rows of T token bytes, so the
//                          tensor-core fragments along the token axis are
//                          contiguous bytes
//     [2*T*D, ...)         K scales, K zeros, V scales, V zeros: [NG][T] f16 each
// A sub-block is the unit one bulk (TMA) copy moves into shared memory.
//
// Raw bf16 pools (the unquantized comparison format) use the same blocks and
// pages with sub-blocks of T = 32 tokens (64 at D = 64) of T * 4 * D bytes:
//     [0, 2*T*D)           K rows, token-major bf16; the 16-byte chunks of odd
//                          rows swapped pairwise (chunk ^ 1) so the decode
//                          kernel's shared-memory reads are conflict free
//     [2*T*D, 4*T*D)       V transposed: D rows of T bf16
//
// 4-bit pools use sub-blocks of T = 64 tokens of T * (D + 8*NG) bytes, a K
// half and a V half of 32*D + 256*NG bytes each (one bulk copy each):
// Token t of a sub-block is row r (hi = 0) or r + 8 (hi = 1) of the 16-token
// tile u, with t = 16 (r / 2) + 4 u + 2 hi + r % 2: a lane of the V operand then
// holds 16 consecutive tokens over the four tiles.
//     K half, [0, 32*D)    K codes in the order of the decode kernel's MMA
//                          operand: 16-token x 16-element tiles of 32 lane
//                          words, the four tiles of 64 elements interleaved so
//                          that one 16-byte load per lane fetches them. Byte
//                          (2h + hi) of word k holds the codes d (low nibble)
//                          and d + 2 (high) of one token, d = 16c + 4k + h
//             [32*D, ...)  K scales, K zeros: [NG][T] f16, token at 8 r + 2 u +
//                          hi, so that the eight tokens of one operand row are
//                          16 consecutive bytes
//     V half, [0, 32*D)    V codes, tiles of 16 elements x 16 tokens, the four
//                          token tiles interleaved; a byte holds the codes d
//                          and d + 8 of one token
//             [32*D, ...)  V scales, V zeros, as for K
// Every code byte belongs to one token, so tokens are written independently.
//
// A pool with block summaries ends each page with spb rows of 2*D bytes (per
// K channel of the sub-block: mid, then half-range, as int8 in units of
// sigma) followed by spb f32 sigmas, padded to 16 bytes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace krill {

constexpr int kBlockTokens = 256;
// Tokens per sub-block for head dim D.
__host__ __device__ constexpr int sub_tokens(int D) { return D >= 256 ? 32 : 64; }
// Tokens per sub-block of a raw bf16 pool.
__host__ __device__ constexpr int sub_tokens_raw(int D) { return D >= 128 ? 32 : 64; }
// Pool formats.
constexpr int kFmtInt8 = 0;
constexpr int kFmtBf16 = 1;
constexpr int kFmtInt4 = 2;
// Tokens per sub-block of a 4-bit pool.
constexpr int kSub4 = 64;

struct Geom {
  int L;        // layers in the pool
  int Hkv;      // kv heads
  int Hq;       // query heads
  int g;        // Hq / Hkv
  int D;        // head dim
  int G;        // group size
  int NG;       // D / G
  int ring;     // blocks in a windowed sequence's ring; 0 = full history
  int window;   // sliding window (tokens); 0 = full history
  int quant_variant;
  int fmt;      // kFmtInt8, kFmtBf16 or kFmtInt4
  int subt;     // tokens per sub-block
  int spb;      // sub-blocks per 256-token block
  int64_t sb_bytes;
  int64_t sum_off;  // byte offset of a page's block summaries; 0 = none
  int64_t page_bytes;
  int64_t block_bytes;
};

// Bytes of a page's block summaries (spb sub-blocks).
__host__ __device__ inline int64_t summary_bytes(int D, int spb) {
  return ((int64_t)spb * (2 * D + 4) + 15) / 16 * 16;
}

inline Geom make_geom(int L, int Hkv, int Hq, int D, int G, int ring, int window, int qv,
                      int fmt = kFmtInt8, bool summaries = false) {
  Geom g;
  g.L = L; g.Hkv = Hkv; g.Hq = Hq; g.g = Hq / Hkv; g.D = D; g.G = G; g.NG = D / G;
  g.ring = ring; g.window = window; g.quant_variant = qv; g.fmt = fmt;
  g.subt = fmt == kFmtBf16 ? sub_tokens_raw(D) : fmt == kFmtInt4 ? kSub4 : sub_tokens(D);
  g.spb = kBlockTokens / g.subt;
  g.sb_bytes = fmt == kFmtBf16   ? (int64_t)g.subt * 4 * D
               : fmt == kFmtInt4 ? (int64_t)g.subt * (D + 8 * g.NG)
                                 : (int64_t)g.subt * (2 * D + 8 * g.NG);
  g.page_bytes = g.sb_bytes * g.spb;
  g.sum_off = summaries ? g.page_bytes : 0;
  if (summaries) g.page_bytes += summary_bytes(D, g.spb);
  g.block_bytes = g.page_bytes * L * Hkv;
  return g;
}

// Byte offsets inside a sub-block.
__host__ __device__ inline int64_t sb_voff(int D) { return (int64_t)sub_tokens(D) * D; }
__host__ __device__ inline int64_t sb_meta_off(int D) { return (int64_t)2 * sub_tokens(D) * D; }
// meta array a (0 = K scale, 1 = K zero, 2 = V scale, 3 = V zero), group gi, token t
__host__ __device__ inline int64_t sb_meta(int D, int NG, int a, int gi, int t) {
  return sb_meta_off(D) + ((int64_t)(a * NG + gi) * sub_tokens(D) + t) * 2;
}
// Physical byte offset of K code (token t in sub-block, element d).
__host__ __device__ inline int64_t sb_kcode(int D, int t, int d) {
  int chunk = d >> 4;
  if (D >= 128) chunk ^= (t & 1) << 2;
  return (int64_t)t * D + chunk * 16 + (d & 15);
}
__host__ __device__ inline int64_t sb_vcode(int D, int t, int d) {
  return sb_voff(D) + (int64_t)d * sub_tokens(D) + t;
}

// Raw bf16 sub-block of T tokens: byte offsets of K (token t, element d) and
// V (element d, token t).
__host__ __device__ inline int64_t raw_koff(int D, int t, int d) {
  return ((int64_t)t * D + (((d >> 3) ^ (t & 1)) << 3) + (d & 7)) * 2;
}
__host__ __device__ inline int64_t raw_voff(int D, int T, int t, int d) {
  return ((int64_t)T * D + (int64_t)d * T + t) * 2;
}

// Tile, row and half of a token of a 4-bit sub-block (see above).
__host__ __device__ constexpr int q4_tile(int t) { return (t >> 2) & 3; }
__host__ __device__ constexpr int q4_row(int t) { return ((t >> 4) << 1) | (t & 1); }
__host__ __device__ constexpr int q4_hi(int t) { return (t >> 1) & 1; }
// 4-bit sub-block: byte j (0..7) of 16-element chunk c of token t. K: codes
// d = 16c + 4(j/2) + j%2 (low nibble) and d + 2; V: codes d = 16c + j and d + 8.
__host__ __device__ inline int q4_kbyte(int D, int t, int c, int j) {
  return (((q4_tile(t) * (D >> 6) + (c >> 2)) * 32 + q4_row(t) * 4 + (c & 3)) << 4) + (j >> 1) * 4 + (j & 1) * 2 +
         q4_hi(t);
}
// Bytes of the K half, and of the V half that follows it.
__host__ __device__ constexpr int q4_half(int D, int NG) { return 32 * D + 256 * NG; }
__host__ __device__ inline int q4_vbyte(int D, int NG, int t, int c, int j) {
  return q4_half(D, NG) + ((c * 32 + j * 4 + (t >> 4)) << 4) + q4_tile(t) * 4 + (t & 1) * 2 + q4_hi(t);
}
// meta array a (0 = K scale, 1 = K zero, 2 = V scale, 3 = V zero), group gi, token t
__host__ __device__ inline int q4_meta(int D, int NG, int a, int gi, int t) {
  return (a >> 1) * q4_half(D, NG) + 32 * D + (((a & 1) * NG + gi) * kSub4 + q4_row(t) * 8 + q4_tile(t) * 2 + q4_hi(t)) * 2;
}
// Element of a 4-bit chunk held in the low nibble of its byte j, and the
// distance to the one in the high nibble.
__host__ __device__ constexpr int q4_elem(bool is_k, int j) { return is_k ? 4 * (j >> 1) + (j & 1) : j; }
__host__ __device__ constexpr int q4_step(bool is_k) { return is_k ? 2 : 8; }

// Error flag bits written by kernels (pool-owned int, read + cleared by host).
constexpr int kErrTimeout = 1;
constexpr int kErrBadArg = 2;
// The pool's device words (int32): [0] error flag bits, [1] large-scale flag,
// [2] scratch of the peer fetch, [5] testing only: non-zero makes a wait of
// CTA 0 in the next decode launches run out.
constexpr int kDevWords = 8;
constexpr int kDevTestStall = 5;
constexpr int kDefaultWaitUs = 100000;  // 100 ms

#ifdef __CUDACC__
__device__ inline float load_in(const void* p, int64_t i, int dtype) {
  return dtype == 0 ? __half2float(reinterpret_cast<const __half*>(p)[i])
                    : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
// Round a float to the input dtype (f16 or bf16), RN-even, back to float.
__device__ inline float round_in(float v, int dtype) {
  return dtype == 0 ? __half2float(__float2half_rn(v)) : __bfloat162float(__float2bfloat16_rn(v));
}
__device__ inline uint32_t smem_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
#endif

}  // namespace krill
