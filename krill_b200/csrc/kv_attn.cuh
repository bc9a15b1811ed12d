// kv_attn.cuh — decode attention over the quantized cache, dequantize fused into q·Kᵀ and ·V:
// the kernel templates, instantiated per pool format in kv_attn.cu and its siblings.
//
// Replaces, for one query token per (layer, sequence): the full-cache
// dequantize of QuantizedKVCache.update (Sources/KrillCache/QuantizedKVCache.swift:71-74,
// dequantize :200-204) and MLXFast.scaledDotProductAttention with GQA
// (Sources/KrillCore/Gemma4Model.swift:516, Attention.swift:95). K/V are
// dequantized tile by tile with the reference's two fp16 roundings, so the
// only differences from the reference math are fp32 accumulation order and
// the fp16 rounding of the softmax weights fed to the ·V product.
//
// Structure (persistent, one CTA per SM):
//   - the host plans work items = (layer, seq, kv-head, range of 64-token
//     sub-blocks) and assigns them to CTAs by longest-processing-time;
//   - a producer warp streams each item's sub-blocks HBM -> shared memory with
//     plain bulk async copies (cp.async.bulk, one CTA each) into an NSTAGE ring
//     guarded by mbarriers;
//   - NCW consumer warps take the item's sub-blocks round-robin. Tensor-core
//     path (mma.sync m16n8k16, f16 in / f32 accumulate):
//        Sᵀ[16 tok × 8 heads] = Kdeq[16 tok × D] · Qᵀ[D × 8]   (GQA group <= 8)
//        Oᵀ[D × 8]           += Vdeqᵀ[D × 16 tok] · Pᵀ[16 tok × 8]
//     with Pᵀ obtained from the Sᵀ accumulators by movmatrix.trans, online
//     softmax in the exp2 domain;
//   - warps of one head combine in shared memory; a unit split over several
//     items writes fp32 partial records, merged by attn_combine_kernel in
//     bandwidth-bound plans and, in latency-bound plans, by the item that
//     arrives last (an epoch-tagged counter per unit and head).
//   - in a decode step the kernel may be launched as the append kernel's
//     programmatic dependent; every thread waits for that grid
//     (griddepcontrol.wait) before reading the pool.
// Every mbarrier wait is bounded; on timeout the kernel raises an error flag
// and runs to completion instead of hanging.
#pragma once
#include <algorithm>
#include <atomic>
#include <cstdio>
#include <type_traits>

#include "kv_device.cuh"

namespace krill {
namespace {

// A consumer may reach a stage several uses ahead of the producer (its
// stages are HPR*R apart and it may skip items), and a parity wait cannot
// tell phase u+1 from phase u-1. The producer therefore tags each stage with
// the sequence number it is filling before arming the barrier; a consumer
// first waits (bounded) for its own tag, after which the parity wait is exact.
__device__ bool wait_tag(volatile uint32_t* tag, uint32_t want, volatile int* cta_abort, int* err) {
  if (*tag == want) return true;
  const uint32_t limit = wait_limit_units(cta_abort);
  const uint64_t t0 = globaltimer();
  while (*tag != want) {
    if (((globaltimer() - t0) >> 10) > limit) {
      *cta_abort = 1;
      atomicOr(err, kErrTimeout);
      return false;
    }
  }
  return true;
}

// Bounded wait for a shared-memory word to reach `want`; on timeout raises the
// error flag and returns.
__device__ __forceinline__ void wait_count(volatile uint32_t* cnt, uint32_t want, volatile int* cta_abort,
                                           int* err) {
  const uint32_t limit = wait_limit_units(cta_abort);
  const uint64_t t0 = globaltimer();
  while (*cnt < want) {
    if (((globaltimer() - t0) >> 10) > limit) {
      *cta_abort = 1;
      atomicOr(err, kErrTimeout);
      return;
    }
  }
}

__device__ __forceinline__ uint32_t movm_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// True when every K and V scale of the sub-block has |s| < 64 (and is finite),
// i.e. the fast dequant is exact for the whole sub-block. Warp-uniform.
template <int D, int NG>
__device__ __forceinline__ bool scales_small(const uint8_t* __restrict__ sb, int lane) {
  using SG = SubGeom<D, NG>;
  constexpr int BYTES = NG * SG::T * 2;  // one [NG][T] f16 array
  bool big = false;
  for (int off = lane * 16; off < 2 * BYTES; off += 512) {
    const int a = off / BYTES;  // 0: K scales, 1: V scales (meta array 2)
    const uint4 w = *reinterpret_cast<const uint4*>(sb + SG::META + a * 2 * BYTES + (off - a * BYTES));
    big |= (__vcmpgeu2(w.x & 0x7fff7fffu, 0x54005400u) | __vcmpgeu2(w.y & 0x7fff7fffu, 0x54005400u) |
            __vcmpgeu2(w.z & 0x7fff7fffu, 0x54005400u) | __vcmpgeu2(w.w & 0x7fff7fffu, 0x54005400u)) != 0;
  }
  return !__any_sync(0xffffffffu, big);
}

template <int D>
struct TCState {
  float o[D / 16][4];
  float m[2], l[2];
  uint32_t qf[D / 64][8];
};


// This lane's Qᵀ fragments for one (unit, head): q[head = r][16*(tig+4hh) +
// 0..15], fetched as raw words ahead of use (fetch_q) so that the next item's
// query arrives while the current one computes, then converted (set_q).
template <int D>
struct QRaw {
  uint4 w[D / 64][2];
};

// Column r = lane / 4 of the tile (see AttnUnit::nq): query r / g, head r % g.
template <int D>
__device__ __forceinline__ void fetch_q(QRaw<D>& qr, const void* q, int64_t row_elem, int g, int cols,
                                        int64_t row_elems, int lane) {
  const int r = lane >> 2, tig = lane & 3;
  const int64_t cbase = row_elem + col_off(r, g, row_elems, D);
#pragma unroll
  for (int hh = 0; hh < D / 64; ++hh) {
    if (r < cols) {
      const int64_t e = cbase + 16 * (tig + 4 * hh);
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(q) + e);
      qr.w[hh][0] = __ldg(p);
      qr.w[hh][1] = __ldg(p + 1);
    } else {
      qr.w[hh][0] = make_uint4(0u, 0u, 0u, 0u);
      qr.w[hh][1] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// st.qf from fetched words (bf16 queries become f16 for the int8 path).
template <int D, int FMT = kFmtInt8>
__device__ __forceinline__ void set_q(TCState<D>& st, const QRaw<D>& qr, int q_dtype) {
#pragma unroll
  for (int hh = 0; hh < D / 64; ++hh) {
    const uint4 a = qr.w[hh][0], b = qr.w[hh][1];
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (FMT == kFmtInt8 && q_dtype == 1) {  // bf16 -> f16 (exact in the f16 normal range)
        __nv_bfloat162 bv = *reinterpret_cast<__nv_bfloat162*>(&w[i]);
        float2 f = __bfloat1622float2(bv);
        w[i] = f2h2(f.x, f.y);
      }
      st.qf[hh][i] = w[i];
    }
  }
}

template <int D>
__device__ __forceinline__ void reset_state(TCState<D>& st) {
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
    for (int c = 0; c < 4; ++c) st.o[mt][c] = 0.f;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
}

// Process one 64-token sub-block resident in shared memory at `sb` for QT
// query tiles of 8 columns (st[q]; QT = 2 for multi-query units of more than
// 8 columns): each K and V fragment is dequantized once and feeds the MMAs of
// every tile. pos0 = absolute position of its token 0; tokens outside
// [t_lo, t_hi) are masked (only checked when `boundary`), and for this lane's
// two columns 2*tig and 2*tig + 1 of tile q also those at or past th[q][0] /
// th[q][1] (<= t_hi).
template <int D, int NG, bool FAST, int QT>
__device__ __forceinline__ void tc_subblock(const uint8_t* __restrict__ sb, TCState<D> (&st)[QT],
                                            int lane, float scale_log2, bool boundary, int pos0,
                                            int t_lo, int t_hi, const int (&th)[QT][2]) {
  using SG = SubGeom<D, NG>;
  constexpr bool SWZ = D >= 128;
  const int r = lane >> 2, tig = lane & 3;
  const uint32_t selh = (r & 1) ? 0x3232u : 0x1010u;

  // ---- K phase: Sᵀ = Kdeq · Qᵀ for NU m-tiles of 16 tokens ----
  // Rows r and r + 8 of m-tile u hold tokens TPT*(r>>1) + 4u + (r&1) and that
  // plus 2: after movmatrix.trans this is exactly the token order of the V
  // fragments, where lane tig holds tokens TPT*tig + 4u + 0..3.
  constexpr int NU = SG::NU, TPT = SG::TPT;
  float s[QT][NU][4];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int tbase = TPT * (r >> 1) + 4 * u;
    const int ta = tbase + (r & 1);
    const int tb = ta + 2;
    float acc[QT][4];
#pragma unroll
    for (int q = 0; q < QT; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.f;
#pragma unroll
    for (int hh = 0; hh < D / 64; ++hh) {
      const int grp = (64 * hh) / SG::G;
      const int chunk = tig + 4 * hh;
      const int phys = SWZ ? (chunk ^ ((r & 1) << 2)) : chunk;
      const uint4 wa = *reinterpret_cast<const uint4*>(sb + ta * D + phys * 16);
      const uint4 wb = *reinterpret_cast<const uint4*>(sb + tb * D + phys * 16);
      const uint2 ks4 = *reinterpret_cast<const uint2*>(sb + SG::meta(0, grp, tbase));
      const uint2 kz4 = *reinterpret_cast<const uint2*>(sb + SG::meta(1, grp, tbase));
      const uint32_t sA = __byte_perm(ks4.x, 0, selh), sB = __byte_perm(ks4.y, 0, selh);
      const uint32_t zA = __byte_perm(kz4.x, 0, selh), zB = __byte_perm(kz4.y, 0, selh);
      const uint32_t wav[4] = {wa.x, wa.y, wa.z, wa.w};
      const uint32_t wbv[4] = {wb.x, wb.y, wb.z, wb.w};
      const uint32_t nsA = neg1024(sA), nsB = neg1024(sB);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a0, a1, a2, a3;
        if constexpr (FAST) {
          a0 = deq2_fast(wav[k], 0x4140u, sA, nsA, zA);
          a1 = deq2_fast(wbv[k], 0x4140u, sB, nsB, zB);
          a2 = deq2_fast(wav[k], 0x4342u, sA, nsA, zA);
          a3 = deq2_fast(wbv[k], 0x4342u, sB, nsB, zB);
        } else {
          a0 = deq2(wav[k], 0x4140u, sA, zA);
          a1 = deq2(wbv[k], 0x4140u, sB, zB);
          a2 = deq2(wav[k], 0x4342u, sA, zA);
          a3 = deq2(wbv[k], 0x4342u, sB, zB);
        }
#pragma unroll
        for (int q = 0; q < QT; ++q)
          mma16816(acc[q], a0, a1, a2, a3, st[q].qf[hh][2 * k], st[q].qf[hh][2 * k + 1]);
      }
    }
#pragma unroll
    for (int q = 0; q < QT; ++q) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[q][u][c] = acc[q][c] * scale_log2;
      if (boundary) {  // fragment: [0] (ta, col 2tig), [1] (ta, 2tig+1), [2] (tb, 2tig), [3] (tb, 2tig+1)
        const int pa = pos0 + ta, pb = pos0 + tb;
        if (pa < t_lo || pa >= th[q][0]) s[q][u][0] = -INFINITY;
        if (pa < t_lo || pa >= th[q][1]) s[q][u][1] = -INFINITY;
        if (pb < t_lo || pb >= th[q][0]) s[q][u][2] = -INFINITY;
        if (pb < t_lo || pb >= th[q][1]) s[q][u][3] = -INFINITY;
      }
    }
  }

  // ---- online softmax per tile (heads 2*tig, 2*tig+1 live in this lane) ----
  uint32_t pb[QT][NU][2];
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      mx0 = fmaxf(mx0, fmaxf(s[q][u][0], s[q][u][2]));
      mx1 = fmaxf(mx1, fmaxf(s[q][u][1], s[q][u][3]));
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
    }
    const float mn0 = fmaxf(st[q].m[0], mx0), mn1 = fmaxf(st[q].m[1], mx1);
    const float b0 = (mn0 == -INFINITY) ? 0.f : mn0;
    const float b1 = (mn1 == -INFINITY) ? 0.f : mn1;
    const float al0 = exp2f(st[q].m[0] - b0), al1 = exp2f(st[q].m[1] - b1);
    st[q].m[0] = mn0;
    st[q].m[1] = mn1;
    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const float p0 = exp2f(s[q][u][0] - b0), p1 = exp2f(s[q][u][1] - b1);
      const float p2 = exp2f(s[q][u][2] - b0), p3 = exp2f(s[q][u][3] - b1);
      ps0 += p0 + p2;
      ps1 += p1 + p3;
      pb[q][u][0] = movm_trans(f2h2(p0, p1));
      pb[q][u][1] = movm_trans(f2h2(p2, p3));
    }
    st[q].l[0] = st[q].l[0] * al0 + ps0;
    st[q].l[1] = st[q].l[1] * al1 + ps1;
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt) {
      st[q].o[mt][0] *= al0;
      st[q].o[mt][1] *= al1;
      st[q].o[mt][2] *= al0;
      st[q].o[mt][3] *= al1;
    }
  }

  // ---- V phase: Oᵀ += Vdeqᵀ · Pᵀ ----
  const uint8_t* vt = sb + SG::VOFF;
#pragma unroll
  for (int grp = 0; grp < NG; ++grp) {
    // this lane's TPT tokens: TPT*tig .. TPT*tig + TPT - 1 (TPT/2 words of two)
    constexpr int NW = TPT / 2;
    uint32_t vs[NW], vz[NW];
#pragma unroll
    for (int c = 0; c < NW / 4; ++c) {
      const uint4 sw = *reinterpret_cast<const uint4*>(sb + SG::meta(2, grp, TPT * tig + 8 * c));
      const uint4 zw = *reinterpret_cast<const uint4*>(sb + SG::meta(3, grp, TPT * tig + 8 * c));
      vs[4 * c] = sw.x; vs[4 * c + 1] = sw.y; vs[4 * c + 2] = sw.z; vs[4 * c + 3] = sw.w;
      vz[4 * c] = zw.x; vz[4 * c + 1] = zw.y; vz[4 * c + 2] = zw.z; vz[4 * c + 3] = zw.w;
    }
    if (boundary) {
      // Invalid tokens get scale = zero = 0 so their (possibly stale) codes
      // dequantize to exactly 0 and cannot inject non-finite values.
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int p = pos0 + TPT * tig + 2 * i;
        const uint32_t m = ((p >= t_lo && p < t_hi) ? 0x0000ffffu : 0u) |
                           ((p + 1 >= t_lo && p + 1 < t_hi) ? 0xffff0000u : 0u);
        vs[i] &= m;
        vz[i] &= m;
      }
    }
    uint32_t nvs[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) nvs[i] = FAST ? neg1024(vs[i]) : 0u;
#pragma unroll
    for (int mi = 0; mi < SG::G / 16; ++mi) {
      const int mt = grp * (SG::G / 16) + mi;
      const int d = 16 * mt + r;
      uint32_t xv[NU], yv[NU];
      if constexpr (NU == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(vt + d * SG::T + TPT * tig);
        const uint4 y = *reinterpret_cast<const uint4*>(vt + (d + 8) * SG::T + TPT * tig);
        xv[0] = x.x; xv[1] = x.y; xv[2] = x.z; xv[3] = x.w;
        yv[0] = y.x; yv[1] = y.y; yv[2] = y.z; yv[3] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(vt + d * SG::T + TPT * tig);
        const uint2 y = *reinterpret_cast<const uint2*>(vt + (d + 8) * SG::T + TPT * tig);
        xv[0] = x.x; xv[1] = x.y;
        yv[0] = y.x; yv[1] = y.y;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        uint32_t a0, a1, a2, a3;
        if constexpr (FAST) {
          a0 = deq2_fast(xv[u], 0x4140u, vs[2 * u], nvs[2 * u], vz[2 * u]);
          a1 = deq2_fast(yv[u], 0x4140u, vs[2 * u], nvs[2 * u], vz[2 * u]);
          a2 = deq2_fast(xv[u], 0x4342u, vs[2 * u + 1], nvs[2 * u + 1], vz[2 * u + 1]);
          a3 = deq2_fast(yv[u], 0x4342u, vs[2 * u + 1], nvs[2 * u + 1], vz[2 * u + 1]);
        } else {
          a0 = deq2(xv[u], 0x4140u, vs[2 * u], vz[2 * u]);
          a1 = deq2(yv[u], 0x4140u, vs[2 * u], vz[2 * u]);
          a2 = deq2(xv[u], 0x4342u, vs[2 * u + 1], vz[2 * u + 1]);
          a3 = deq2(yv[u], 0x4342u, vs[2 * u + 1], vz[2 * u + 1]);
        }
#pragma unroll
        for (int q = 0; q < QT; ++q) mma16816(st[q].o[mt], a0, a1, a2, a3, pb[q][u][0], pb[q][u][1]);
      }
    }
  }
}


// Process one raw bf16 sub-block (the unquantized comparison format):
// Sᵀ = K·Qᵀ on bf16 tensor cores (K and q are bf16, exact products), then the
// same online softmax and Oᵀ += Vᵀ·Pᵀ in f16 with V converted exactly (V
// magnitudes beyond the f16 range are not supported). Same fragment
// permutation as tc_subblock, so q fragments and the state are shared.
template <int D>
__device__ __forceinline__ void tc_subblock_raw(const uint8_t* __restrict__ sb, TCState<D>& st,
                                                int lane, float scale_log2, bool boundary, int pos0,
                                                int t_lo, int t_hi) {
  using SG = SubGeom<D, 1, kFmtBf16>;
  constexpr int NU = SG::NU, TPT = SG::TPT;
  const int r = lane >> 2, tig = lane & 3;
  float s[NU][4];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int ta = TPT * (r >> 1) + 4 * u + (r & 1);
    const int tb = ta + 2;  // same parity as ta
    const int sw = ta & 1;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int hh = 0; hh < D / 64; ++hh) {
      // logical 16-byte chunks c, c+1 (d = 16 (tig + 4 hh) .. + 15) sit at
      // physical chunks c ^ sw, (c + 1) ^ sw of their row
      const int c = 2 * (tig + 4 * hh);
      const uint8_t* ra = sb + (size_t)ta * D * 2;
      const uint8_t* rb = sb + (size_t)tb * D * 2;
      const uint4 a0 = *reinterpret_cast<const uint4*>(ra + ((c ^ sw) << 4));
      const uint4 a1 = *reinterpret_cast<const uint4*>(ra + (((c + 1) ^ sw) << 4));
      const uint4 b0 = *reinterpret_cast<const uint4*>(rb + ((c ^ sw) << 4));
      const uint4 b1 = *reinterpret_cast<const uint4*>(rb + (((c + 1) ^ sw) << 4));
      const uint32_t wa[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
      const uint32_t wb[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma16816_bf16(acc, wa[2 * k], wb[2 * k], wa[2 * k + 1], wb[2 * k + 1], st.qf[hh][2 * k],
                      st.qf[hh][2 * k + 1]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) s[u][c] = acc[c] * scale_log2;
    if (boundary) {
      const int pa = pos0 + ta, pb = pos0 + tb;
      if (pa < t_lo || pa >= t_hi) s[u][0] = s[u][1] = -INFINITY;
      if (pb < t_lo || pb >= t_hi) s[u][2] = s[u][3] = -INFINITY;
    }
  }
  float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    mx0 = fmaxf(mx0, fmaxf(s[u][0], s[u][2]));
    mx1 = fmaxf(mx1, fmaxf(s[u][1], s[u][3]));
  }
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
  }
  const float mn0 = fmaxf(st.m[0], mx0), mn1 = fmaxf(st.m[1], mx1);
  const float b0 = (mn0 == -INFINITY) ? 0.f : mn0;
  const float b1 = (mn1 == -INFINITY) ? 0.f : mn1;
  const float al0 = exp2f(st.m[0] - b0), al1 = exp2f(st.m[1] - b1);
  st.m[0] = mn0;
  st.m[1] = mn1;
  float ps0 = 0.f, ps1 = 0.f;
  uint32_t pb[NU][2];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const float p0 = exp2f(s[u][0] - b0), p1 = exp2f(s[u][1] - b1);
    const float p2 = exp2f(s[u][2] - b0), p3 = exp2f(s[u][3] - b1);
    ps0 += p0 + p2;
    ps1 += p1 + p3;
    pb[u][0] = movm_trans(f2h2(p0, p1));
    pb[u][1] = movm_trans(f2h2(p2, p3));
  }
  st.l[0] = st.l[0] * al0 + ps0;
  st.l[1] = st.l[1] * al1 + ps1;
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    st.o[mt][0] *= al0;
    st.o[mt][1] *= al1;
    st.o[mt][2] *= al0;
    st.o[mt][3] *= al1;
  }
  // ---- V: rows d and d + 8, this lane's tokens TPT*tig .. +TPT-1 ----
  const uint8_t* vt = sb + SG::VOFF;
  constexpr int NW = TPT / 2;  // bf16 pairs per row
  uint32_t vmask[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    // invalid tokens read as zero so stale contents cannot inject non-finite values
    const int pp = pos0 + TPT * tig + 2 * i;
    vmask[i] = !boundary ? 0xffffffffu
                         : (((pp >= t_lo && pp < t_hi) ? 0x0000ffffu : 0u) |
                            ((pp + 1 >= t_lo && pp + 1 < t_hi) ? 0xffff0000u : 0u));
  }
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    const int d = 16 * mt + r;
    uint32_t xv[NW], yv[NW];
#pragma unroll
    for (int q4 = 0; q4 < NW / 4; ++q4) {
      const uint4 x = *reinterpret_cast<const uint4*>(vt + ((size_t)d * SG::T + TPT * tig) * 2 + 16 * q4);
      const uint4 y = *reinterpret_cast<const uint4*>(vt + ((size_t)(d + 8) * SG::T + TPT * tig) * 2 + 16 * q4);
      xv[4 * q4] = x.x; xv[4 * q4 + 1] = x.y; xv[4 * q4 + 2] = x.z; xv[4 * q4 + 3] = x.w;
      yv[4 * q4] = y.x; yv[4 * q4 + 1] = y.y; yv[4 * q4 + 2] = y.z; yv[4 * q4 + 3] = y.w;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const uint32_t a0 = bf2h2(xv[2 * u] & vmask[2 * u]);
      const uint32_t a1 = bf2h2(yv[2 * u] & vmask[2 * u]);
      const uint32_t a2 = bf2h2(xv[2 * u + 1] & vmask[2 * u + 1]);
      const uint32_t a3 = bf2h2(yv[2 * u + 1] & vmask[2 * u + 1]);
      mma16816(st.o[mt], a0, a1, a2, a3, pb[u][0], pb[u][1]);
    }
  }
}

// ---------------------------------------------------------------------------
// 4-bit pools. A value is c * s + z, with a scale s and zero z per (token,
// group), so the products need only the codes c in the MMA and the rest in
// f32 on its results:
//   q.k_t = sum_g s_tg (sum_{d in g} q_d c_td) + z_tg (sum_{d in g} q_d)
//   o_d   = sum_t (p_t s_tg) c_td + sum_t p_t z_tg            (g = group of d)
// A code needs no conversion: its bits, masked in place, are the f16
// subnormal c * 2^-24 (nibble at bit 0 of a half) or 16 c * 2^-24 (bit 4),
// which the tensor core multiplies exactly. The powers of two are folded into
// the query (elements k + 8 of a tile carry 1/16) and into the output rows.
// What is rounded: p to f16 (as on the int8 path), p s to f16 and z + 7.5 s to
// f16; the query is exact (normalised by a power of two per head). To keep the
// rounding error of p s at the size of the values and not of the codes'
// offset, z is split as (z + 7.5 s) - 7.5 s, and the second part uses the
// rounded p s (their sum comes from one more MMA against a constant). Each sub-block's P.V starts from zero
// accumulators and joins the running output by one f32 fma per element, which
// is also its rescale: the truncation of the tensor core's accumulation, a
// bias on sums of non-negative codes, does not build up over a long sequence.
// p carries a factor 2^bias (8, or 0 while some scale of the pool is 64 or
// more) that keeps p s of small scales above the f16 subnormals.
template <int NG>
struct Q4State {
  float cs[2];      // softmax scale * log2(e) * 2^24 / normalisation, per column
  float zs[2][NG];  // sum of p (z + 7.5 s) over this lane's tokens, less an eighth of 7.5 sum (p s)
  uint32_t zb[2];   // the group sums of the query, as the B operand of the zeros' MMA (see set_q4)
};
__device__ __forceinline__ float2 q4_floats(uint32_t w, int q_dtype) {
  return q_dtype == 1 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(u2h(w));
}

// st.qf and x from fetched words: q * f in f16 with f a power of two that puts
// the head's largest element in [2^14, 2^15). A negative softmax scale enters
// by its sign here, so that the scores' scale is positive.
template <int D, int NG>
__device__ __forceinline__ void set_q4(TCState<D>& st, Q4State<NG>& x, const QRaw<D>& qr, int q_dtype,
                                       float scale_log2, int lane) {
  const int tig = lane & 3;
  float mx = 0.f;
#pragma unroll
  for (int hh = 0; hh < D / 64; ++hh) {
    const uint4 a = qr.w[hh][0], b = qr.w[hh][1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = q4_floats(w[i], q_dtype);
      mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
    }
  }
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  const int fe = min(max(268 - (int)(__float_as_uint(mx) >> 23), 1), 253);  // biased exponent of f
  const float f = copysignf(__uint_as_float((uint32_t)fe << 23), scale_log2);
  float sum[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
  for (int hh = 0; hh < D / 64; ++hh) {
    const uint4 a = qr.w[hh][0], b = qr.w[hh][1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = q4_floats(w[i], q_dtype);
      const float lo = v.x * f, hi = v.y * f;
      sum[hh * NG / (D / 64)] += lo + hi;
      st.qf[hh][i] = (i & 1) ? f2h2(lo * 0.0625f, hi * 0.0625f) : f2h2(lo, hi);
    }
  }
  // (not below 1e-37, so that a masked score of -inf stays one for a scale of 0)
  const float cs = fmaxf(fabsf(scale_log2) * __uint_as_float((uint32_t)(254 - fe) << 23) * 16777216.f, 1e-37f);
#pragma unroll
  for (int c = 0; c < 2; ++c) x.cs[c] = __shfl_sync(0xffffffffu, cs, (2 * tig + c) * 4);
  // The zeros' term sum_g z_tg Q_g, Q_g = 2^-24 sum of the normalised query
  // over group g, is one MMA per token tile: lane tig = g of a token row holds
  // (z, z) at k = 2g, 2g + 1 and again at k + 8, and of a column the f16 parts
  // of Q_g there, high, middle and low. What they leave out is below 2^-25.
  float mine = 0.f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float t = sum[g] + __shfl_xor_sync(0xffffffffu, sum[g], 1);
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    if (tig == g) mine = t * 5.9604644775390625e-08f;  // 2^-24
    x.zs[0][g] = x.zs[1][g] = 0.f;
  }
  const __half h0 = __float2half_rn(mine);
  const float r0 = mine - __half2float(h0);
  const __half h1 = __float2half_rn(r0), h2 = __float2half_rn(r0 - __half2float(h1));
  x.zb[0] = h2u(__halves2half2(h0, h1));
  x.zb[1] = h2u(__halves2half2(h2, __ushort_as_half(0)));
}

// to[0..1] += a[0..1] * b
__device__ __forceinline__ void f2_fma_to(float* to, const float* a, F2 b) {
  const F2 y = f2_fma(f2(a[0], a[1]), b, f2(to[0], to[1]));
  to[0] = f2_lo(y);
  to[1] = f2_hi(y);
}
__device__ __forceinline__ uint32_t q4_word(const uint4& w, int u) {
  return u == 0 ? w.x : u == 1 ? w.y : u == 2 ? w.z : w.w;
}
__device__ __forceinline__ float2 q4_pair(const uint4& w, int u) { return __half22float2(u2h(q4_word(w, u))); }

// tc_subblock for 4-bit pools in two parts (same arguments; row r of token
// tile u is token 16 (r / 2) + 4u + r % 2, rows r + 8 the tokens 2 further): the K half gives
// the scores s and, after the online softmax, p * 2^bias in their place, the
// f16 pairs ph and the rescale al of what came before; the V half adds P.V.
// ILV token tiles (K) or row tiles (V) advance together, so that consecutive
// MMAs are independent.
template <int D, int NG, int QT, int ILV>
__device__ __forceinline__ void q4_scores(const uint8_t* __restrict__ sb, TCState<D> (&st)[QT],
                                          Q4State<NG> (&x)[QT], int lane, bool boundary, int pos0, int t_lo,
                                          const int (&th)[QT][2], float (&s)[QT][4][4]) {
  using SG = SubGeom<D, NG, kFmtInt4>;
  constexpr int NHH = D / 64, HPG = NHH / NG, NU = SG::NU;
  static_assert(NU == 4 && NHH % NG == 0, "four token tiles per sub-block, groups of whole 64-element runs");
  const int r = lane >> 2, tig = lane & 3;
  const uint8_t* meta = sb + SG::META4 + r * 16;  // scales, + (NG + group) * 128 zeros

  // s = sum_g z Q_g, then + s_g (q . c)_g
  {
    const uint4 kzw = *reinterpret_cast<const uint4*>(meta + (NG + min(tig, NG - 1)) * 128);
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const uint32_t za = __byte_perm(q4_word(kzw, u), 0, 0x1010), zb = __byte_perm(q4_word(kzw, u), 0, 0x3232);
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        s[q][u][0] = s[q][u][1] = s[q][u][2] = s[q][u][3] = 0.f;
        mma16816(s[q][u], za, zb, za, zb, x[q].zb[0], x[q].zb[1]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint4 ksw = *reinterpret_cast<const uint4*>(meta + g * 128);
#pragma unroll
    for (int u0 = 0; u0 < NU; u0 += ILV) {
      float acc[QT][ILV][4];
#pragma unroll
      for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int i = 0; i < ILV; ++i) acc[q][i][0] = acc[q][i][1] = acc[q][i][2] = acc[q][i][3] = 0.f;
#pragma unroll
      for (int hg = 0; hg < HPG; ++hg) {
        const int hh = g * HPG + hg;
        uint4 w[ILV];
#pragma unroll
        for (int i = 0; i < ILV; ++i)
          w[i] = *reinterpret_cast<const uint4*>(sb + (((u0 + i) * NHH + hh) * 32 + lane) * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < ILV; ++i) {
            const uint32_t c = q4_word(w[i], k), v = c >> 8;
            const uint32_t a0 = c & 0x000f000fu, a2 = c & 0x00f000f0u;
            const uint32_t a1 = v & 0x000f000fu, a3 = v & 0x00f000f0u;
#pragma unroll
            for (int q = 0; q < QT; ++q)
              mma16816(acc[q][i], a0, a1, a2, a3, st[q].qf[hh][2 * k], st[q].qf[hh][2 * k + 1]);
          }
      }
#pragma unroll
      for (int i = 0; i < ILV; ++i) {
        const float2 ks = q4_pair(ksw, u0 + i);
#pragma unroll
        for (int q = 0; q < QT; ++q)
          for (int c = 0; c < 4; c += 2) f2_fma_to(s[q][u0 + i] + c, acc[q][i] + c, c < 2 ? f2(ks.x, ks.x) : f2(ks.y, ks.y));
      }
    }
  }
  if (boundary) {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int pa = pos0 + 16 * (r >> 1) + 4 * u + (r & 1), pb = pa + 2;
        if (pa < t_lo || pa >= th[q][0]) s[q][u][0] = -INFINITY;
        if (pa < t_lo || pa >= th[q][1]) s[q][u][1] = -INFINITY;
        if (pb < t_lo || pb >= th[q][0]) s[q][u][2] = -INFINITY;
        if (pb < t_lo || pb >= th[q][1]) s[q][u][3] = -INFINITY;
      }
  }

}

template <int D, int NG, int QT>
__device__ __forceinline__ void q4_softmax(TCState<D> (&st)[QT], const Q4State<NG> (&x)[QT], float bias,
                                           float (&s)[QT][4][4], uint32_t (&ph)[QT][4][2], float (&al)[QT][2]) {
  constexpr int NU = 4;
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      mx0 = fmaxf(mx0, fmaxf(s[q][u][0], s[q][u][2]));
      mx1 = fmaxf(mx1, fmaxf(s[q][u][1], s[q][u][3]));
    }
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
    }
    const float mn0 = fmaxf(st[q].m[0], mx0 * x[q].cs[0]), mn1 = fmaxf(st[q].m[1], mx1 * x[q].cs[1]);
    const float b0 = (mn0 == -INFINITY) ? 0.f : mn0;
    const float b1 = (mn1 == -INFINITY) ? 0.f : mn1;
    al[q][0] = ex2_ftz(st[q].m[0] - b0);
    al[q][1] = ex2_ftz(st[q].m[1] - b1);
    st[q].m[0] = mn0;
    st[q].m[1] = mn1;
    const F2 e = f2(bias - b0, bias - b1), cs = f2(x[q].cs[0], x[q].cs[1]);
    F2 ps = f2(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const F2 y = f2_fma(f2(s[q][u][c], s[q][u][c + 1]), cs, e);
        s[q][u][c] = ex2_ftz(f2_lo(y));
        s[q][u][c + 1] = ex2_ftz(f2_hi(y));
        ps = f2_add(ps, f2(s[q][u][c], s[q][u][c + 1]));
        ph[q][u][c / 2] = f2h2(s[q][u][c], s[q][u][c + 1]);
      }
    ps = f2_fma(f2(st[q].l[0], st[q].l[1]), f2(al[q][0], al[q][1]), ps);
    st[q].l[0] = f2_lo(ps);
    st[q].l[1] = f2_hi(ps);
  }

}

// The weights times the V scales as B operands, per group, and the zeros' part
// of the output; s and ph are not needed after it.
template <int D, int NG, int QT>
__device__ __forceinline__ void q4_weights(const uint8_t* __restrict__ vb, Q4State<NG> (&x)[QT], int lane,
                                           bool boundary, int pos0, int t_lo, int t_hi, const float (&s)[QT][4][4],
                                           const uint32_t (&ph)[QT][4][2], const float (&al)[QT][2],
                                           uint32_t (&pb)[QT][NG][4][2]) {
  constexpr int NU = 4;
  const int r = lane >> 2;
  const uint8_t* meta = vb + SubGeom<D, NG, kFmtInt4>::META4 + r * 16;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    uint4 vsw = *reinterpret_cast<const uint4*>(meta + g * 128);
    uint4 vzw = *reinterpret_cast<const uint4*>(meta + (NG + g) * 128);
    if (boundary) {  // a token outside the range may hold any scale: it counts as zero
      uint32_t mk[4];
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int pa = pos0 + 16 * (r >> 1) + 4 * u + (r & 1), pc = pa + 2;
        mk[u] = ((pa >= t_lo && pa < t_hi) ? 0x0000ffffu : 0u) | ((pc >= t_lo && pc < t_hi) ? 0xffff0000u : 0u);
      }
      vsw = make_uint4(vsw.x & mk[0], vsw.y & mk[1], vsw.z & mk[2], vsw.w & mk[3]);
      vzw = make_uint4(vzw.x & mk[0], vzw.y & mk[1], vzw.z & mk[2], vzw.w & mk[3]);
    }
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      F2 zs = f2(0.f, 0.f);
      float one[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const uint32_t vs = q4_word(vsw, u);
        const float2 z = __half22float2(__hfma2(u2h(0x47804780u), u2h(vs), u2h(q4_word(vzw, u))));  // z + 7.5 s
        zs = f2_fma(f2(s[q][u][0], s[q][u][1]), f2(z.x, z.x), zs);
        zs = f2_fma(f2(s[q][u][2], s[q][u][3]), f2(z.y, z.y), zs);
        pb[q][g][u][0] = movm_trans(h2u(__hmul2(u2h(ph[q][u][0]), u2h(__byte_perm(vs, 0, 0x1010)))));
        pb[q][g][u][1] = movm_trans(h2u(__hmul2(u2h(ph[q][u][1]), u2h(__byte_perm(vs, 0, 0x3232)))));
        mma16816(one, 0x3b803b80u, 0x3b803b80u, 0x3b803b80u, 0x3b803b80u, pb[q][g][u][0], pb[q][g][u][1]);  // 7.5 / 8
      }
      x[q].zs[0][g] = fmaf(x[q].zs[0][g], al[q][0], f2_lo(zs) - one[0]);
      x[q].zs[1][g] = fmaf(x[q].zs[1][g], al[q][1], f2_hi(zs) - one[1]);
    }
  }
}

template <int D, int NG, int QT, int ILV>
__device__ __forceinline__ void q4_output(const uint8_t* __restrict__ vb, TCState<D> (&st)[QT], int lane,
                                          const uint32_t (&pb)[QT][NG][4][2], const float (&al)[QT][2]) {
  constexpr int NU = 4, MG = D / 16 / NG;
#pragma unroll
  for (int mt0 = 0; mt0 < D / 16; mt0 += ILV) {
    const int g = mt0 / MG;
    uint4 w[ILV];
    float acc[QT][ILV][4];
#pragma unroll
    for (int i = 0; i < ILV; ++i) {
      w[i] = *reinterpret_cast<const uint4*>(vb + ((mt0 + i) * 32 + lane) * 16);
#pragma unroll
      for (int q = 0; q < QT; ++q) acc[q][i][0] = acc[q][i][1] = acc[q][i][2] = acc[q][i][3] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < ILV; ++i) {
        const uint32_t c = q4_word(w[i], u), v = c >> 8;
        const uint32_t a0 = c & 0x000f000fu, a1 = c & 0x00f000f0u;
        const uint32_t a2 = v & 0x000f000fu, a3 = v & 0x00f000f0u;
#pragma unroll
        for (int q = 0; q < QT; ++q) mma16816(acc[q][i], a0, a1, a2, a3, pb[q][g][u][0], pb[q][g][u][1]);
      }
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int i = 0; i < ILV; ++i)
        for (int c = 0; c < 4; c += 2) {
          const F2 y = f2_fma(f2(st[q].o[mt0 + i][c], st[q].o[mt0 + i][c + 1]), f2(al[q][0], al[q][1]),
                              f2(acc[q][i][c], acc[q][i][c + 1]));
          st[q].o[mt0 + i][c] = f2_lo(y);
          st[q].o[mt0 + i][c + 1] = f2_hi(y);
        }
  }
}

// The accumulators of an item become the output rows and the running max that
// of unbiased weights, as on the other formats.
template <int D, int NG>
__device__ __forceinline__ void finalize4(TCState<D>& st, const Q4State<NG>& x, float bias) {
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float z[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      z[c] = x.zs[c][g];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) z[c] += __shfl_xor_sync(0xffffffffu, z[c], off);
    }
    constexpr int MG = D / 16 / NG;
#pragma unroll
    for (int mi = 0; mi < MG; ++mi)
#pragma unroll
      for (int c = 0; c < 4; ++c)  // rows r: c * 2^-24; rows r + 8: 16 c * 2^-24
        st.o[g * MG + mi][c] = fmaf(st.o[g * MG + mi][c], c < 2 ? 16777216.f : 1048576.f, z[c & 1]);
  }
  st.m[0] -= bias;
  st.m[1] -= bias;
}

template <int D, int NG, int NCW, int R, int NSTAGE, int FMT = kFmtInt8>
struct AttnSmem {
  static constexpr int SB = SubGeom<D, NG, FMT>::SB;
  static constexpr int STAGE_BYTES = NSTAGE * SB;
  static constexpr int BAR_OFF = STAGE_BYTES;                 // 2*NSTAGE u64
  static constexpr int NV = D / 16 * 4 + 4;                   // per-lane state floats
  static constexpr int CB_OFF = BAR_OFF + 2 * NSTAGE * 8;     // [NCW - NCW/R][NV][32] f32
  static constexpr int CB_BYTES = R == 1 ? 0 : (NCW - (FMT == kFmtInt4 && R >= 4 ? 0 : NCW / R)) * NV * 32 * 4;
  static constexpr int TAG_OFF = CB_OFF + CB_BYTES;           // [NSTAGE] u32 stage tags
  static constexpr int MISC_OFF = TAG_OFF + ((NSTAGE * 4 + 15) / 16) * 16;  // abort flag
  static constexpr int LAST_OFF = MISC_OFF + 16;  // [8] per head: its piece arrived last (int4)
  static constexpr int TOTAL = LAST_OFF + (FMT == kFmtInt4 ? 32 : 0);
};

// Number of stages that fit next to the rest of the shared memory.
template <int D, int NG, int NCW, int R, int FMT = kFmtInt8>
constexpr int stages_for() {
  constexpr int fixed = AttnSmem<D, NG, NCW, R, 0, FMT>::TOTAL;
  constexpr int most = FMT == kFmtInt4 ? 24 : 16;
  constexpr int n = (232448 - fixed - 2 * 8 * most - (FMT == kFmtInt4 ? 4 * most : 0)) / AttnSmem<D, NG, NCW, R, 0, FMT>::SB;
  return n > most ? most : n;
}

// Column hq of a split unit's kv head h from its n_split partial records, by
// one warp: lane i holds the max and normalizer of record i (32 at a time), the
// lanes together one row of D outputs, and the records' rows are summed in
// record order, eight of them in flight. Read through L2: other CTAs of the
// same launch may have written them.
template <int D>
__device__ __forceinline__ void combine_row(const AttnParams& p, const AttnUnit& un, int h, int hq, int lane) {
  constexpr int V = D < 128 ? 2 : 4, EPT = D / (32 * V);  // EPT vectors of V floats per lane
  using Vec = typename std::conditional<V == 4, float4, float2>::type;
  const float* base = p.partials + ((int64_t)un.first_split * p.Hkv + h) * partial_floats(D);
  const int64_t stride = (int64_t)p.Hkv * partial_floats(D);
  const int n = un.n_split;
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(base + i * stride + hq));
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  float Ls = 0.f, Os[EPT][V];
#pragma unroll
  for (int e = 0; e < EPT; ++e)
#pragma unroll
    for (int c = 0; c < V; ++c) Os[e][c] = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane, m = min(32, n - i0);
    const float mi = i < n ? __ldcg(base + i * stride + hq) : -INFINITY;
    const float li = i < n ? __ldcg(base + i * stride + 8 + hq) : 0.f;
    const float wi = mi == -INFINITY ? 0.f : exp2f(mi - M);
    const float* o = base + i0 * stride + 16 + hq * D + lane * V;
#pragma unroll 8
    for (int k = 0; k < m; ++k) {
      Vec x[EPT];
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = __ldcg(reinterpret_cast<const Vec*>(o + k * stride + e * 32 * V));
      const float mk = __shfl_sync(0xffffffffu, mi, k);
      const float lk = __shfl_sync(0xffffffffu, li, k), wk = __shfl_sync(0xffffffffu, wi, k);
      Ls += (mk == -INFINITY) ? 0.f : lk * wk;
#pragma unroll
      for (int e = 0; e < EPT; ++e)
#pragma unroll
        for (int c = 0; c < V; ++c) {  // (an empty record's O may be anything)
          const float oi = reinterpret_cast<const float*>(&x[e])[c];
          Os[e][c] = (mk != -INFINITY) ? Os[e][c] + oi * wk : Os[e][c];
        }
    }
  }
  const float inv = 1.f / Ls;
  const int64_t orow =
      ((int64_t)un.qo_row * p.Hq + (int64_t)h * p.g) * D + col_off(hq, p.g, (int64_t)p.Hq * D, D);
#pragma unroll
  for (int e = 0; e < EPT; ++e)
#pragma unroll
    for (int c = 0; c < V; ++c) store_out(p.out, p.out_dtype, orow + (e * 32 + lane) * V + c, Os[e][c] * inv);
}

// Merge a split unit's n_split partial records for kv head h into the output,
// in one warp: the piece that finished last does this in place of a combine
// kernel. The arithmetic and its order are those of attn_combine_kernel
// (max, then the weighted sums in record order), so both give the same bits.
// Records written by other CTAs are read through L2 (ld.global.cg).
template <int D>
__device__ __forceinline__ void merge_split(const AttnParams& p, const AttnUnit& un, int h, int lane) {
  const int g = p.g, n = un.n_split, cols = unit_cols(un, g);
  const int64_t row_elems = (int64_t)p.Hq * D;
  const int64_t stride = (int64_t)p.Hkv * partial_floats(D);
  const float* base = p.partials + ((int64_t)un.first_split * p.Hkv + h) * partial_floats(D);
  // lane j < g: max and normalizer of query head j
  float M = -INFINITY, Ls = 0.f;
  if (lane < cols) {
#pragma unroll 8
    for (int i = 0; i < n; ++i) M = fmaxf(M, __ldcg(base + i * stride + lane));
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float mi = __ldcg(base + i * stride + lane);
      Ls += (mi == -INFINITY) ? 0.f : __ldcg(base + i * stride + 8 + lane) * exp2f(mi - M);
    }
  }
  const float inv = 1.f / Ls;
  constexpr int NC = D / 32;  // output dims per lane and query head
  float acc[8][NC];
#pragma unroll
  for (int hq = 0; hq < 8; ++hq)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[hq][c] = 0.f;
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const float* ri = base + i * stride;
    const float mj = lane < cols ? __ldcg(ri + lane) : -INFINITY;
    const float wj = (mj == -INFINITY) ? 0.f : exp2f(mj - M);
#pragma unroll
    for (int hq = 0; hq < 8; ++hq) {
      if (hq < cols) {
        const float mh = __shfl_sync(0xffffffffu, mj, hq);
        const float wh = __shfl_sync(0xffffffffu, wj, hq);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float o = __ldcg(ri + 16 + hq * D + lane + 32 * c);
          acc[hq][c] = (mh == -INFINITY) ? acc[hq][c] : acc[hq][c] + o * wh;
        }
      }
    }
  }
  const int64_t orow = ((int64_t)un.qo_row * p.Hq + (int64_t)h * g) * D;
#pragma unroll
  for (int hq = 0; hq < 8; ++hq) {
    if (hq < cols) {
      const float ih = __shfl_sync(0xffffffffu, inv, hq);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        store_out(p.out, p.out_dtype, orow + col_off(hq, g, row_elems, D) + lane + 32 * c, acc[hq][c] * ih);
    }
  }
}

// Count this piece's arrival at (unit, head h); true for the piece that
// completes the unit (n_split - n_pre decode pieces; the n_pre prefix records
// were finished by an earlier kernel). Called by the whole warp after its
// partial record is stored.
__device__ __forceinline__ bool arrive_split(const AttnParams& p, const AttnUnit& un, int h, int lane) {
  __threadfence();  // this lane's record stores, device-wide, before the count
  __syncwarp();
  int last = 0;
  if (lane == 0) {
    unsigned long long* c = p.split_ctr + (int64_t)un.first_split * p.Hkv + h;
    const unsigned long long need = (unsigned long long)(un.n_split - un.n_pre);
    unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(c);
    int tries = 0;
    for (; tries < (1 << 16); ++tries) {
      const unsigned long long cnt = (old >> 32) == p.epoch ? (old & 0xffffffffull) : 0ull;
      const unsigned long long got = atomicCAS(c, old, ((unsigned long long)p.epoch << 32) | (cnt + 1));
      if (got == old) {
        last = cnt + 1 == need;
        break;
      }
      old = got;
    }
    if (tries == (1 << 16)) atomicOr(p.err, kErrTimeout);
    if (last) __threadfence();  // the other pieces' records, before reading them
  }
  return __shfl_sync(0xffffffffu, last, 0) != 0;
}

// Finish one (item, head) in the warp that holds the merged state: write the
// normalized output, or a partial record plus, for the piece that arrives
// last, the merge of the unit's records.
template <int D>
__device__ __forceinline__ void finish_head(const AttnParams& p, TCState<D>& st, float l0,
                                            float l1, const AttnUnit& un, const AttnItem& item,
                                            int h, int lane) {
  const int r = lane >> 2, tig = lane & 3;
  const int g = p.g;
  const int Hkv = p.Hkv;
  const int64_t orow = ((int64_t)un.qo_row * p.Hq + (int64_t)h * g) * D;
  const int h0 = 2 * tig, h1 = 2 * tig + 1;
  const int cols = unit_cols(un, g);
  if (un.n_split == 1) {
    if (un.n_pre > 0) {
      // merge the shared-prefix records the cascade kernel completed earlier
      // in the stream (heads beyond the GQA group hold no data and are unused)
      // (loops unrolled and the O loads unconditional, so that the loads of
      // a record, and of two records, are in flight together)
      const float* rec = p.partials + ((int64_t)un.first_split * Hkv + h) * partial_floats(D);
      const int64_t stride = (int64_t)Hkv * partial_floats(D);
      const int n_pre = un.n_pre;
      float M0 = st.m[0], M1 = st.m[1];
#pragma unroll 4
      for (int i = 0; i < n_pre; ++i) {
        M0 = fmaxf(M0, rec[i * stride + (h0 & 7)]);
        M1 = fmaxf(M1, rec[i * stride + (h1 & 7)]);
      }
      const float a0 = st.m[0] == -INFINITY ? 0.f : exp2f(st.m[0] - M0);
      const float a1 = st.m[1] == -INFINITY ? 0.f : exp2f(st.m[1] - M1);
      l0 *= a0;
      l1 *= a1;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        st.o[mt][0] *= a0;
        st.o[mt][1] *= a1;
        st.o[mt][2] *= a0;
        st.o[mt][3] *= a1;
      }
      // Records of heads h0, h1 >= g are never written: their words are read
      // (the buffer spans all 8 head slots) but always discarded by the
      // selects, as are the words of empty records (b == 0).
#pragma unroll 2
      for (int i = 0; i < n_pre; ++i) {
        const float* ri = rec + i * stride;
        const float m0 = ri[h0 & 7], m1 = ri[h1 & 7];
        const float lv0 = ri[8 + (h0 & 7)], lv1 = ri[8 + (h1 & 7)];
        float ov[D / 16][4];
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          ov[mt][0] = ri[16 + (h0 & 7) * D + 16 * mt + r];
          ov[mt][2] = ri[16 + (h0 & 7) * D + 16 * mt + r + 8];
          ov[mt][1] = ri[16 + (h1 & 7) * D + 16 * mt + r];
          ov[mt][3] = ri[16 + (h1 & 7) * D + 16 * mt + r + 8];
        }
        const float b0 = m0 == -INFINITY ? 0.f : exp2f(m0 - M0);
        const float b1 = m1 == -INFINITY ? 0.f : exp2f(m1 - M1);
        const bool t0 = b0 != 0.f && h0 < cols, t1 = b1 != 0.f && h1 < cols;
        l0 = t0 ? l0 + lv0 * b0 : l0;
        l1 = t1 ? l1 + lv1 * b1 : l1;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          st.o[mt][0] = t0 ? st.o[mt][0] + ov[mt][0] * b0 : st.o[mt][0];
          st.o[mt][2] = t0 ? st.o[mt][2] + ov[mt][2] * b0 : st.o[mt][2];
          st.o[mt][1] = t1 ? st.o[mt][1] + ov[mt][1] * b1 : st.o[mt][1];
          st.o[mt][3] = t1 ? st.o[mt][3] + ov[mt][3] * b1 : st.o[mt][3];
        }
      }
    }
    const float i0 = 1.f / l0, i1 = 1.f / l1;
    const int64_t row_elems = (int64_t)p.Hq * D;
    const int64_t o0 = orow + col_off(h0, g, row_elems, D), o1 = orow + col_off(h1, g, row_elems, D);
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt) {
      const int d = 16 * mt + r;
      if (h0 < cols) {
        store_out(p.out, p.out_dtype, o0 + d, st.o[mt][0] * i0);
        store_out(p.out, p.out_dtype, o0 + d + 8, st.o[mt][2] * i0);
      }
      if (h1 < cols) {
        store_out(p.out, p.out_dtype, o1 + d, st.o[mt][1] * i1);
        store_out(p.out, p.out_dtype, o1 + d + 8, st.o[mt][3] * i1);
      }
    }
    return;
  }
  const int64_t rec = ((int64_t)un.first_split + item.idx) * Hkv + h;
  float* part = p.partials + rec * partial_floats(D);
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    const int d = 16 * mt + r;
    part[16 + h0 * D + d] = st.o[mt][0];
    part[16 + h0 * D + d + 8] = st.o[mt][2];
    part[16 + h1 * D + d] = st.o[mt][1];
    part[16 + h1 * D + d + 8] = st.o[mt][3];
  }
  if (r == 0) {
    part[h0] = st.m[0];
    part[h1] = st.m[1];
    part[8 + h0] = l0;
    part[8 + h1] = l1;
  }
  if (p.split_ctr != nullptr && arrive_split(p, un, h, lane)) merge_split<D>(p, un, h, lane);
}

// Merge the partial records of split units: one warp per (split unit, kv head,
// column of the query tile). The latency of its reads bounds it: one CTA per
// (unit, kv head) whose 128 threads walked all the columns took 106 us for
// 12 x 2 x 4 (unit, head) pairs of 32 records at head_dim 128 (12.8 MB); this
// takes 10 us, and as the programmatic dependent of the attention kernel its
// blocks are there when that one ends.
constexpr int kCombineWarps = 4;
template <int D>
__global__ void __launch_bounds__(32 * kCombineWarps) attn_combine_kernel(AttnParams p) {
  const int Hkv = p.Hkv, lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
  const int hq = (int)(w % p.max_cols), h = (int)(w / p.max_cols % Hkv);
  const int64_t ui = w / p.max_cols / Hkv;
  if (ui >= p.n_split_units) return;
  const AttnUnit un = p.units[p.split_units[ui]];  // (written before the attention kernel began)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (hq < unit_cols(un, p.g)) combine_row<D>(p, un, h, hq, lane);
}
template <int D>
cudaError_t run_combine(const AttnParams& p, cudaStream_t stream) {
  const int64_t warps = (int64_t)p.n_split_units * p.Hkv * p.max_cols;
  return launch_dependent(attn_combine_kernel<D>, dim3((unsigned)((warps + kCombineWarps - 1) / kCombineWarps)),
                          32 * kCombineWarps, stream, p);
}

// Work split inside a CTA: an item covers hg kv heads; HPR = NCW / R of them
// are processed at once, each by R warps (R = 1 when hg >= NCW), in hg / HPR
// rounds. For an item of n_sb sub-blocks the
// producer issues, per round, sub-block k of head hr as stage J0 + k*HPR + hr;
// warp (hr, r) takes the sub-blocks k = r, r + R, ...
// Threads: NCW consumer warps (two warpgroups) + one producer warpgroup, of
// which one warp issues the copies. At start the producer warpgroup gives its
// registers back (setmaxnreg.dec to 56) and the consumers take them
// (setmaxnreg.inc to 224): 128*56 + 256*224 = 384*168, the launch budget.
// (With 40 the producer's metadata prefetch spilled; 224 still holds every
// consumer without spills.)
constexpr int kProducerRegs = 56;
constexpr int kConsumerRegs = 224;

// Merges the R warps of one head through a lane-major buffer; warp rr = 0 of
// them ends with the merged state.
template <int D, int NCW, int R, typename SM>
__device__ __forceinline__ void merge_warps(TCState<D>& st, float& l0, float& l1, uint8_t* smem, int hr, int rr,
                                            int lane) {
  if constexpr (R > 1) {
    float* cb = reinterpret_cast<float*>(smem + SM::CB_OFF);
    const int nbar = 1 + hr;
    asm volatile("bar.sync %0, %1;" ::"r"(nbar), "r"(R * 32) : "memory");  // buffer free
    if (rr != 0) {
      float* mine = cb + (size_t)(hr * (R - 1) + rr - 1) * SM::NV * 32;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int c = 0; c < 4; ++c) mine[(mt * 4 + c) * 32 + lane] = st.o[mt][c];
      mine[(D / 4 + 0) * 32 + lane] = st.m[0];
      mine[(D / 4 + 1) * 32 + lane] = st.m[1];
      mine[(D / 4 + 2) * 32 + lane] = l0;
      mine[(D / 4 + 3) * 32 + lane] = l1;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(nbar), "r"(R * 32) : "memory");
    if (rr == 0) {
#pragma unroll(R <= 4 ? R : 1)
      for (int w = 1; w < R; ++w) {
        const float* o = cb + (size_t)(hr * (R - 1) + w - 1) * SM::NV * 32;
        const float m0 = o[(D / 4 + 0) * 32 + lane], m1 = o[(D / 4 + 1) * 32 + lane];
        const float M0 = fmaxf(st.m[0], m0), M1 = fmaxf(st.m[1], m1);
        const float a0 = (st.m[0] == -INFINITY) ? 0.f : exp2f(st.m[0] - M0);
        const float a1 = (st.m[1] == -INFINITY) ? 0.f : exp2f(st.m[1] - M1);
        const float b0 = (m0 == -INFINITY) ? 0.f : exp2f(m0 - M0);
        const float b1 = (m1 == -INFINITY) ? 0.f : exp2f(m1 - M1);
        l0 = l0 * a0 + o[(D / 4 + 2) * 32 + lane] * b0;
        l1 = l1 * a1 + o[(D / 4 + 3) * 32 + lane] * b1;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          st.o[mt][0] = st.o[mt][0] * a0 + o[(mt * 4 + 0) * 32 + lane] * b0;
          st.o[mt][1] = st.o[mt][1] * a1 + o[(mt * 4 + 1) * 32 + lane] * b1;
          st.o[mt][2] = st.o[mt][2] * a0 + o[(mt * 4 + 2) * 32 + lane] * b0;
          st.o[mt][3] = st.o[mt][3] * a1 + o[(mt * 4 + 3) * 32 + lane] * b1;
        }
        st.m[0] = M0;
        st.m[1] = M1;
      }
    }
  }
}

// Consumer warps of attn_tc_kernel. FAST selects the one-fma dequantization,
// exact only while every scale in the pool is below 64 in magnitude; the
// kernel picks one specialization per launch from the pool's large-scale flag
// (set by the kernels that store scales), so the hot loop carries one path.
// QT = 2: every unit of the launch is the first 8 columns of a multi-query
// unit whose other columns are the next unit (AttnUnit::nq; its shadow, with
// the same sequence, layer and pieces, but its own queries, bounds and
// records); both tiles are computed from each staged sub-block.
// SEL: the items' sub-block ranges index the picked blocks of a (unit, head)
// (AttnParams::sel) instead of the sequence; the last picked block is always
// the sequence's last, the only one that may end inside.
template <int D, int NG, int NCW, int R, int NSTAGE, int FMT, bool FAST, int QT, bool SEL>
__device__ __forceinline__ void attn_consume(const AttnParams& p, uint8_t* smem, uint8_t* stages,
                                             uint32_t bar_base, volatile int* cta_abort,
                                             volatile uint32_t* tags, int warp, int lane, int it0,
                                             int it1, int rounds) {
  using SM = AttnSmem<D, NG, NCW, R, NSTAGE, FMT>;
  constexpr int SB = SM::SB;
  constexpr int HPR = NCW / R;
  static_assert(QT == 1 || (R == 1 && FMT == kFmtInt8), "two query tiles: one warp per head, int8");
  static_assert(QT == 1 || !SEL, "picked blocks: one query per sequence");
  const int hr = warp / R, rr = warp % R;
  TCState<D> sts[QT];
  TCState<D>& st = sts[0];
  uint32_t J = 0;
  AttnItem item_next{};
  AttnUnit un_next{};
  // The query of the next (item, round) is fetched while this one computes:
  // the next item's unit after this warp's first sub-block (the item record
  // has arrived by then), its q words after the second, so neither load
  // stalls the warp. qr always holds the q of the (item, round) about to run.
  QRaw<D> qr;
  auto q_row = [&](const AttnUnit& u, int hh) {
    return ((int64_t)u.qo_row * p.Hq + (int64_t)hh * p.g) * D;
  };
  const int64_t q_row_elems = (int64_t)p.Hq * D;
  // query index (within a multi-query unit) of this lane's two columns
  const int col_q0 = D <= 128 ? (2 * (lane & 3)) / p.g : 0;
  const int col_q1 = D <= 128 ? (2 * (lane & 3) + 1) / p.g : 0;
  if (it0 < it1) {
    item_next = p.items[it0];
    un_next = p.units[item_next.unit];
    if constexpr (QT == 1)
      fetch_q<D>(qr, p.q, q_row(un_next, item_next.h0 + hr), p.g, unit_cols(un_next, p.g),
                 q_row_elems, lane);
  }
  for (int it = it0; it < it1; ++it) {
    const AttnItem item = item_next;
    const AttnUnit un = un_next;
    if (it + 1 < it1) item_next = p.items[it + 1];
    const int n_sb = item.sb_end - item.sb_begin;
    for (int rd = 0; rd < rounds; ++rd) {
      const int h = item.h0 + rd * HPR + hr;
      // with two tiles both queries are fetched here (no prefetch across the
      // item, whose registers the second tile needs); items are long
      if constexpr (QT == 2)
        fetch_q<D>(qr, p.q, q_row(un, h), p.g, unit_cols(un, p.g), q_row_elems, lane);
      reset_state(st);
      set_q<D, FMT>(st, qr, p.q_dtype);
      // the shadow unit's queries (second tile), fetched here: items are long
      // (the shadow record is read again at the finish, not kept in registers)
      AttnUnit un2 = un;
      if constexpr (QT == 2) {
        un2 = p.units[item.unit + 1];
        QRaw<D> qr2;
        fetch_q<D>(qr2, p.q, q_row(un2, h), p.g, unit_cols(un2, p.g), q_row_elems, lane);
        reset_state(sts[1]);
        set_q<D, FMT>(sts[1], qr2, p.q_dtype);
      }
      // prefetch state: 0 nothing yet, 1 next unit requested, 2 next q fetched
      int pf = 0;
      auto prefetch_step = [&]() {
        if (rd + 1 < rounds) {  // next round: same unit, the next head group
          if constexpr (QT == 1)
            fetch_q<D>(qr, p.q, q_row(un, h + HPR), p.g, unit_cols(un, p.g), q_row_elems, lane);
          pf = 2;
        } else if (it + 1 >= it1) {
          pf = 2;
        } else if (pf == 0) {
          un_next = p.units[item_next.unit];
          pf = 1;
        } else {
          if constexpr (QT == 1)
            fetch_q<D>(qr, p.q, q_row(un_next, item_next.h0 + hr), p.g, unit_cols(un_next, p.g),
                       q_row_elems, lane);
          pf = 2;
        }
      };
      // per-column bounds of a multi-query unit (AttnUnit::nq); the tiles'
      // union of positions is [t_lo, t_hi), the first column's bound b_min
      int th[QT][2];
      int b_min = INT32_MAX, t_hi = 0;
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const AttnUnit& uq = q == 0 ? un : un2;
        const int nq1 = uq.nq > 1 ? uq.nq - 1 : 0;  // column c: t_hi - (nq - 1 - c / g)
        if constexpr (D <= 128) {  // per-lane quotients computed once per launch
          th[q][0] = uq.t_hi - (nq1 - min(col_q0, nq1));
          th[q][1] = uq.t_hi - (nq1 - min(col_q1, nq1));
        } else {  // (at head_dim 256 two more live registers cost spills)
          th[q][0] = uq.t_hi - (nq1 - (2 * (lane & 3)) / p.g);
          th[q][1] = uq.t_hi - (nq1 - (2 * (lane & 3) + 1) / p.g);
        }
        b_min = min(b_min, uq.t_hi - nq1);
        t_hi = max(t_hi, uq.t_hi);
      }
      for (int k = rr; k < n_sb; k += R) {
        const uint32_t jj = J + (uint32_t)k * HPR + hr;
        const uint32_t stage = jj % NSTAGE;
        wait_tag(tags + stage, jj, cta_abort, p.err);
        mbar_wait(bar_base + 8 * stage, (jj / NSTAGE) & 1, cta_abort, p.err);
        const int j = item.sb_begin + k;
        constexpr int T = SubGeom<D, NG, FMT>::T;
        int pos0 = j * T;
        bool boundary = pos0 < un.t_lo || pos0 + T > b_min;
        if constexpr (SEL) {  // only the last picked block, the sequence's last, may be partial
          pos0 = (t_hi - 1) / T * T;
          boundary = j == min(p.sel_stride, (t_hi + T - 1) / T) - 1 && pos0 + T > t_hi;
        }
        const uint8_t* sbp = stages + (size_t)stage * SB;
        if constexpr (FMT == kFmtBf16)
          tc_subblock_raw<D>(sbp, st, lane, p.scale_log2, boundary, pos0, un.t_lo, un.t_hi);
        else
          tc_subblock<D, NG, FAST, QT>(sbp, sts, lane, p.scale_log2, boundary, pos0, un.t_lo, t_hi, th);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_base + 8 * (NSTAGE + stage));
        if (pf < 2) prefetch_step();
      }
      while (pf < 2) prefetch_step();
      J += (uint32_t)n_sb * HPR;

      float l0 = st.l[0], l1 = st.l[1];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      merge_warps<D, NCW, R, SM>(st, l0, l1, smem, hr, rr, lane);
      if (rr == 0) finish_head<D>(p, st, l0, l1, un, item, h, lane);
      if constexpr (QT == 2) {
        float m0 = sts[1].l[0], m1 = sts[1].l[1];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          m0 += __shfl_xor_sync(0xffffffffu, m0, off);
          m1 += __shfl_xor_sync(0xffffffffu, m1, off);
        }
        finish_head<D>(p, sts[1], m0, m1, p.units[item.unit + 1], item, h, lane);
      }
    }
  }
}

// Finish one (item, head) with its R warps together (R >= 4): every warp leaves
// its state in shared memory, then each takes a share of the output elements
// and merges, normalises and stores it (or the partial record; the warps of
// the piece that arrives last then merge the unit's records, a column each).
// One warp doing all of it took 4 of a short item's 20 us at head_dim 256.
template <int D, int NCW, int R, typename SM>
__device__ __forceinline__ void finish_together(const AttnParams& p, const TCState<D>& st, float l0, float l1,
                                                uint8_t* smem, int unit, const AttnItem& item, int h, int hr, int rr,
                                                int lane) {
  const int r = lane >> 2, tig = lane & 3, c0 = 2 * tig, c1 = c0 + 1;
  float* cb = reinterpret_cast<float*>(smem + SM::CB_OFF) + (size_t)hr * R * SM::NV * 32 + lane;
  volatile int* last_s = reinterpret_cast<volatile int*>(smem + SM::LAST_OFF) + hr;
  auto sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + hr), "r"(R * 32) : "memory"); };
  sync();  // the buffer's last readers are done
  {
    float* mine = cb + rr * SM::NV * 32;
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int c = 0; c < 4; ++c) mine[(mt * 4 + c) * 32] = st.o[mt][c];
    mine[(D / 4 + 0) * 32] = st.m[0];
    mine[(D / 4 + 1) * 32] = st.m[1];
    mine[(D / 4 + 2) * 32] = l0;
    mine[(D / 4 + 3) * 32] = l1;
  }
  sync();
  const AttnUnit un = p.units[unit];
  const int cols = unit_cols(un, p.g), n_pre = un.n_split == 1 ? un.n_pre : 0;
  const float* rec = p.partials + ((int64_t)un.first_split * p.Hkv + h) * partial_floats(D);
  const int64_t stride = (int64_t)p.Hkv * partial_floats(D);
  float M0 = -INFINITY, M1 = -INFINITY, a0[R], a1[R], L0 = 0.f, L1 = 0.f;
#pragma unroll
  for (int w = 0; w < R; ++w) {
    a0[w] = cb[(w * SM::NV + D / 4 + 0) * 32];
    a1[w] = cb[(w * SM::NV + D / 4 + 1) * 32];
    M0 = fmaxf(M0, a0[w]);
    M1 = fmaxf(M1, a1[w]);
  }
  for (int i = 0; i < n_pre; ++i) {  // prefix records that the cascade kernel left
    M0 = fmaxf(M0, rec[i * stride + c0]);
    M1 = fmaxf(M1, rec[i * stride + c1]);
  }
#pragma unroll
  for (int w = 0; w < R; ++w) {
    a0[w] = a0[w] == -INFINITY ? 0.f : exp2f(a0[w] - M0);
    a1[w] = a1[w] == -INFINITY ? 0.f : exp2f(a1[w] - M1);
    L0 += cb[(w * SM::NV + D / 4 + 2) * 32] * a0[w];
    L1 += cb[(w * SM::NV + D / 4 + 3) * 32] * a1[w];
  }
  // (columns past the unit's hold no prefix record: their words are read, as
  // the buffer spans all eight, and discarded)
  for (int i = 0; i < n_pre; ++i) {
    const float* ri = rec + i * stride;
    L0 += ri[c0] == -INFINITY || c0 >= cols ? 0.f : ri[8 + c0] * exp2f(ri[c0] - M0);
    L1 += ri[c1] == -INFINITY || c1 >= cols ? 0.f : ri[8 + c1] * exp2f(ri[c1] - M1);
  }
  const bool split = un.n_split > 1;
  const float i0 = 1.f / L0, i1 = 1.f / L1;
  const int64_t row_elems = (int64_t)p.Hq * D, orow = ((int64_t)un.qo_row * p.Hq + (int64_t)h * p.g) * D;
  const int64_t o0 = orow + col_off(c0, p.g, row_elems, D), o1 = orow + col_off(c1, p.g, row_elems, D);
  float* part = p.partials + (((int64_t)un.first_split + item.idx) * p.Hkv + h) * partial_floats(D);
#pragma unroll 2
  for (int e = rr; e < D / 8; e += R) {  // row half e % 2 of row tile e / 2
    float x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < R; ++w) {
      x0 = fmaf(cb[(w * SM::NV + 2 * e) * 32], a0[w], x0);
      x1 = fmaf(cb[(w * SM::NV + 2 * e + 1) * 32], a1[w], x1);
    }
    const int d = 8 * e + r;
    for (int i = 0; i < n_pre; ++i) {
      const float* ri = rec + i * stride;
      const float v0 = ri[16 + c0 * D + d], v1 = ri[16 + c1 * D + d];
      if (ri[c0] != -INFINITY && c0 < cols) x0 = fmaf(v0, exp2f(ri[c0] - M0), x0);
      if (ri[c1] != -INFINITY && c1 < cols) x1 = fmaf(v1, exp2f(ri[c1] - M1), x1);
    }
    if (split) {
      part[16 + c0 * D + d] = x0;
      part[16 + c1 * D + d] = x1;
    } else {
      if (c0 < cols) store_out(p.out, p.out_dtype, o0 + d, x0 * i0);
      if (c1 < cols) store_out(p.out, p.out_dtype, o1 + d, x1 * i1);
    }
  }
  if (!split) return;
  if (rr == 0 && r == 0) {
    part[c0] = M0;
    part[c1] = M1;
    part[8 + c0] = L0;
    part[8 + c1] = L1;
  }
  if (p.split_ctr == nullptr) return;
  __threadfence();  // this lane's stores, device-wide, before the head's count
  sync();
  if (rr == 0) {
    const int last = arrive_split(p, un, h, lane) ? 1 : 0;
    if (lane == 0) *last_s = last;
  }
  sync();
  if (*last_s) {
    __threadfence();  // the other pieces' records, before reading them
    for (int hq = rr; hq < cols; hq += R) combine_row<D>(p, un, h, hq, lane);
  }
}

// Consumer warps for 4-bit pools. Little is kept in registers between items
// (the producer warp has their records and queries in the caches by then).
// 8 layers of 32 sequences of 512 to 8192 tokens, 8 kv heads of 128, 4 queries
// each: 170 us for 909 MB, 0.82 of copy bandwidth (the copies alone: 144 us).
// 12 layers of 2 x 32768 tokens, 4 heads, 8 queries: 91 us for 453 MB, 0.76.
// Two warps a scheduler issue in 46 % of the cycles (ALU pipe 47 %, tensor pipe
// 35 %), waiting for one another's results, not for a stage. More warps leave
// too few registers (12: 211 us, 16: 223 us, when eight took 179); the next
// sub-block's scores beside this one's output gave 169 and 98 us.
template <int D, int NG, int NCW, int R, int NSTAGE, int QT, bool SEL>
__device__ __forceinline__ void attn_consume4(const AttnParams& p, uint8_t* smem, uint8_t* stages,
                                              uint32_t bar_base, volatile int* cta_abort, volatile uint32_t* tags,
                                              int warp, int lane, int it0, int it1, int rounds) {
  using SM = AttnSmem<D, NG, NCW, R, NSTAGE, kFmtInt4>;
  constexpr int SB = SM::SB, HPR = NCW / R, T = kSub4;
  // token / row tiles advanced together: what the registers allow
  constexpr int ILV = QT == 2 ? 2 : 4;
  static_assert(QT == 1 || (R == 1 && !SEL), "two query tiles: one warp per head, whole sequences");
  const int hr = warp / R, rr = warp % R;
  // exponent bias of the softmax weights (see Q4State)
  const float bias = *reinterpret_cast<volatile const int*>(p.large_scale) == 0 ? 8.f : 0.f;
  const int64_t row_elems = (int64_t)p.Hq * D;
  uint32_t J = 0;
  for (int it = it0; it < it1; ++it) {
    const AttnItem item = p.items[it];
    const int n_sb = item.sb_end - item.sb_begin;
    for (int rd = 0; rd < rounds; ++rd) {
      const int h = item.h0 + rd * HPR + hr;
      TCState<D> st[QT];
      Q4State<NG> x[QT];
      // per-column bounds (AttnUnit::nq) as in attn_consume
      int th[QT][2], t_lo = 0, t_hi = 0, b_min = INT32_MAX;
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const AttnUnit un = p.units[item.unit + q];
        QRaw<D> qr;
        fetch_q<D>(qr, p.q, ((int64_t)un.qo_row * p.Hq + (int64_t)h * p.g) * D, p.g, unit_cols(un, p.g), row_elems, lane);
        reset_state(st[q]);
        set_q4<D, NG>(st[q], x[q], qr, p.q_dtype, p.scale_log2, lane);
        const int nq1 = un.nq > 1 ? un.nq - 1 : 0;
        th[q][0] = un.t_hi - (nq1 - min((2 * (lane & 3)) / p.g, nq1));
        th[q][1] = un.t_hi - (nq1 - min((2 * (lane & 3) + 1) / p.g, nq1));
        b_min = min(b_min, un.t_hi - nq1);
        t_hi = max(t_hi, un.t_hi);
        t_lo = un.t_lo;
      }
#pragma unroll 1
      for (int k = rr; k < n_sb; k += R) {
        const uint32_t jj = J + (uint32_t)k * HPR + hr;
        const uint32_t stage = jj % NSTAGE;
        const int j = item.sb_begin + k;
        int pos0 = j * T;
        bool boundary = pos0 < t_lo || pos0 + T > b_min;
        if constexpr (SEL) {  // only the last picked block, the sequence's last, may be partial
          pos0 = (t_hi - 1) / T * T;
          boundary = j == min(p.sel_stride, (t_hi + T - 1) / T) - 1 && pos0 + T > t_hi;
        }
        float s[QT][4][4], al[QT][2];
        uint32_t ph[QT][4][2], pb[QT][NG][4][2];
        wait_tag(tags + stage, jj, cta_abort, p.err);
        mbar_wait(bar_base + 8 * stage, (jj / NSTAGE) & 1, cta_abort, p.err);
        const uint8_t* kb = stages + (size_t)stage * SB;
        const uint8_t* vb = kb + q4_half(D, NG);
        q4_scores<D, NG, QT, ILV>(kb, st, x, lane, boundary, pos0, t_lo, th, s);
        q4_softmax<D, NG, QT>(st, x, bias, s, ph, al);
        q4_weights<D, NG, QT>(vb, x, lane, boundary, pos0, t_lo, t_hi, s, ph, al, pb);
        q4_output<D, NG, QT, ILV>(vb, st, lane, pb, al);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_base + 8 * (NSTAGE + stage));
      }
      J += (uint32_t)n_sb * HPR;
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        finalize4<D, NG>(st[q], x[q], bias);
        float l0 = st[q].l[0], l1 = st[q].l[1];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, off);
          l1 += __shfl_xor_sync(0xffffffffu, l1, off);
        }
        if constexpr (R >= 4) {
          finish_together<D, NCW, R, SM>(p, st[q], l0, l1, smem, item.unit, item, h, hr, rr, lane);
        } else {  // (two warps: the other one goes on with the next item meanwhile)
          merge_warps<D, NCW, R, SM>(st[q], l0, l1, smem, hr, rr, lane);
          if (rr == 0) finish_head<D>(p, st[q], l0, l1, p.units[item.unit + q], item, h, lane);
        }
      }
    }
  }
}

// Producer of 4-bit pools and of picked blocks: W lanes issue W consecutive
// copies at a time. (A 4-bit sub-block is half an int8 one; issued
// by one lane, whose wait, tag, arrive and copy follow one another, the copies
// of the batch of 32 sequences alone took 183 us where their bytes need 139.)
// Sources are found 32 at a time, one per lane (the picked block's index, then
// the block table entry: two dependent loads of a microsecond together), a
// batch ahead of the copies.
template <int D, int NG, int NCW, int R, int NSTAGE, int FMT, bool SEL>
__device__ __forceinline__ void produce_wide(const AttnParams& p, uint8_t* stages, uint32_t bar_base,
                                             volatile int* cta_abort, volatile uint32_t* tags, int lane, int it0,
                                             int it1, int rounds) {
  using SG = SubGeom<D, NG, FMT>;
  // copies of a step: a third of the stages at most, so that waiting for the
  // last of them does not hold back many that are free
  constexpr int HPR = NCW / R, SB = SG::SB, SPB = SG::SPB, W = NSTAGE >= 20 ? 8 : NSTAGE >= 12 ? 4 : 2;
  static_assert(NSTAGE >= W, "a step's copies must not wait for one another");
  const int Hkv = p.Hkv;
  // copy i of round rd of an item: its sub-block i / HPR of head i % HPR
  auto source = [&](const AttnItem& item, int layer, int si, int rd, int i) {
    const int h = item.h0 + rd * HPR + i % HPR;
    int sb = item.sb_begin + i / HPR;
    // (not through the read-only path: the choice may still write when this grid starts)
    if (SEL) sb = __ldcg(p.sel + ((int64_t)item.unit * Hkv + h) * p.sel_stride + sb);
    int bi = sb / SPB;
    if (p.ring > 0) bi %= p.ring;
    const int b = __ldg(p.bt + (int64_t)si * p.bt_stride + bi);
    return p.pool + (((int64_t)b * p.L + layer) * Hkv + h) * p.page_bytes + (int64_t)(sb % SPB) * SB;
  };
  if (it0 >= it1) return;
  AttnItem item = p.items[it0], item_n{};
  int layer = p.units[item.unit].layer, si = p.units[item.unit].si, layer_n = 0, si_n = 0;
  const uint8_t* src = nullptr;  // of copy q + lane
  if (lane < (item.sb_end - item.sb_begin) * HPR) src = source(item, layer, si, 0, lane);
  uint32_t J = 0;
  for (int it = it0; it < it1; ++it) {
    if (it + 1 < it1) {
      item_n = p.items[it + 1];
      layer_n = p.units[item_n.unit].layer;
      si_n = p.units[item_n.unit].si;
      if constexpr (FMT == kFmtInt4) {  // its query rows (adjacent: hg * g of them), for the consumers
        const AttnUnit* un = p.units + item_n.unit;
        const char* q0 = static_cast<const char*>(p.q) + ((int64_t)un->qo_row * p.Hq + (int64_t)item_n.h0 * p.g) * D * 2;
        for (int i = lane * 128; i < p.hg * p.g * D * 2; i += 32 * 128)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(q0 + i));
      }
    }
    const int total = (item.sb_end - item.sb_begin) * HPR;
    for (int rd = 0; rd < rounds; ++rd) {
      for (int q = 0; q < total; q += 32) {
        const uint8_t* next = nullptr;
        if (q + 32 < total) {
          if (q + 32 + lane < total) next = source(item, layer, si, rd, q + 32 + lane);
        } else if (rd + 1 < rounds) {
          if (lane < total) next = source(item, layer, si, rd + 1, lane);
        } else if (it + 1 < it1) {
          if (lane < (item_n.sb_end - item_n.sb_begin) * HPR) next = source(item_n, layer_n, si_n, 0, lane);
        }
        for (int j = 0; j < min(32, total - q); j += W) {
          const uint8_t* from =
              reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), (j + lane) & 31));
          if (lane < W && q + j + lane < total) {
            const uint32_t Jh = J + (uint32_t)(q + j + lane);
            const uint32_t stage = Jh % NSTAGE;
            if (Jh >= (uint32_t)NSTAGE)
              mbar_wait(bar_base + 8 * (NSTAGE + stage), ((Jh / NSTAGE) - 1) & 1, cta_abort, p.err);
            const uint32_t full = bar_base + 8 * stage;
            tags[stage] = Jh;  // released by the arrive below
            mbar_expect_tx(full, SB);
            bulk_g2s(smem_u32(stages + (size_t)stage * SB), from, SB, full);
          }
          __syncwarp();
        }
        src = next;
      }
      J += (uint32_t)total;
    }
    item = item_n;
    layer = layer_n;
    si = si_n;
  }
}

template <int D, int NG, int NCW, int R, int NSTAGE, int FMT, int QT = 1, bool SEL = false>
__global__ void __launch_bounds__((NCW + 4) * 32, 1) attn_tc_kernel(AttnParams p) {
  static_assert(NCW == 8, "two consumer warpgroups");
  using SM = AttnSmem<D, NG, NCW, R, NSTAGE, FMT>;
  constexpr int SB = SM::SB;
  constexpr int HPR = NCW / R;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* stages = smem;
  const uint32_t bar_base = smem_u32(smem + SM::BAR_OFF);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(smem + SM::MISC_OFF);
  volatile uint32_t* tags = reinterpret_cast<volatile uint32_t*>(smem + SM::TAG_OFF);
  volatile uint32_t* stall_word = reinterpret_cast<volatile uint32_t*>(smem + SM::MISC_OFF + 8);

  asm volatile("griddepcontrol.launch_dependents;");  // the combine kernel, which waits for this grid
  const int tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < NSTAGE; ++s) {
      mbar_init(bar_base + 8 * s, 1);             // full: producer arrive + tx
      mbar_init(bar_base + 8 * (NSTAGE + s), 1);  // empty: the consuming warp
    }
    for (int s = 0; s < NSTAGE; ++s) tags[s] = 0xffffffffu;
    init_wait_state(cta_abort, p.wait_us);
    *stall_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // Launched as the programmatic dependent of a decode step's append (see
  // launch_tc), this grid may start while the append runs: wait for it to
  // complete before reading the pool or the large-scale flag it writes.
  // Without that launch attribute this returns at once.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int it0 = p.cta_off[blockIdx.x], it1 = p.cta_off[blockIdx.x + 1];
  const int Hkv = p.Hkv;
  const int rounds = p.hg / HPR;

  if (warp >= NCW) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    // Testing only (the pool's kDevTestStall word): an otherwise idle warp of
    // CTA 0 waits for a word that nothing raises, so that its bounded wait
    // runs out (error flag set; the launch still ends, its outputs not valid).
    if (warp == NCW + 1 && blockIdx.x == 0 && lane == 0 &&
        reinterpret_cast<volatile const int*>(p.err)[kDevTestStall] != 0)
      wait_count(stall_word, 1u, cta_abort, p.err);
    if (warp != NCW) return;
    // ---------------- producer ----------------
    // The lanes fetch an item's block ids together (one coalesced load per 32
    // blocks); lane 0 issues the bulk copies with no dependent global load in
    // the issue loop.
    // The next item's record, unit and first 32 block ids are fetched while
    // this item's copies are issued (one step per issued sub-block), so that
    // the chain item -> unit -> block table never idles the copy engine
    // between items.
    const int64_t blk_stride = (int64_t)p.L * Hkv * p.page_bytes;
    constexpr int SPB = SubGeom<D, NG, FMT>::SPB;
    auto first_blocks = [&](const AttnItem& itm, const AttnUnit& u) {
      const int b0 = itm.sb_begin / SPB;
      const int nblk = (itm.sb_end - 1) / SPB - b0 + 1;
      int bi = b0 + lane;
      if (p.ring > 0) bi %= p.ring;
      return lane < nblk ? p.bt[(int64_t)u.si * p.bt_stride + bi] : 0;
    };
    if constexpr (SEL || FMT == kFmtInt4) {
      produce_wide<D, NG, NCW, R, NSTAGE, FMT, SEL>(p, stages, bar_base, cta_abort, tags, lane, it0, it1, rounds);
      return;
    }
    AttnItem item_n{};
    AttnUnit un_n{};
    int blk_n = 0;
    if (it0 < it1) {
      item_n = p.items[it0];
      un_n = p.units[item_n.unit];
      blk_n = first_blocks(item_n, un_n);
    }
    uint32_t J = 0;
    for (int it = it0; it < it1; ++it) {
      const AttnItem item = item_n;
      const AttnUnit un = un_n;
      const int blk_first = blk_n;
      const bool more = it + 1 < it1;
      if (more) item_n = p.items[it + 1];
      int pf = more ? 0 : 2;  // 0: next record requested, 1: its unit, 2: its block ids
      auto prefetch_step = [&]() {
        if (pf == 0) {
          un_n = p.units[item_n.unit];
          pf = 1;
        } else if (pf == 1) {
          blk_n = first_blocks(item_n, un_n);
          pf = 2;
        }
      };
      const int32_t* bt = p.bt + (int64_t)un.si * p.bt_stride;
      const int n_sb = item.sb_end - item.sb_begin;
      const int b0 = item.sb_begin / SPB;
      const int nblk = (item.sb_end - 1) / SPB - b0 + 1;
      for (int rd = 0; rd < rounds; ++rd) {
        const uint8_t* layer_base =
            p.pool + ((int64_t)un.layer * Hkv + item.h0 + rd * HPR) * p.page_bytes;
        for (int c0 = 0; c0 < nblk; c0 += 32) {
          int bi = b0 + c0 + lane;
          if (p.ring > 0) bi %= p.ring;
          const int blk = c0 == 0 ? blk_first : (c0 + lane < nblk) ? bt[bi] : 0;
          const int jlo = max(item.sb_begin, (b0 + c0) * SPB);
          const int jhi = min(item.sb_end, (b0 + c0 + 32) * SPB);
          for (int j = jlo; j < jhi; ++j) {
            const int b = __shfl_sync(0xffffffffu, blk, j / SPB - b0 - c0);
            if (lane == 0) {
              const uint8_t* sb_src = layer_base + (int64_t)b * blk_stride + (int64_t)(j % SPB) * SB;
              for (int hr = 0; hr < HPR; ++hr) {
                const uint32_t Jh = J + (uint32_t)(j - item.sb_begin) * HPR + hr;
                const uint32_t stage = Jh % NSTAGE;
                if (Jh >= (uint32_t)NSTAGE)
                  mbar_wait(bar_base + 8 * (NSTAGE + stage), ((Jh / NSTAGE) - 1) & 1, cta_abort,
                            p.err);
                const uint32_t full = bar_base + 8 * stage;
                tags[stage] = Jh;  // released by the arrive below
                mbar_expect_tx(full, SB);
                bulk_g2s(smem_u32(stages + (size_t)stage * SB), sb_src + (int64_t)hr * p.page_bytes,
                         SB, full);
              }
            }
            if (pf < 2) prefetch_step();
          }
        }
        J += (uint32_t)n_sb * HPR;
      }
      while (pf < 2) prefetch_step();
    }
    return;
  }

  // ---------------- consumers ----------------
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  if constexpr (FMT == kFmtInt4)
    attn_consume4<D, NG, NCW, R, NSTAGE, QT, SEL>(p, smem, stages, bar_base, cta_abort, tags, warp, lane, it0, it1,
                                                  rounds);
  else if (FMT == kFmtInt8 && *reinterpret_cast<volatile const int*>(p.large_scale) != 0)
    attn_consume<D, NG, NCW, R, NSTAGE, FMT, false, QT, SEL>(p, smem, stages, bar_base, cta_abort, tags, warp, lane,
                                                         it0, it1, rounds);
  else
    attn_consume<D, NG, NCW, R, NSTAGE, FMT, true, QT, SEL>(p, smem, stages, bar_base, cta_abort, tags, warp,
                                                        lane, it0, it1, rounds);
}

template <int D, int NG, int NCW, int R, int FMT, int QT = 1, bool SEL = false>
cudaError_t launch_tc(const AttnParams& p, int grid, cudaStream_t stream) {
  constexpr int NSTAGE = stages_for<D, NG, NCW, R, FMT>();
  using SM = AttnSmem<D, NG, NCW, R, NSTAGE, FMT>;
  static_assert(NSTAGE >= 4, "too few stages");
  static_assert(SM::TOTAL <= 232448, "shared memory budget");
  // the shared-memory opt-in is a per-device attribute: set it once per device
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    // setmaxnreg.inc waits until the producer's released registers cover it:
    // refuse to launch a build whose register count would not balance
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, attn_tc_kernel<D, NG, NCW, R, NSTAGE, FMT, QT, SEL>);
    if (e != cudaSuccess) return e;
    if (fa.numRegs * (NCW + 4) * 32 < 128 * kProducerRegs + NCW * 32 * kConsumerRegs)
      return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(attn_tc_kernel<D, NG, NCW, R, NSTAGE, FMT, QT, SEL>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit);
  }
  if (p.pdl) {
    // programmatic dependent of the append launched just before it
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((NCW + 4) * 32);
    cfg.dynamicSmemBytes = SM::TOTAL;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_tc_kernel<D, NG, NCW, R, NSTAGE, FMT, QT, SEL>, p);
  }
  attn_tc_kernel<D, NG, NCW, R, NSTAGE, FMT, QT, SEL><<<grid, (NCW + 4) * 32, SM::TOTAL, stream>>>(p);
  return cudaGetLastError();
}

template <int D, int NG, int NCW, int FMT = kFmtInt8, bool SEL = false>
cudaError_t launch_tc_r(const AttnParams& p, int grid, cudaStream_t stream) {
  const int hpr = p.hg < NCW ? p.hg : NCW;
  if (NCW % hpr != 0 || p.hg % hpr != 0) return cudaErrorInvalidValue;
  cudaError_t e = cudaErrorInvalidValue;
  if (p.qt == 2) {  // two query tiles per unit: one warp per head only
    if constexpr (FMT != kFmtBf16 && D <= 128 && !SEL)
      if (hpr == NCW) e = launch_tc<D, NG, NCW, 1, FMT, 2>(p, grid, stream);
  } else switch (NCW / hpr) {
    case 1: e = launch_tc<D, NG, NCW, 1, FMT, 1, SEL>(p, grid, stream); break;
    case 2: e = launch_tc<D, NG, NCW, 2, FMT, 1, SEL>(p, grid, stream); break;
    case 4: e = launch_tc<D, NG, NCW, 4, FMT, 1, SEL>(p, grid, stream); break;
    case 8:
      if constexpr (NCW == 8) e = launch_tc<D, NG, NCW, 8, FMT, 1, SEL>(p, grid, stream);
      break;
    default: break;
  }
  if (e != cudaSuccess || p.n_split_units == 0 || p.split_ctr != nullptr) return e;
  return run_combine<D>(p, stream);
}

template <int D, int NG, int NCW, int R, int FMT>
int tc_desc(char* buf, size_t cap) {
  return snprintf(buf, cap, "attn_tc_kernel<%d,%d,%d,%d,%d,%d>", D, NG, NCW, R,
                  stages_for<D, NG, NCW, R, FMT>(), FMT);
}
template <int D, int NG, int FMT = kFmtInt8>
int tc_desc_r(const AttnParams& p, char* buf, size_t cap) {
  const int hpr = p.hg < 8 ? p.hg : 8;
  if (p.qt == 2)
    return snprintf(buf, cap, "attn_tc_kernel<%d,%d,8,1,%d,%d,2>", D, NG, stages_for<D, NG, 8, 1, FMT>(), FMT);
  if (hpr <= 0 || 8 % hpr != 0) return snprintf(buf, cap, "none");
  switch (8 / hpr) {
    case 1: return tc_desc<D, NG, 8, 1, FMT>(buf, cap);
    case 2: return tc_desc<D, NG, 8, 2, FMT>(buf, cap);
    case 4: return tc_desc<D, NG, 8, 4, FMT>(buf, cap);
    default: return tc_desc<D, NG, 8, 8, FMT>(buf, cap);
  }
}

}  // namespace
}  // namespace krill
