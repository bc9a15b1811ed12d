// kv_select.cu — block summaries and the choice of the blocks that a query
// attends (block-sparse decode).
//
// Summary of a full sub-block of T tokens, per K channel d over its values:
//   mid_d = rint(((max + min) / 2) / sigma), half_d = rint(((max - min) / 2) / sigma)
// as int8, with sigma = max |k| / 127 (f32). A query head is rounded to whole
// numbers a_d of tau = max |q| / 127. Its score of a block is
//   (sum_d a_d mid_d + |a_d| half_d) * sigma * tau,
// an upper estimate of the largest q.k in the block; a kv head's score is the
// largest of its query heads'. The sum is a whole number, exact in any order,
// and the two products round once each, so that the choice does not depend on
// how the sum is split. Equal scores go to the lowest index.
#include <cooperative_groups.h>

#include "kv_device.cuh"

namespace krill {
namespace {

namespace cg = cooperative_groups;

constexpr int kSumThreads = 128;

// One CTA per (sub-block, kv head). min / max of the sub-block's K values per
// channel, partial over the threads' token subsets, joined in shared memory.
// Runs once for a sub-block, when it fills up: 19 us for 512 x 8 of 4 bits at
// head_dim 128, 30 us of 8 bits (20 and 37 MB: 3 and 6 us), beside 47 and 69 us
// for their append; bound by the latency of its steps.
template <int FMT>
__global__ void __launch_bounds__(kSumThreads) block_summary_kernel(uint8_t* __restrict__ pool, Geom geom,
                                                                    const SumItem* __restrict__ items) {
  __shared__ __align__(8) float mn_s[8][256], mx_s[8][256], red[4];
  const int D = geom.D, NG = geom.NG;
  const SumItem it = items[blockIdx.x / geom.Hkv];
  const int h = blockIdx.x % geom.Hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* page = pool + (((int64_t)it.block * geom.L + it.layer) * geom.Hkv + h) * geom.page_bytes;
  const uint8_t* sb = page + (int64_t)it.sub * geom.sb_bytes;
  int subsets;
  if (FMT == kFmtInt4) {
    // warp w takes token tile w; lane (r, tig) the tile's rows r and r + 8 and the
    // channels 16 tig .. + 15 of each run of 64
    subsets = 4;
    const int r = lane >> 2, tig = lane & 3, u = warp;
    for (int hh = 0; hh < D / 64; ++hh) {
      const int gi = 64 * hh / geom.G;
      const uint4 w4 = *reinterpret_cast<const uint4*>(sb + ((u * (D / 64) + hh) * 32 + lane) * 16);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      const float2 s = __half22float2(u2h(*reinterpret_cast<const uint32_t*>(sb + q4_meta(D, NG, 0, gi, 0) + (8 * r + 2 * u) * 2)));
      const float2 z = __half22float2(u2h(*reinterpret_cast<const uint32_t*>(sb + q4_meta(D, NG, 1, gi, 0) + (8 * r + 2 * u) * 2)));
      float lo[16], hi[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = e >> 2, sh = (e & 1) * 16 + ((e >> 1) & 1) * 4;  // d = 4k + h + 2 * high nibble
        const float a = fmaf((float)((w[k] >> sh) & 15u), s.x, z.x);
        const float b = fmaf((float)((w[k] >> (sh + 8)) & 15u), s.y, z.y);
        lo[e] = fminf(a, b);
        hi[e] = fmaxf(a, b);
      }
      // over the eight rows: at each step a lane keeps half of its channels and
      // hands the other half over, so that it ends with channels 2r, 2r + 1
#pragma unroll
      for (int n = 8; n >= 2; n /= 2) {
        const bool up = (r & (n / 2)) != 0;
#pragma unroll
        for (int e = 0; e < n; ++e) {
          const float l = __shfl_xor_sync(0xffffffffu, up ? lo[e] : lo[e + n], 2 * n);
          const float m = __shfl_xor_sync(0xffffffffu, up ? hi[e] : hi[e + n], 2 * n);
          lo[e] = fminf(up ? lo[e + n] : lo[e], l);
          hi[e] = fmaxf(up ? hi[e + n] : hi[e], m);
        }
      }
      const int d = 64 * hh + 16 * tig + 2 * r;
      *reinterpret_cast<float2*>(&mn_s[u][d]) = make_float2(lo[0], lo[1]);
      *reinterpret_cast<float2*>(&mx_s[u][d]) = make_float2(hi[0], hi[1]);
    }
  } else {
    // D/4 threads cover a token's channels, four each
    const int per = D / 4, c4 = tid % per, t0 = tid / per;
    subsets = kSumThreads / per;
    float lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
    const int gi = 4 * c4 / geom.G;
    for (int t = t0; t < geom.subt; t += subsets) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(sb + sb_kcode(D, t, 4 * c4));
      const __half s = *reinterpret_cast<const __half*>(sb + sb_meta(D, NG, 0, gi, t));
      const __half z = *reinterpret_cast<const __half*>(sb + sb_meta(D, NG, 1, gi, t));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __half2float(__hadd_rn(__hmul_rn(__ushort2half_rn((w >> (8 * e)) & 255u), s), z));
        lo[e] = fminf(lo[e], x);
        hi[e] = fmaxf(hi[e], x);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mn_s[t0][4 * c4 + e] = lo[e];
      mx_s[t0][4 * c4 + e] = hi[e];
    }
  }
  __syncthreads();
  float lo[2], hi[2], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = tid + i * kSumThreads;
    if (d < D) {
      lo[i] = mn_s[0][d];
      hi[i] = mx_s[0][d];
      for (int k = 1; k < subsets; ++k) {
        lo[i] = fminf(lo[i], mn_s[k][d]);
        hi[i] = fmaxf(hi[i], mx_s[k][d]);
      }
      amax = fmaxf(amax, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
    }
  }
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if (lane == 0) red[warp] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float sigma = __fdiv_rn(amax, 127.0f);
  const float inv = sigma > 0.f ? __fdiv_rn(1.0f, sigma) : 0.f;
  int8_t* out = reinterpret_cast<int8_t*>(page + geom.sum_off) + (int64_t)it.sub * 2 * D;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = tid + i * kSumThreads;
    if (d < D) {
      const float mid = __fmul_rn(__fmul_rn(__fadd_rn(hi[i], lo[i]), 0.5f), inv);
      const float half = __fmul_rn(__fmul_rn(__fsub_rn(hi[i], lo[i]), 0.5f), inv);
      out[d] = (int8_t)max(-127, min(127, __float2int_rn(mid)));
      out[D + d] = (int8_t)max(-127, min(127, __float2int_rn(half)));
    }
  }
  if (tid == 0) *reinterpret_cast<float*>(page + geom.sum_off + (int64_t)geom.spb * 2 * D + 4 * it.sub) = sigma;
}

constexpr int kSelThreads = 128, kSelWarps = kSelThreads / 32;
constexpr uint32_t kForced = 0xffffffffu;  // above the key of every score

// Order-preserving key of a score, at least 1 and below kForced (equal scores,
// +-0 included, get equal keys).
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
  if (isnan(x)) return 1u;
  return (b & 0x80000000u) ? max(~b, 1u) : (b | 0x80000000u);
}

__device__ __forceinline__ void imma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct PickSmem {
  uint32_t bins[256];
  uint32_t lo[kSelWarps], hi[kSelWarps];
  uint32_t gt[kSelWarps], eq[kSelWarps];  // per warp: keys above the threshold, equal to it
  uint32_t bin, above, in_bin;
};

// Up to 32 * KPT keys by one warp, held in registers: bisection over the bits in
// which the scored keys differ, until exactly `want` keys are above the
// threshold (after about log2 n steps) or all bits are found; then the order by
// ballots. No barrier; the CTA's other warps are done.
template <int KPT>
__device__ __forceinline__ void pick_in_warp(const uint32_t* keys, int n, int want, int32_t* out, int lane) {
  uint32_t k[KPT], lo = kForced, hi = 0u;
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    const int i = 32 * j + lane;
    k[j] = i < n ? keys[i] : 0u;
    if (k[j] != 0u && k[j] != kForced) {
      lo = min(lo, k[j]);
      hi = max(hi, k[j]);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  uint32_t c = 0u, forced = 0u;
#pragma unroll
  for (int j = 0; j < KPT; ++j) forced += k[j] == kForced ? 1u : 0u;
  forced = __reduce_add_sync(0xffffffffu, forced);
  const uint32_t target = (uint32_t)want + forced;  // keys to pick, forced ones among them
  uint32_t K = kForced - 1u;  // picked: keys > K, and of those equal to K the first `need`
  int need = 0;
  if (want > 0) {
    const int top = 32 - __clz(lo ^ hi);
    K = top >= 32 ? 0u : lo >> top << top;
    bool exact = false;
    for (int bit = top - 1; bit >= 0 && !exact; --bit) {
      const uint32_t cand = K | (1u << bit);
      c = 0u;
#pragma unroll
      for (int j = 0; j < KPT; ++j) c += k[j] >= cand ? 1u : 0u;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c >= target) K = cand;
      exact = c == target;
    }
    if (exact) {
      K -= 1u;
    } else {
      c = 0u;
#pragma unroll
      for (int j = 0; j < KPT; ++j) c += k[j] > K ? 1u : 0u;
      need = (int)(target - __reduce_add_sync(0xffffffffu, c));
    }
  }
  const uint32_t below = (1u << lane) - 1u;
  int gb = 0, eb = 0;
#pragma unroll
  for (int j = 0; j < KPT; ++j) {
    const bool gt = k[j] > K, eq = k[j] == K && k[j] != 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
    const int g = gb + __popc(mg & below), e = eb + __popc(me & below);
    if (gt || (eq && e < need)) out[g + min(e, need)] = 32 * j + lane;
    gb += __popc(mg);
    eb += __popc(me);
  }
}

// Any number of keys: the threshold is found eight bits at a time, from the
// highest bit in which the scored keys differ, by histograms over the keys that
// share the bits found so far; usually two passes leave as many keys as are
// still wanted. `want`: keys to pick besides the forced ones.
__device__ __forceinline__ void pick_by_digits(const uint32_t* keys, int n, int want, int32_t* out, PickSmem& sm,
                                               int tid, int warp, int lane) {
  uint32_t lo = kForced, hi = 0u;
#pragma unroll 4
  for (int i = tid; i < n; i += kSelThreads) {
    const uint32_t k = keys[i];
    if (k != kForced) {
      lo = min(lo, k);
      hi = max(hi, k);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    sm.lo[warp] = lo;
    sm.hi[warp] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w) {
    lo = min(lo, sm.lo[w]);
    hi = max(hi, sm.hi[w]);
  }
  // picked: keys > K, and of those equal to K the first `need`
  uint32_t K = kForced - 1u;
  int need = 0;
  if (want > 0) {
    int rem = 32 - __clz(lo ^ hi);  // bits not found yet
    uint32_t P = rem >= 32 ? 0u : lo >> rem << rem;
    need = want;
    bool all = false;  // every key from P on is picked
    while (rem > 0 && !all) {
      const int width = min(8, rem), shift = rem - width;
      for (int i = tid; i < 256; i += kSelThreads) sm.bins[i] = 0u;
      __syncthreads();
#pragma unroll 4
      for (int i = tid; i < n; i += kSelThreads) {
        const uint32_t k = keys[i];
        if (k != kForced && (rem >= 32 || k >> rem == P >> rem)) atomicAdd(&sm.bins[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {  // lane l: bins 8 (31 - l) .. + 7, so that lower lanes hold larger keys
        uint32_t c[8], sum = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = sm.bins[8 * (31 - lane) + e];
          sum += c[e];
        }
        uint32_t upto = sum;  // keys in this lane's bins and above
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
          if (lane >= off) upto += o;
        }
        uint32_t above = upto - sum;
        if ((int)above < need && (int)upto >= need) {  // the threshold's bin is one of this lane's
#pragma unroll
          for (int e = 7; e >= 0; --e) {
            if ((int)above < need && (int)(above + c[e]) >= need) {
              sm.bin = 8 * (31 - lane) + e;
              sm.above = above;
              sm.in_bin = c[e];
            }
            above += c[e];
          }
        }
      }
      __syncthreads();
      P |= sm.bin << shift;
      need -= (int)sm.above;
      all = (int)sm.in_bin == need;
      rem = shift;
    }
    K = all && P > 0u ? P - 1u : P;  // (keys are at least 1: K = 0 takes every one)
    if (all) need = 0;
  }
  // order: each warp a contiguous quarter
  const int per = (n + kSelThreads - 1) / kSelThreads * 32, i0 = warp * per, i1 = min(n, i0 + per);
  uint32_t ng = 0u, ne = 0u;
#pragma unroll 4
  for (int i = i0; i < i1; i += 32) {
    const uint32_t k = i + lane < i1 ? keys[i + lane] : 0u;
    ng += __popc(__ballot_sync(0xffffffffu, k > K));
    ne += __popc(__ballot_sync(0xffffffffu, k == K && k != 0u));
  }
  if (lane == 0) {
    sm.gt[warp] = ng;
    sm.eq[warp] = ne;
  }
  __syncthreads();
  int gb = 0, eb = 0;
#pragma unroll
  for (int w = 0; w < kSelWarps; ++w)
    if (w < warp) {
      gb += sm.gt[w];
      eb += sm.eq[w];
    }
  const uint32_t below = (1u << lane) - 1u;
#pragma unroll 4
  for (int i = i0; i < i1; i += 32) {
    const uint32_t k = i + lane < i1 ? keys[i + lane] : 0u;
    const bool gt = k > K, eq = k == K && k != 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
    const int g = gb + __popc(mg & below), e = eb + __popc(me & below);
    if (gt || (eq && e < need)) out[g + min(e, need)] = i + lane;
    gb += __popc(mg);
    eb += __popc(me);
  }
}

// One cluster of CTAs per (unit, kv head). The cluster's warps score 16 blocks
// at a time against the head's (at most 8) query heads in one chain of int8
// MMAs (rows = blocks, columns = query heads, K = the 2 D summary bytes; the
// byte order along K is permuted alike on both sides, so that a lane's operand
// is 16 consecutive bytes); the keys go to the first CTA's shared memory (or
// to scratch, for sequences of more blocks than fit), which picks. Latency
// bounds it: the summaries of a warp's next 16 blocks are fetched while it
// works on the ones before (the first while the query is rounded), their block
// ids a step earlier. At head_dim 128: 11.2 us for 8 layers of 32 sequences of
// 512 to 8192 tokens, 8 heads (28 MB, 4.3 us), 13.3 us for 4 layers of 2 of
// 131072 tokens, 4 heads (17 MB, 2.6 us).
template <int D>
__global__ void __launch_bounds__(kSelThreads) select_blocks_kernel(SelectParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(16) uint32_t keys_smem[];
  __shared__ __align__(16) int8_t qa[8][2 * D];
  __shared__ float tau_s[8];
  __shared__ PickSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int uid = blockIdx.x / CL, ui = uid / p.Hkv, h = uid % p.Hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const AttnUnit* unit = p.units + ui;
  const int si = unit->si, layer = unit->layer, qo_row = unit->qo_row;
  const int n = (unit->t_hi + p.T - 1) / p.T;
  int32_t* out = p.sel + (int64_t)uid * p.budget;
  if (n <= p.budget) {  // every block
    if (rank == 0)
      for (int i = tid; i < p.budget; i += kSelThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int g = p.g, lo = p.first, hi = n - p.last;  // scored blocks [lo, hi)
  const int r = lane >> 2, tig = lane & 3;
  constexpr int NC = 2 * D / 64;
  const int32_t* bt = p.bt + (int64_t)si * p.bt_stride;
  const uint8_t* base = p.pool + ((int64_t)layer * p.Hkv + h) * p.page_bytes + p.sum_off;
  const int64_t blk_stride = (int64_t)p.L * p.Hkv * p.page_bytes;
  const int spb_bytes = p.spb * 2 * D, step = 16 * CL * kSelWarps;
  uint4 xa[NC], xb[NC];
  float sa = 0.f, sb = 0.f;
  auto block_of = [&](int i) { return __ldg(bt + min(i, hi - 1) / p.spb); };
  auto fetch = [&](int i0, int ba, int bb) {
    const int ra = min(i0 + r, hi - 1) % p.spb, rb = min(i0 + r + 8, hi - 1) % p.spb;
    const uint8_t* pa = base + (int64_t)ba * blk_stride;
    const uint8_t* pb = base + (int64_t)bb * blk_stride;
    const uint4* wa = reinterpret_cast<const uint4*>(pa + ra * 2 * D) + tig;
    const uint4* wb = reinterpret_cast<const uint4*>(pb + rb * 2 * D) + tig;
    sa = __ldg(reinterpret_cast<const float*>(pa + spb_bytes) + ra);
    sb = __ldg(reinterpret_cast<const float*>(pb + spb_bytes) + rb);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      xa[c] = __ldg(wa + 4 * c);
      xb[c] = __ldg(wb + 4 * c);
    }
  };
  int i0 = lo + 16 * (rank * kSelWarps + warp);
  int ba = block_of(i0 + r), bb = block_of(i0 + r + 8);
  int ba_n = block_of(i0 + step + r), bb_n = block_of(i0 + step + r + 8);
  // The first CTA's shared memory may be written once that CTA is known to have
  // started: every CTA arrives here and waits before its first key, with the
  // rounding of the query between. (The return above is the whole cluster's.)
  if (CL > 1) cluster.barrier_arrive();
  // ---- the query heads in whole numbers, one warp per head (two rounds) ----
  constexpr int QR = 8 / kSelWarps;
  float x[QR][D / 32];
#pragma unroll
  for (int j = 0; j < QR; ++j) {
    const int hq = warp + j * kSelWarps;
    const int64_t q0 = ((int64_t)qo_row * p.Hq + (int64_t)h * g + hq) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x[j][i] = hq < g ? load_in(p.q, q0 + lane + 32 * i, p.q_dtype) : 0.f;
  }
  if (i0 < hi) fetch(i0, ba, bb);
#pragma unroll
  for (int j = 0; j < QR; ++j) {
    const int hq = warp + j * kSelWarps;
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if (!isfinite(x[j][i])) x[j][i] = 0.f;
      mx = fmaxf(mx, fabsf(x[j][i]));
    }
    // (non-negative floats order like their bits)
    mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
    const float tau = __fdiv_rn(mx, 127.0f);
    const float inv = tau > 0.f ? __fdiv_rn(1.0f, tau) : 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int a = max(-127, min(127, __float2int_rn(__fmul_rn(x[j][i], inv))));
      qa[hq][lane + 32 * i] = (int8_t)a;
      qa[hq][D + lane + 32 * i] = (int8_t)abs(a);
    }
    if (lane == 0) tau_s[hq] = tau;
  }
  __syncthreads();
  const float tau0 = tau_s[2 * tig], tau1 = tau_s[2 * tig + 1];
  const bool has0 = 2 * tig < g, has1 = 2 * tig + 1 < g;
  uint32_t* keys = p.scratch ? p.scratch + (int64_t)uid * p.scratch_stride
                             : cluster.map_shared_rank(keys_smem, 0);
  if (CL > 1) cluster.barrier_wait();
  for (; i0 < hi; i0 += step) {
    int acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; ++c) {  // column r = query head r
      const uint4 bq = *reinterpret_cast<const uint4*>(&qa[r][64 * c + 16 * tig]);
      imma16832(acc, xa[c].x, xb[c].x, xa[c].y, xb[c].y, bq.x, bq.y);
      imma16832(acc, xa[c].z, xb[c].z, xa[c].w, xb[c].w, bq.z, bq.w);
    }
    const float ta = sa, tb = sb;
    if (i0 + step < hi) {
      fetch(i0 + step, ba_n, bb_n);
      ba_n = block_of(i0 + 2 * step + r);
      bb_n = block_of(i0 + 2 * step + r + 8);
    }
    float va = -INFINITY, vb = -INFINITY;
    if (has0) {
      va = __fmul_rn(__fmul_rn((float)acc[0], ta), tau0);
      vb = __fmul_rn(__fmul_rn((float)acc[2], tb), tau0);
    }
    if (has1) {
      va = fmaxf(va, __fmul_rn(__fmul_rn((float)acc[1], ta), tau1));
      vb = fmaxf(vb, __fmul_rn(__fmul_rn((float)acc[3], tb), tau1));
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      va = fmaxf(va, __shfl_xor_sync(0xffffffffu, va, off));
      vb = fmaxf(vb, __shfl_xor_sync(0xffffffffu, vb, off));
    }
    if (tig == 0) {
      if (i0 + r < hi) keys[i0 + r] = score_key(va);
      if (i0 + r + 8 < hi) keys[i0 + r + 8] = score_key(vb);
    }
  }
  if (rank == 0)
    for (int i = tid; i < lo + p.last; i += kSelThreads) keys[i < lo ? i : hi + i - lo] = kForced;
  if (CL > 1) {
    if (p.scratch) __threadfence();
    cluster.sync();  // every CTA's keys are in place; only rank 0 goes on
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  if (!p.scratch) keys = keys_smem;
  const int want = p.budget - p.first - p.last;
  if (n > 256) pick_by_digits(keys, n, want, out, sm, tid, warp, lane);
  else if (warp > 0) return;
  else if (n > 128) pick_in_warp<8>(keys, n, want, out, lane);
  else pick_in_warp<4>(keys, n, want, out, lane);
}

template <int D>
cudaError_t launch_select_d(const SelectParams& p, int n_units, int64_t max_n, int num_sms, cudaStream_t stream) {
  const int64_t pairs = (int64_t)n_units * p.Hkv;
  // CTAs per (unit, head): enough to have two CTAs per SM, while each still
  // has 64 blocks (one pass of its 4 warps) to score
  int cl = 1;
  while (cl < 8 && pairs * cl < 2 * num_sms && max_n / (2 * cl) >= 64) cl *= 2;
  if (pairs * cl > INT32_MAX) return cudaErrorInvalidValue;
  const size_t smem = p.scratch ? 0 : (size_t)max_n * 4;
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(select_blocks_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(kSelectSmemKeys * 4));
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * cl));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, select_blocks_kernel<D>, p);
}

}  // namespace

cudaError_t launch_summaries(const Geom& g, uint8_t* pool, const SumItem* d_items, int64_t n_items,
                             cudaStream_t stream) {
  if (n_items == 0) return cudaSuccess;
  if (n_items * g.Hkv > INT32_MAX) return cudaErrorInvalidValue;
  const unsigned blocks = (unsigned)(n_items * g.Hkv);
  if (g.fmt == kFmtInt4) block_summary_kernel<kFmtInt4><<<blocks, kSumThreads, 0, stream>>>(pool, g, d_items);
  else block_summary_kernel<kFmtInt8><<<blocks, kSumThreads, 0, stream>>>(pool, g, d_items);
  return cudaGetLastError();
}

cudaError_t launch_select(const Geom& g, const SelectParams& p, int n_units, int64_t max_n, int num_sms,
                          cudaStream_t stream) {
  if (g.D == 64) return launch_select_d<64>(p, n_units, max_n, num_sms, stream);
  if (g.D == 128) return launch_select_d<128>(p, n_units, max_n, num_sms, stream);
  if (g.D == 256) return launch_select_d<256>(p, n_units, max_n, num_sms, stream);
  return cudaErrorInvalidValue;
}

}  // namespace krill
