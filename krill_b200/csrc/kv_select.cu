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
template <int FMT>
__global__ void __launch_bounds__(kSumThreads) block_summary_kernel(uint8_t* __restrict__ pool, Geom geom,
                                                                    const SumItem* __restrict__ items) {
  __shared__ float mn_s[8][256], mx_s[8][256], red[4];
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
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = e >> 2, sh = (e & 1) * 16 + ((e >> 1) & 1) * 4;  // d = 4k + h + 2 * high nibble
        const float a = fmaf((float)((w[k] >> sh) & 15u), s.x, z.x);
        const float b = fmaf((float)((w[k] >> (sh + 8)) & 15u), s.y, z.y);
        float lo = fminf(a, b), hi = fmaxf(a, b);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        }
        if (r == 0) {
          mn_s[u][64 * hh + 16 * tig + e] = lo;
          mx_s[u][64 * hh + 16 * tig + e] = hi;
        }
      }
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
constexpr int kRegKeys = 16;             // keys a thread holds while it picks
constexpr uint32_t kForced = 0xffffffffu;  // above the key of every score

// Order-preserving key of a score, at least 1 (equal scores, +-0 included, get
// equal keys).
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
  uint32_t red[2][kSelWarps];          // double-buffered block reductions
  uint32_t cnt[kRegKeys][kSelWarps];   // per key round and warp: picked-for-sure | equal << 16
};

// Sum / min / max over the NW warps that pick (one: no barrier).
template <int NW, typename F>
__device__ __forceinline__ uint32_t pick_reduce(uint32_t x, PickSmem& sm, int& buf, int warp, int lane, F op) {
  if (NW == 1) return x;
  if (lane == 0) sm.red[buf][warp] = x;
  __syncthreads();
  x = sm.red[buf][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) x = op(x, sm.red[buf][w]);
  buf ^= 1;
  return x;
}

// The `want` largest keys (equal ones: the first) besides the forced ones, at
// most kRegKeys * 32 * NW of them, by bisection over the bits in which the keys
// differ, each thread holding its keys in registers; their indices to `out` in
// order. NW warps call it.
template <int NW>
__device__ __forceinline__ void pick_in_registers(const uint32_t* keys, int n, int want, int32_t* out, PickSmem& sm,
                                                  int warp, int lane) {
  constexpr int STEP = 32 * NW;
  const int at = warp * 32 + lane, rounds = (n + STEP - 1) / STEP;
  uint32_t k[kRegKeys], lo = 0xffffffffu, hi = 0u;
  int buf = 0;
#pragma unroll
  for (int j = 0; j < kRegKeys; ++j) {
    k[j] = 0u;
    if (j < rounds) {
      if (at + j * STEP < n) k[j] = keys[at + j * STEP];
      if (k[j] != 0u && k[j] != kForced) {
        lo = min(lo, k[j]);
        hi = max(hi, k[j]);
      }
    }
  }
  lo = pick_reduce<NW>(__reduce_min_sync(0xffffffffu, lo), sm, buf, warp, lane, [](uint32_t a, uint32_t b) { return min(a, b); });
  hi = pick_reduce<NW>(__reduce_max_sync(0xffffffffu, hi), sm, buf, warp, lane, [](uint32_t a, uint32_t b) { return max(a, b); });
  // K: the largest threshold with at least `want` keys in [K, kForced)
  uint32_t K = kForced - 1u;
  int above = 0;
  if (want > 0) {
    const int top = 32 - __clz(lo ^ hi);  // bits that differ
    K = top >= 32 ? 0u : lo >> top << top;
    for (int bit = top - 1; bit >= 0; --bit) {
      const uint32_t cand = K | (1u << bit);
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < kRegKeys; ++j)
        if (j < rounds) c += k[j] >= cand && k[j] != kForced ? 1u : 0u;
      c = pick_reduce<NW>(__reduce_add_sync(0xffffffffu, c), sm, buf, warp, lane, [](uint32_t a, uint32_t b) { return a + b; });
      if ((int)c >= want) K = cand;
      if ((int)c == want) break;  // exactly the keys from K on
    }
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < kRegKeys; ++j)
      if (j < rounds) c += k[j] > K && k[j] != kForced ? 1u : 0u;
    above = (int)pick_reduce<NW>(__reduce_add_sync(0xffffffffu, c), sm, buf, warp, lane, [](uint32_t a, uint32_t b) { return a + b; });
  }
  const int need = want - above;  // of the keys equal to K, the first ones
  // positions: keys above K (forced ones among them) before, and equal ones
  uint32_t mg[kRegKeys], me[kRegKeys];
#pragma unroll
  for (int j = 0; j < kRegKeys; ++j)
    if (j < rounds) {
      mg[j] = __ballot_sync(0xffffffffu, k[j] > K);
      me[j] = __ballot_sync(0xffffffffu, k[j] == K && K != 0u);
      if (NW > 1 && lane == 0) sm.cnt[j][warp] = __popc(mg[j]) | (__popc(me[j]) << 16);
    }
  if (NW > 1) __syncthreads();
  const uint32_t below = (1u << lane) - 1u;
  int g0 = 0, e0 = 0;
#pragma unroll
  for (int j = 0; j < kRegKeys; ++j)
    if (j < rounds) {
      int gb = g0, eb = e0;
      if (NW == 1) {
        g0 += __popc(mg[j]);
        e0 += __popc(me[j]);
      } else {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const uint32_t c = sm.cnt[j][w];
          if (w < warp) {
            gb += c & 0xffff;
            eb += c >> 16;
          }
          g0 += c & 0xffff;
          e0 += c >> 16;
        }
      }
      gb += __popc(mg[j] & below);
      eb += __popc(me[j] & below);
      const bool gt = (mg[j] >> lane) & 1u, eq = (me[j] >> lane) & 1u;
      if (gt || (eq && eb < need)) out[gb + min(eb, need)] = at + j * STEP;
    }
}

// The same for any number of keys, read again in every round.
__device__ __forceinline__ void pick_in_memory(const uint32_t* keys, int n, int budget, int32_t* out, PickSmem& sm,
                                               int tid, int warp, int lane) {
  int buf = 0;
  auto add = [](uint32_t a, uint32_t b) { return a + b; };
  auto count = [&](uint32_t from) {
    uint32_t c = 0;
    for (int i = tid; i < n; i += kSelThreads) c += keys[i] >= from ? 1u : 0u;
    return (int)pick_reduce<kSelWarps>(__reduce_add_sync(0xffffffffu, c), sm, buf, warp, lane, add);
  };
  uint32_t K = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = K | (1u << bit);
    if (count(cand) >= budget) K = cand;
  }
  const int need = budget - (K == kForced ? 0 : count(K + 1u));
  int gt_before = 0, eq_before = 0;
  for (int i0 = 0; i0 < n; i0 += kSelThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < n ? keys[i] : 0u;
    const bool gt = i < n && k > K, eq = i < n && k == K;
    const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) sm.red[buf][warp] = __popc(mg) | (__popc(me) << 16);
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kSelWarps; ++w) {
      if (w < warp) before += sm.red[buf][w];
      total += sm.red[buf][w];
    }
    const uint32_t below = (1u << lane) - 1u;
    const int gb = gt_before + (before & 0xffff) + __popc(mg & below);
    const int eb = eq_before + (before >> 16) + __popc(me & below);
    if (gt || (eq && eb < need)) out[gb + min(eb, need)] = i;
    gt_before += total & 0xffff;
    eq_before += total >> 16;
    buf ^= 1;
  }
}

// One cluster of CTAs per (unit, kv head). The cluster's warps score 16 blocks
// at a time against the head's (at most 8) query heads in one chain of int8
// MMAs (rows = blocks, columns = query heads, K = the 2 D summary bytes; the
// byte order along K is permuted alike on both sides, so that a lane's operand
// is 16 consecutive bytes); the keys go to the first CTA's shared memory (or
// to scratch, for sequences of more blocks than fit), which picks: up to 512
// blocks in one warp without barriers, up to 2048 in four, more by reading the
// keys again for each bit.
template <int D>
__global__ void __launch_bounds__(kSelThreads) select_blocks_kernel(SelectParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ uint32_t keys_smem[];
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
  // ---- the query heads in whole numbers, one warp per head ----
#pragma unroll
  for (int hq = warp; hq < 8; hq += kSelWarps) {
    float x[D / 32], mx = 0.f;
    const int64_t q0 = ((int64_t)qo_row * p.Hq + (int64_t)h * g + hq) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      x[i] = hq < g ? load_in(p.q, q0 + lane + 32 * i, p.q_dtype) : 0.f;
      if (!isfinite(x[i])) x[i] = 0.f;
      mx = fmaxf(mx, fabsf(x[i]));
    }
    // (non-negative floats order like their bits)
    mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
    const float tau = __fdiv_rn(mx, 127.0f);
    const float inv = tau > 0.f ? __fdiv_rn(1.0f, tau) : 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int a = max(-127, min(127, __float2int_rn(__fmul_rn(x[i], inv))));
      qa[hq][lane + 32 * i] = (int8_t)a;
      qa[hq][D + lane + 32 * i] = (int8_t)abs(a);
    }
    if (lane == 0) tau_s[hq] = tau;
  }
  __syncthreads();
  const int r = lane >> 2, tig = lane & 3;
  constexpr int NC = 2 * D / 64;
  uint4 bq[NC];  // column r = query head r
#pragma unroll
  for (int c = 0; c < NC; ++c) bq[c] = *reinterpret_cast<const uint4*>(&qa[r][64 * c + 16 * tig]);
  const float tau0 = tau_s[2 * tig], tau1 = tau_s[2 * tig + 1];
  const bool has0 = 2 * tig < g, has1 = 2 * tig + 1 < g;
  uint32_t* keys = p.scratch ? p.scratch + (int64_t)uid * p.scratch_stride
                             : cluster.map_shared_rank(keys_smem, 0);
  const int32_t* bt = p.bt + (int64_t)si * p.bt_stride;
  const uint8_t* base = p.pool + ((int64_t)layer * p.Hkv + h) * p.page_bytes + p.sum_off;
  const int64_t blk_stride = (int64_t)p.L * p.Hkv * p.page_bytes;
  const int spb_bytes = p.spb * 2 * D;
#pragma unroll 2
  for (int i0 = lo + 16 * (rank * kSelWarps + warp); i0 < hi; i0 += 16 * CL * kSelWarps) {
    const int ra = min(i0 + r, hi - 1), rb = min(i0 + r + 8, hi - 1);
    const uint8_t* pa = base + (int64_t)__ldg(bt + ra / p.spb) * blk_stride;
    const uint8_t* pb = base + (int64_t)__ldg(bt + rb / p.spb) * blk_stride;
    const uint4* wa = reinterpret_cast<const uint4*>(pa + (ra % p.spb) * 2 * D) + tig;
    const uint4* wb = reinterpret_cast<const uint4*>(pb + (rb % p.spb) * 2 * D) + tig;
    const float sa = __ldg(reinterpret_cast<const float*>(pa + spb_bytes) + ra % p.spb);
    const float sb = __ldg(reinterpret_cast<const float*>(pb + spb_bytes) + rb % p.spb);
    uint4 xa[NC], xb[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      xa[c] = __ldg(wa + 4 * c);
      xb[c] = __ldg(wb + 4 * c);
    }
    int acc[4] = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      imma16832(acc, xa[c].x, xb[c].x, xa[c].y, xb[c].y, bq[c].x, bq[c].y);
      imma16832(acc, xa[c].z, xb[c].z, xa[c].w, xb[c].w, bq[c].z, bq[c].w);
    }
    float va = -INFINITY, vb = -INFINITY;
    if (has0) {
      va = __fmul_rn(__fmul_rn((float)acc[0], sa), tau0);
      vb = __fmul_rn(__fmul_rn((float)acc[2], sb), tau0);
    }
    if (has1) {
      va = fmaxf(va, __fmul_rn(__fmul_rn((float)acc[1], sa), tau1));
      vb = fmaxf(vb, __fmul_rn(__fmul_rn((float)acc[3], sb), tau1));
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
  if (n <= 32 * kRegKeys) {
    if (warp == 0) pick_in_registers<1>(keys, n, want, out, sm, 0, lane);
  } else if (n <= kSelThreads * kRegKeys) {
    pick_in_registers<kSelWarps>(keys, n, want, out, sm, warp, lane);
  } else {
    pick_in_memory(keys, n, p.budget, out, sm, tid, warp, lane);
  }
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
