// The whole layer for a few tokens in two launches: router, top-k, and the experts hit, weights in bf16 or in e4m3 with
// 128 x 128 scales (the activations keep 16 bits: a step of a few tokens is bound by the bytes of the weights).
//
//   layer_router_kernel   logits = x Wr^T + b in fp32; the token rows as padded 16-bit operands; counters to zero
//   layer_experts_kernel  cooperative, one CTA per SM: top-k and lists of rows (each CTA for itself), gate_up with GLU,
//                         grid barrier, down, grid barrier, weighted sum of a token's K rows in slot order
//
// Bound by HBM where the weights of the experts hit exceed some 50 MB, by latency below.  What carries it:
//  * The weights do not depend on anything but the routing, so every warp streams its tiles of 8 KB through a ring of its
//    own (TMA, 24 tiles = 192 KB in flight per SM), on across units and across the grid barrier: HBM works through the
//    reductions, and when the activations are ready the first third of the down weights of a token already lies in
//    shared memory.
//  * Both phases are cut into equal shares of tiles, not of output columns: a unit (64 output columns of one expert,
//    the whole reduction) may be split over two CTAs, which meet in memory; no sum depends on who comes first.
//  * The products are m16n8k16 of mma.sync with the WEIGHT columns as M and up to eight rows as N: the tensor core
//    is far from busy, and a weight costs the same number of instructions for one row as for eight.  Within a tile the
//    reduction index is permuted (the same way for both operands), so that the rows come by 8- or 16-byte loads.
//
// Roundings: logits, softmax, sums and GLU are fp32.  e4m3 weights become f16 exactly, and what they multiply becomes f16
// times a power of two that brings the largest value of its row to 2^14: token rows exactly but for values under 2^-29 of
// the largest, activations to 11 bits (under 2^-28 of the largest, 2^-39 of it).  With bf16 weights an activation is
// the sum of two bf16 numbers, which take neighbouring columns of N.
#pragma once
#include <cuda_fp16.h>

#include "epilogues.cuh"
#include "tcgen05.cuh"

namespace yb {

constexpr int kLayerMaxT = 32, kLayerMaxS = 256, kLayerMaxK = 32;
constexpr int kLayerThreads = 256, kLayerWarps = 8;
constexpr int kLayerTileBytes = 8192, kLayerSlots = 3;             // ring per warp
constexpr int kLayerUnit = 64;                                     // output columns of a unit
constexpr int kLayerRows = 16;                                     // rows of an expert that share a pass over its weights
constexpr int kLayerRedPitch = 68;
constexpr int kLayerRingBytes = kLayerWarps * kLayerSlots * kLayerTileBytes;
constexpr int kLayerSmem = kLayerRingBytes + kLayerWarps * 8 * kLayerRedPitch * 4 + 1024;
constexpr int kLayerStatusBarrier = 8;                             // device status: a grid barrier gave up

struct LayerArgs {
  const __nv_bfloat16* x;            // [T, H]
  const __nv_bfloat16* router;       // [E, H]
  const __nv_bfloat16* router_bias;  // [E] or null
  const __nv_bfloat16 *bias_gu, *bias_dn;
  const float *scale_gu, *scale_dn;  // e4m3: strides below
  int64_t gu_b, gu_r, gu_g, dn_b, dn_r, dn_g;
  __nv_bfloat16 *out, *scores;
  // workspace
  int32_t* header;                   // kHdrStatus
  int32_t* counters;                 // [2] grid barriers, [kLayerMaxCtas + 1] tickets of split units
  float* logits;                     // [T, E]
  uint16_t* xh;                      // [T, Hp] rows as operands (bf16 or f16)
  float* x_scale;                    // [T] what their products are multiplied by
  uint16_t* act;                     // [S, Hp] fp32 (e4m3 weights), or [2 S, Hp] bf16 (value, rest)
  uint32_t* act_max;                 // [S] largest magnitude of an activation row, as bits
  float* part;                       // [ctas][2][kLayerRows][kLayerUnit] halves of split gate_up units
  float* y;                          // [S][2][H] down rows, second half for split units
  int T, H, Hp, E, K;
  int64_t capacity;
};
constexpr int kLayerMaxCtas = 256;

__device__ __forceinline__ float2 bf16x2_to_float2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// 2^k and 2^-k with k = 14 - exponent of the largest magnitude (bits), within what a float can be; 1 for infinities and NaN,
// which stay what they are
__device__ __forceinline__ void layer_factor(uint32_t most, float& factor, float& inverse) {
  const int shift = most >= 0x7f800000u ? 0 : min(max(14 + 127 - (int)(most >> 23), -120), 120);
  factor = __uint_as_float((uint32_t)(127 + shift) << 23);
  inverse = __uint_as_float((uint32_t)(127 - shift) << 23);
}

// ---- router ---------------------------------------------------------------------------------------------------------
// A CTA per expert.  A warp takes a token, or several warps share one (T < 8).
template <bool FP8>
__global__ void __launch_bounds__(kLayerThreads)
layer_router_kernel(const LayerArgs a) {
  __shared__ float s_part[kLayerWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e = blockIdx.x, nvec = a.H / 8;
  pdl_trigger();
  if (e == 0) {
    for (int i = threadIdx.x; i < 16; i += kLayerThreads) a.header[i] = 0;
    for (int i = threadIdx.x; i < kLayerMaxCtas + 3; i += kLayerThreads) a.counters[i] = 0;
  }
  // logits
  const int wpt = a.T >= 8 ? 1 : a.T > 4 ? 1 : a.T > 2 ? 2 : a.T == 2 ? 4 : 8, tokens = kLayerWarps / wpt;
  const uint4* wr = reinterpret_cast<const uint4*>(a.router + (int64_t)e * a.H);
  for (int t0 = 0; t0 < a.T; t0 += tokens) {
    const int t = t0 + w / wpt;
    float sum = 0.f;
    if (t < a.T) {
      const uint4* xr = reinterpret_cast<const uint4*>(a.x + (int64_t)t * a.H);
#pragma unroll 4
      for (int i = (w % wpt) * 32 + lane; i < nvec; i += wpt * 32) {
        const uint4 p = __ldg(wr + i), q = __ldg(xr + i);
        const uint32_t pu[4] = {p.x, p.y, p.z, p.w}, qu[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = bf16x2_to_float2(pu[j]), g = bf16x2_to_float2(qu[j]);
          sum = fmaf(f.x, g.x, sum);
          sum = fmaf(f.y, g.y, sum);
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (wpt > 1) {
      __syncthreads();
      if (lane == 0) s_part[w] = sum;
      __syncthreads();
      sum = 0.f;
      for (int i = 0; i < wpt; ++i) sum += s_part[(w / wpt) * wpt + i];
    }
    if (lane == 0 && w % wpt == 0 && t < a.T)
      a.logits[(int64_t)t * a.E + e] = sum + (a.router_bias != nullptr ? __bfloat162float(a.router_bias[e]) : 0.f);
  }
  // token rows as operands, and the columns behind the activations' H (weights there are zeros, these must be finite)
  for (int t = e; t < a.T; t += a.E) {
    const __nv_bfloat16* xr = a.x + (int64_t)t * a.H;
    uint16_t* dst = a.xh + (int64_t)t * a.Hp;
    float factor = 1.f;
    if constexpr (FP8) {
      uint32_t most = 0;
      for (int i = threadIdx.x; i < a.H; i += kLayerThreads) {
        const uint32_t b = __float_as_uint(__bfloat162float(xr[i])) & 0x7fffffffu;
        if (b < 0x7f800000u) most = max(most, b);
      }
      most = __reduce_max_sync(0xffffffffu, most);
      __syncthreads();
      if (lane == 0) s_part[w] = __uint_as_float(most);
      __syncthreads();
      float top = 0.f, inverse;
      for (int i = 0; i < kLayerWarps; ++i) top = fmaxf(top, s_part[i]);
      layer_factor(__float_as_uint(top), factor, inverse);
      if (threadIdx.x == 0) a.x_scale[t] = inverse;
    } else if (threadIdx.x == 0) {
      a.x_scale[t] = 1.f;
    }
    for (int i = threadIdx.x; i < a.Hp; i += kLayerThreads) {
      uint16_t v = 0;
      if (i < a.H) v = FP8 ? __half_as_ushort(__float2half_rn(__bfloat162float(xr[i]) * factor)) : __bfloat16_as_ushort(xr[i]);
      dst[i] = v;
    }
  }
  const int pad = a.Hp - a.H, rows = a.T * a.K * 2;          // fp32 rows are as long as two of 16 bits
  for (int i = e * kLayerThreads + threadIdx.x; i < rows * pad; i += a.E * kLayerThreads) {
    const int r = i / pad, c = i - r * pad;
    if constexpr (FP8) a.act[(int64_t)(r >> 1) * 2 * a.Hp + 2 * a.H + (r & 1) * pad + c] = 0;
    else a.act[(int64_t)r * a.Hp + a.H + c] = 0;
  }
  if constexpr (FP8) {
    for (int i = e * kLayerThreads + threadIdx.x; i < a.T * a.K; i += a.E * kLayerThreads) a.act_max[i] = 0;
  }
}

// ---- experts --------------------------------------------------------------------------------------------------------

// Rank of a logit as an unsigned number: NaN above all, ties by value left to the caller
__device__ __forceinline__ uint32_t layer_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);      // -0 and +0 are equal
  return ((b >> 31) ? ~b : (b | 0x80000000u)) + 1u;            // 0: taken
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, bool f16) {
  if (f16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}

// Row of a weight tile that stands at M index g (0..7) of a fragment, e4m3: the two rows that eight lanes read in one go
// differ by four, so that with the 128-byte swizzle they lie on different banks.
template <bool FP8>
__device__ __forceinline__ int layer_m_row(int g) { return FP8 ? (g >> 1) + 4 * (g & 1) : g; }

// One tile of weights (e4m3: 64 rows of 128 reduction bytes; bf16: 64 reduction rows of 64 columns) times up to 8 * NT rows.
// rows[n]: the lane's row of n-tile n at the tile's first reduction index, or null.
template <bool FP8, int NT>
__device__ __forceinline__ void layer_load_rows(const uint16_t* const* rows, int lane, uint4 (&b)[NT][FP8 ? 4 : 2]) {
  const int c = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 4; ++i)        // 64 reduction indices: 16 per lane, two loads
        b[n][i] = rows[n] != nullptr ? __ldcg(reinterpret_cast<const uint4*>(rows[n] + 64 * (i >> 1) + 16 * c) + (i & 1))
                                     : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {      // steps 2 i and 2 i + 1: 4 per lane and step
        uint2 p = make_uint2(0, 0), q = p;
        if (rows[n] != nullptr) {
          p = __ldcg(reinterpret_cast<const uint2*>(rows[n] + 32 * i + 4 * c));
          q = __ldcg(reinterpret_cast<const uint2*>(rows[n] + 32 * i + 16 + 4 * c));
        }
        b[n][i] = make_uint4(p.x, p.y, q.x, q.y);
      }
    }
  }
}

// The same from fp32 rows, times each row's factor, as f16
template <int NT>
__device__ __forceinline__ void layer_load_rows_f32(const float* const* rows, const float* factor, int lane, uint4 (&b)[NT][4]) {
  const int c = lane & 3;
  float4 v[NT][8];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[n][i] = rows[n] != nullptr ? __ldcg(reinterpret_cast<const float4*>(rows[n] + 64 * (i >> 2) + 16 * c) + (i & 3))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 p = v[n][2 * i], q = v[n][2 * i + 1];
      const float f = factor[n];
      const __half2 h[4] = {__floats2half2_rn(p.x * f, p.y * f), __floats2half2_rn(p.z * f, p.w * f),
                            __floats2half2_rn(q.x * f, q.y * f), __floats2half2_rn(q.z * f, q.w * f)};
      b[n][i] = *reinterpret_cast<const uint4*>(h);
    }
}

template <bool FP8, int NT>
__device__ __forceinline__ void layer_tile(uint32_t tile, int lane, const uint4 (&b)[NT][FP8 ? 4 : 2], float scale,
                                           float (*acc)[4][4]) {
  const int g = lane >> 2, c = lane & 3;
  if constexpr (FP8) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      uint32_t raw[2][2][4];               // [row g, row g + 8][half of the reduction]
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = m * 16 + r * 8 + layer_m_row<true>(g);
          const uint32_t addr = tile + row * 128 + (((4 * h + c) ^ (row & 7)) << 4);
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(raw[r][h][0]), "=r"(raw[r][h][1]), "=r"(raw[r][h][2]), "=r"(raw[r][h][3]) : "r"(addr));
        }
      float part[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t lo = raw[0][h][s], hi = raw[1][h][s];
          const uint32_t a0 = e4m3x2_to_f16x2(lo & 0xffffu), a2 = e4m3x2_to_f16x2(lo >> 16);
          const uint32_t a1 = e4m3x2_to_f16x2(hi & 0xffffu), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 q = b[n][2 * h + (s >> 1)];
            mma_16816(part[n], a0, a1, a2, a3, (s & 1) ? q.z : q.x, (s & 1) ? q.w : q.y, true);
          }
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(part[n][i], scale, acc[n][m][i]);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = lane & 7, kh = lane >> 4;
      const int k = 16 * s + 4 * (j >> 1) + 2 * kh + (j & 1);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int chunk = m * 2 + ((lane >> 3) & 1);
        const uint32_t addr = tile + k * 128 + ((chunk ^ (k & 7)) << 4);
        uint32_t a0, a1, a2, a3;
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(a0), "=r"(a1), "=r"(a2), "=r"(a3) : "r"(addr));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 q = b[n][s >> 1];
          mma_16816(acc[n][m], a0, a1, a2, a3, (s & 1) ? q.z : q.x, (s & 1) ? q.w : q.y, false);
        }
      }
    }
  }
}

// All CTAs of the (cooperative) grid have arrived here; false when the wait was given up.
__device__ __forceinline__ bool layer_grid_barrier(int32_t* counter, int ctas) {
  __syncthreads();
  int ok = 1;
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(counter, 1);
    uint64_t t0 = 0;
    for (uint32_t it = 0;; ++it) {
      int v;
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
      if (v >= ctas) break;
      if ((it & 255u) == 255u) {
        const uint64_t now = global_timer_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 > kWaitLimitNs) { ok = 0; break; }
      }
    }
  }
  return __syncthreads_and(threadIdx.x != 0 || ok);
}

struct LayerPhase {
  int64_t tiles;      // of all units
  int kt, units_n;    // tiles of a unit, units of an expert's matrix
  int ctas;           // that share them: no more than there are units, so that a unit has at most two owners
  __device__ __forceinline__ int64_t begin(int c) const { return c >= ctas ? tiles : tiles * c / ctas; }
  // the CTA that has tile g
  __device__ __forceinline__ int owner(int64_t g) const { return (int)(((g + 1) * ctas - 1) / tiles); }
};

template <bool FP8>
__global__ void __launch_bounds__(kLayerThreads, 1)
layer_experts_kernel(const __grid_constant__ CUtensorMap tm_gu, const __grid_constant__ CUtensorMap tm_dn, const LayerArgs a) {
  constexpr int kTileK = FP8 ? 128 : 64;
  constexpr int kNT = FP8 ? kLayerRows / 8 : kLayerRows / 4;        // most columns of N, in eights
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kLayerWarps][kLayerSlots];
  __shared__ int16_t s_e[kLayerMaxS], s_sorted[kLayerMaxS], s_slot_e[kLayerMaxS], s_slot_first[kLayerMaxS + 1], s_slot[kLayerMaxS];
  __shared__ int16_t s_rank[kLayerMaxS];      // among the expert's assignments; -1: dropped
  __shared__ float s_w[kLayerMaxS], s_xs[kLayerMaxT];
  __shared__ int s_slots, s_flag, abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + w * (kLayerSlots * kLayerTileBytes);
  uint8_t* aligned = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  float* red = reinterpret_cast<float*>(aligned + kLayerRingBytes);            // [warp][8][kLayerRedPitch]
  uint32_t* keys = reinterpret_cast<uint32_t*>(aligned) + w * 1024;            // ring space, before the first copy
  const int S = a.T * a.K;

  if (tid == 0) {
    for (int i = 0; i < kLayerWarps; ++i)
      for (int j = 0; j < kLayerSlots; ++j) mbar_init(smem_u32(&bar_full[i][j]), 1);
    abort_flag = 0;
    s_slots = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  // ---- top-k and softmax: a warp per token ----------------------------------------------------------------------------
  for (int t = w; t < a.T; t += kLayerWarps) {
    const float* lg = a.logits + (int64_t)t * a.E;
    for (int e = lane; e < a.E; e += 32) keys[e] = layer_key(__ldcg(lg + e));
    int mine = 0;                            // lane k: the k-th best
    for (int k = 0; k < a.K; ++k) {
      uint32_t best = 0;
      int at = 0x7fffffff;
      for (int e = lane; e < a.E; e += 32) {
        const uint32_t v = keys[e];
        if (v > best) { best = v; at = e; }
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
      const int e = (int)__reduce_min_sync(0xffffffffu, (uint32_t)(best == top ? at : 0x7fffffff));
      if (lane == k) mine = e;
      if ((e & 31) == lane) keys[e] = 0;
    }
    __syncwarp();
    const float v = lane < a.K ? __ldcg(lg + mine) : 0.f, v0 = __shfl_sync(0xffffffffu, v, 0);
    const float ex = lane < a.K ? expf(v - v0) : 0.f;
    float sum = ex;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < a.K) {
      s_e[t * a.K + lane] = (int16_t)mine;
      s_w[t * a.K + lane] = ex / sum;
    }
    if (lane == 0) s_xs[t] = __ldcg(a.x_scale + t);
    if (t % ctas == cta) {                   // the dense row of scores, by one CTA
      __nv_bfloat16* row = a.scores + (int64_t)t * a.E;
      for (int e = lane; e < a.E; e += 32) row[e] = __float2bfloat16_rn(0.f);
      __syncwarp();
      if (lane < a.K) row[mine] = __float2bfloat16_rn(ex / sum);
    }
  }
  __syncthreads();
  // ---- rows of each expert, in ascending order; an expert with many takes several slots --------------------------------
  if (tid < S) {
    const int e = s_e[tid];
    int rank = 0;
    for (int q = 0; q < tid; ++q) rank += s_e[q] == e;
    s_rank[tid] = (int16_t)(rank < a.capacity ? rank : -1);
  }
  __syncthreads();
  if (tid < S) {
    const int e = s_e[tid], rank = s_rank[tid];
    int pos = 0, slot = 0, slots = 0;
    for (int q = 0; q < S; ++q) {
      const int r = s_rank[q];
      const bool lower = r >= 0 && s_e[q] < e, first = r >= 0 && r % kLayerRows == 0;
      pos += lower;
      slot += lower && first;
      slots += first;
    }
    if (rank >= 0) {
      pos += rank;
      slot += rank / kLayerRows;
      s_sorted[pos] = (int16_t)tid;
      if (rank % kLayerRows == 0) {
        s_slot_e[slot] = (int16_t)e;
        s_slot_first[slot] = (int16_t)pos;
      }
    }
    s_slot[tid] = (int16_t)slot;
    if (tid == 0) s_slots = slots;
  }
  const int kept = __syncthreads_count(tid < S && s_rank[tid] >= 0);
  if (tid == 0) s_slot_first[s_slots] = (int16_t)kept;
  // the keys that lay in the ring were written by ordinary stores, the copies come by another way
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();

  const int slots = s_slots;
  LayerPhase ph[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ph[i].kt = (a.H + kTileK - 1) / kTileK;
    ph[i].units_n = ((i == 0 ? 2 * a.H : a.H) + kLayerUnit - 1) / kLayerUnit;
    const int64_t units = (int64_t)slots * ph[i].units_n;
    ph[i].tiles = units * ph[i].kt;
    ph[i].ctas = (int)min((int64_t)ctas, units);
  }
  const int64_t b0 = slots ? ph[0].begin(cta) : 0, e0 = slots ? ph[0].begin(cta + 1) : 0;
  const int64_t b1 = slots ? ph[1].begin(cta) : 0, e1 = slots ? ph[1].begin(cta + 1) : 0;
  // this warp's tiles, one after the other through both phases: w, w + 8, ... of either range
  const int n0 = (int)((e0 - b0 - w + kLayerWarps - 1) / kLayerWarps), n1 = (int)((e1 - b1 - w + kLayerWarps - 1) / kLayerWarps);
  const int mine0 = e0 - b0 > w ? n0 : 0, mine1 = e1 - b1 > w ? n1 : 0;
  bool ok = true;
  auto issue = [&](int j) {                    // the warp's j-th tile into slot j % kLayerSlots
    if (j >= mine0 + mine1 || !ok) return;
    const int i = j < mine0 ? 0 : 1;
    const int64_t tile = (i == 0 ? b0 + w + (int64_t)kLayerWarps * j : b1 + w + (int64_t)kLayerWarps * (j - mine0));
    const int unit = (int)(tile / ph[0].kt), kt = (int)(tile - (int64_t)unit * ph[0].kt);
    const int slot = unit / ph[i].units_n, n = (unit - slot * ph[i].units_n) * kLayerUnit;
    if (lane == 0) {
      const uint32_t bar = smem_u32(&bar_full[w][j % kLayerSlots]), dst = ring + (j % kLayerSlots) * kLayerTileBytes;
      mbar_expect_tx(bar, kLayerTileBytes);
      if constexpr (FP8) tma_load_3d(dst, i == 0 ? &tm_gu : &tm_dn, kt * kTileK, n, s_slot_e[slot], bar);
      else tma_load_3d(dst, i == 0 ? &tm_gu : &tm_dn, n, kt * kTileK, s_slot_e[slot], bar);
    }
  };
  for (int j = 0; j < kLayerSlots; ++j) issue(j);

  int seq = 0;                                 // of this warp's tiles
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && !layer_grid_barrier(a.counters, ctas)) {
      if (tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
    }
    const int64_t begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1;
    const int kt_n = ph[0].kt, units_n = ph[i].units_n, N = i == 0 ? 2 * a.H : a.H;
    const bool pairs = i == 1 && !FP8;         // a row takes two columns: value and rest
    int64_t next = begin + w;                  // this warp's next tile
#pragma unroll 1
    for (int64_t g = begin; g < end;) {
      const int unit = (int)(g / kt_n);
      const int64_t unit_begin = (int64_t)unit * kt_n, seg_end = min(end, unit_begin + kt_n);
      const int slot = unit / units_n, col0 = (unit - slot * units_n) * kLayerUnit, e = s_slot_e[slot];
      const int first = s_slot_first[slot], n_rows = s_slot_first[slot + 1] - first;
      const int cols = pairs ? 2 * n_rows : n_rows, nt = (cols + 7) / 8;
      const int my_col = col0 + 2 * lane;      // of the sums that this thread takes up below
      float2 bias = make_float2(0.f, 0.f);
      if (i == 0 && my_col < N)
        bias = bf16x2_to_float2(__ldg(reinterpret_cast<const uint32_t*>(a.bias_gu + (int64_t)e * N + my_col)));
      const uint16_t* rows[kNT];
      float factor[kNT], inverse[kNT];         // of fp32 rows
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const int ci = n * 8 + (lane >> 2);
        rows[n] = nullptr;
        factor[n] = inverse[n] = 1.f;
        if (ci < cols) {
          const int p = s_sorted[first + (pairs ? ci >> 1 : ci)];
          rows[n] = i == 0 ? a.xh + (int64_t)(p / a.K) * a.Hp : a.act + (int64_t)(2 * p + (pairs ? ci & 1 : 0)) * a.Hp;
          if (FP8 && i == 1) layer_factor(__ldcg(a.act_max + p), factor[n], inverse[n]);
        }
      }
      const float* scales = nullptr;
      int64_t scale_step = 0;
      if constexpr (FP8) {
        scales = i == 0 ? a.scale_gu + e * a.gu_b + (col0 / 128) * a.gu_r : a.scale_dn + e * a.dn_b + (col0 / 128) * a.dn_r;
        scale_step = i == 0 ? a.gu_g : a.dn_g;
      }
      float acc[kNT][4][4];
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[n][m][r] = 0.f;
      auto tiles = [&](auto NTC) {
        constexpr int NT = decltype(NTC)::value;
#pragma unroll 1
        for (; next < seg_end; next += kLayerWarps, ++seq) {
          const int kt = (int)(next - unit_begin), at = seq % kLayerSlots;
          uint4 b[NT][FP8 ? 4 : 2];
          if (FP8 && i == 1) {
            if constexpr (FP8) {
              const float* r[NT];
#pragma unroll
              for (int n = 0; n < NT; ++n) r[n] = rows[n] != nullptr ? reinterpret_cast<const float*>(rows[n]) + kt * kTileK : nullptr;
              layer_load_rows_f32<NT>(r, factor, lane, b);
            }
          } else {
            const uint16_t* r[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) r[n] = rows[n] != nullptr ? rows[n] + kt * kTileK : nullptr;
            layer_load_rows<FP8, NT>(r, lane, b);
          }
          float scale = 1.f;
          if constexpr (FP8) scale = __ldg(scales + kt * scale_step);
          if (ok) ok = mbar_wait_warp(smem_u32(&bar_full[w][at]), (seq / kLayerSlots) & 1, &abort_flag);
          if (ok) layer_tile<FP8, NT>(ring + at * kLayerTileBytes, lane, b, scale, acc);
          __syncwarp();
          issue(seq + kLayerSlots);
        }
      };
      if (nt <= 1) tiles(std::integral_constant<int, 1>());
      else if (nt == 2 || kNT == 2) tiles(std::integral_constant<int, 2>());
      else tiles(std::integral_constant<int, kNT>());

      // ---- the warps' sums come together; a thread takes two columns of one row ---------------------------------------
      const bool whole = g == unit_begin && seg_end == unit_begin + kt_n;
      const int side = g == unit_begin ? 0 : 1, boundary = side == 0 ? cta + 1 : cta;
      auto finish_act = [&](int row, float2 v) {       // row of the slot; gate and up; by a whole warp
        const int p = s_sorted[first + row];
        const float xs = s_xs[p / a.K];
        const float act = my_col < N ? glu_act(fmaf(v.x, xs, bias.x), fmaf(v.y, xs, bias.y)) : 0.f;
        if constexpr (FP8) {
          const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(act) & 0x7fffffffu);
          if (lane == 0) atomicMax(a.act_max + p, most);
          if (my_col < N) reinterpret_cast<float*>(a.act)[(int64_t)p * a.Hp + (my_col >> 1)] = act;
        } else if (my_col < N) {
          const __nv_bfloat16 hi = __float2bfloat16_rn(act);
          uint16_t* dst = a.act + (int64_t)2 * p * a.Hp + (my_col >> 1);
          dst[0] = __bfloat16_as_ushort(hi);
          dst[a.Hp] = __bfloat16_as_ushort(__float2bfloat16_rn(act - __bfloat162float(hi)));
        }
      };
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        if (n >= nt) break;
        float* mine = red + w * (8 * kLayerRedPitch);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            mine[(2 * (lane & 3) + (r & 1)) * kLayerRedPitch + m * 16 + (r >> 1) * 8 + layer_m_row<FP8>(lane >> 2)] = acc[n][m][r];
        __syncthreads();
        const int c = n * 8 + w, row = pairs ? c >> 1 : c;       // warp w: column w of this n-tile
        if (c < cols && !(pairs && (c & 1))) {
          float2 v = make_float2(0.f, 0.f);
#pragma unroll
          for (int q = 0; q < kLayerWarps; ++q) {
            const float* src = red + (q * 8 + w) * kLayerRedPitch + 2 * lane;
            const float2 u = *reinterpret_cast<const float2*>(src);
            v.x += u.x; v.y += u.y;
            if (pairs) {
              const float2 rest = *reinterpret_cast<const float2*>(src + kLayerRedPitch);
              v.x += rest.x; v.y += rest.y;
            }
          }
          if (i == 1) {
            const int p = s_sorted[first + row];
            const float back = __shfl_sync(0xffffffffu, inverse[n], 4 * w);      // the lanes of that column hold it
            if (my_col < N)
              *reinterpret_cast<float2*>(a.y + ((int64_t)p * 2 + side) * a.H + my_col) = make_float2(v.x * back, v.y * back);
          } else if (whole) {
            finish_act(row, v);
          } else {
            float* dst = a.part + (((int64_t)boundary * 2 + side) * kLayerRows + row) * kLayerUnit + 2 * lane;
            *reinterpret_cast<float2*>(dst) = v;
          }
        }
        __syncthreads();
      }
      if (i == 0 && !whole) {
        // the CTA that comes second adds the halves (two numbers: the order does not matter)
        __threadfence();
        __syncthreads();
        if (tid == 0) s_flag = atomicAdd(a.counters + 2 + boundary, 1);
        __syncthreads();
        if (s_flag == 1) {
          __threadfence();
          for (int row = w; row < n_rows; row += kLayerWarps) {
            const float* src = a.part + ((int64_t)boundary * 2 * kLayerRows + row) * kLayerUnit + 2 * lane;
            const float2 u = __ldcg(reinterpret_cast<const float2*>(src));
            const float2 v = __ldcg(reinterpret_cast<const float2*>(src + kLayerRows * kLayerUnit));
            finish_act(row, make_float2(u.x + v.x, u.y + v.y));
          }
        }
        __syncthreads();
      }
      g = seg_end;
    }
  }
  if (!ok) {
    abort_flag = 1;
    atomicMax(a.header + kHdrStatus, (int)kStatusProducerTimeout);
  }
  // ---- out[t] = sum over the kept slots k of w (y + bias) ------------------------------------------------------------------
  if (!layer_grid_barrier(a.counters + 1, ctas)) {
    if (tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
  }
  const int half = a.H / 2;
  for (int i = cta * kLayerThreads + tid; i < a.T * half; i += ctas * kLayerThreads) {
    const int t = i / half, col = 2 * (i - t * half);
    float2 sum = make_float2(0.f, 0.f);
    for (int k = 0; k < a.K; ++k) {
      const int p = t * a.K + k;
      if (s_rank[p] < 0) continue;
      const int64_t unit_begin = ((int64_t)s_slot[p] * ph[1].units_n + col / kLayerUnit) * ph[1].kt;
      const float* src = a.y + (int64_t)p * 2 * a.H + col;
      float2 v = __ldcg(reinterpret_cast<const float2*>(src));
      if (ph[1].owner(unit_begin) != ph[1].owner(unit_begin + ph[1].kt - 1)) {
        const float2 u = __ldcg(reinterpret_cast<const float2*>(src + a.H));
        v.x += u.x; v.y += u.y;
      }
      const float2 bias = bf16x2_to_float2(__ldg(reinterpret_cast<const uint32_t*>(a.bias_dn + (int64_t)s_e[p] * a.H + col)));
      sum.x = fmaf(s_w[p], v.x + bias.x, sum.x);
      sum.y = fmaf(s_w[p], v.y + bias.y, sum.y);
    }
    *reinterpret_cast<uint32_t*>(a.out + (int64_t)t * a.H + col) = pack_bf16x2(sum.x, sum.y);
  }
  if (abort_flag != 0) {
    // copies that may still be in flight get time to land before the shared memory is released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
}

// ---- host side --------------------------------------------------------------------------------------------------------
inline bool layer_shape_ok(int64_t T, int H, int E, int K) {
  return T >= 0 && T <= kLayerMaxT && T * K <= kLayerMaxS && K > 0 && K <= kLayerMaxK && E > 0 && E <= 1024 && K <= E && H > 0 &&
         H % 8 == 0 && H <= 1 << 16;
}

// Workspace: fills the pointers of `a` (base null: only measures) and returns the bytes
inline size_t layer_workspace(LayerArgs& a, char* base) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    off = (off + 255) & ~size_t(255);
    char* p = base != nullptr ? base + off : nullptr;
    off += bytes;
    return p;
  };
  const size_t S = (size_t)a.T * a.K;
  a.Hp = (int)round_up(a.H, 128);
  a.header = reinterpret_cast<int32_t*>(take(256));
  a.counters = reinterpret_cast<int32_t*>(take((kLayerMaxCtas + 3) * 4));
  a.logits = reinterpret_cast<float*>(take((size_t)a.T * a.E * 4));
  a.xh = reinterpret_cast<uint16_t*>(take((size_t)a.T * a.Hp * 2));
  a.x_scale = reinterpret_cast<float*>(take((size_t)a.T * 4));
  a.act = reinterpret_cast<uint16_t*>(take(S * a.Hp * 4));
  a.act_max = reinterpret_cast<uint32_t*>(take(S * 4));
  a.part = reinterpret_cast<float*>(take((size_t)(kLayerMaxCtas + 1) * 2 * kLayerRows * kLayerUnit * 4));
  a.y = reinterpret_cast<float*>(take(S * 2 * a.H * 4));
  return off + 256;
}

template <bool FP8>
inline int launch_moe_layer(const LayerArgs& a, const CUtensorMap& gu, const CUtensorMap& dn, cudaStream_t st) {
  auto kern = layer_experts_kernel<FP8>;
  static PerDevice<int> configured;
  const int dev = current_device_index();
  if (!configured.get(dev)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kLayerSmem) != cudaSuccess) return YAMOE_ERR_CUDA;
    configured.set(dev, 1);
  }
  layer_router_kernel<FP8><<<(unsigned)a.E, kLayerThreads, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return YAMOE_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(umma_sm_count(), kLayerMaxCtas));
  cfg.blockDim = dim3(kLayerThreads);
  cfg.dynamicSmemBytes = kLayerSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;       // its CTAs wait for one another: all of them are resident or none
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, gu, dn, a) != cudaSuccess) return YAMOE_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
