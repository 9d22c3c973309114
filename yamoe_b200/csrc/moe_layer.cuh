// The whole layer for a few tokens in two launches: router, top-k, and the experts hit, weights in bf16 or in e4m3 with
// 128 x 128 scales (the activations keep 16 bits: a step of a few tokens is bound by the bytes of the weights).
//
//   layer_router_kernel   logits = x Wr^T + b in fp32; the token rows as padded 16-bit operands; counters to zero
//   layer_experts_kernel  cooperative, one CTA per SM: top-k and lists of rows (each CTA for itself), gate_up with GLU,
//                         grid barrier, down, grid barrier, weighted sum of a token's K rows in slot order
//
// Bound by HBM where the weights of the experts hit exceed some 50 MB, by latency below.  What carries it:
//  * The weights do not depend on anything but the routing, so one warp streams the CTA's tiles of 32 KB through a ring (TMA,
//    128 KB in flight per SM; half of that is as fast), on across units and across the grid barrier: HBM works through the
//    ends of units, and when the activations are ready the first down weights already lie in shared memory.  The rows that
//    meet a tile come with it, by bulk copies (those of the first down tiles after the barrier); read from global memory by
//    each of the eight warps they took 40 of 197 us with 16 tokens.
//  * A unit is 128 output columns of one expert with the whole reduction, 16 columns to each of eight warps: no sums
//    cross warps (split along the reduction instead, a warp's tiles for itself, they took as long to come together as
//    the products).
//  * Both phases are cut into equal shares of tiles, not of output columns: a unit may be split over up to four CTAs.  Of a
//    split gate_up unit those that do not have its beginning take their part up first of all and leave its sums in memory,
//    each beside a mark; the one that has the beginning, mostly the last thing that it does, finds them there and adds
//    them up in order.  No fence: behind the weights in flight one took 5 us.
//  * The products are m16n8k16 of mma.sync with the WEIGHT columns as M and up to eight rows as N: the tensor core
//    is far from busy, and a weight costs the same number of instructions for one row as for eight.  Within a tile the
//    reduction index is permuted (the same way for both operands), so that the rows come by 8- or 16-byte loads.
//
// 128 experts, H = 2880, K = 4: one token 55 us with bf16 weights (200 MB, 0.55 of copy rate: 23 us are router, launches, first
// copies, barriers and combine), 43 with e4m3 (100 MB); 16 tokens, 64 experts, H = 2048, K = 8, e4m3: 170 (712 MB, 0.64).
// With bf16 weights the router's kernel and the expert op are faster from four tokens on (16 tokens 258 us there, 309 here).
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
constexpr int kLayerWarps = 8, kLayerThreads = 32 * (kLayerWarps + 1);     // one to issue the copies
constexpr int kLayerTileBytes = 32768, kLayerStages = 4;           // a tile: two halves along the reduction
constexpr int kLayerUnit = 16 * kLayerWarps;                       // output columns of a unit
constexpr int kLayerParts = 4;                                     // owners of a unit, at most
constexpr int kLayerRows = 16;                                     // rows of an expert that share a pass over its weights
// Rows of a tile in shared memory: 16 of 256 fp32 or 16-bit values, or 32 of 128 bf16; 16 bytes more than that apart, so that the
// rows that eight lanes read lie on different banks
constexpr int kLayerRowBytes = kLayerRows * (256 * 4 + 16);
constexpr int kLayerStageRows = kLayerStages * kLayerTileBytes;    // where they begin
constexpr int kLayerSmem = kLayerStages * (kLayerTileBytes + kLayerRowBytes) + 1024;
constexpr int kRouterWarps = 8, kRouterThreads = 32 * kRouterWarps;
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
  int32_t* counters;                 // [2] grid barriers
  float* logits;                     // [T, E]
  uint16_t* xh;                      // [T, Hp] rows as operands (bf16 or f16)
  float* x_scale;                    // [T] what their products are multiplied by
  uint16_t* act;                     // [S, Hp] fp32 (e4m3 weights), or [2 S, Hp] bf16 (value, rest)
  uint32_t* act_max;                 // [S] largest magnitude of an activation row, as bits
  uint2* part;                       // [ctas][min(T, kLayerRows)][kLayerUnit] later parts of split gate_up units, marked
  float* y;                          // [S][kLayerParts or 2][H] down rows, the parts of a split unit (0 where there are fewer)
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
// A CTA per expert, and T more for the token rows as operands.  A warp takes a token's logit, or several warps share one (T < 8).
template <bool FP8>
__global__ void __launch_bounds__(kRouterThreads)
layer_router_kernel(const LayerArgs a) {
  __shared__ float s_part[kRouterWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e = blockIdx.x, nvec = a.H / 8;
  if (e == a.E) {
    for (int i = threadIdx.x; i < 16; i += kRouterThreads) a.header[i] = 0;
    if (threadIdx.x < 2) a.counters[threadIdx.x] = 0;
  }
  if (e < a.E) {
    // logits
    const int wpt = a.T > 4 ? 1 : a.T > 2 ? 2 : a.T == 2 ? 4 : 8, tokens = kRouterWarps / wpt;
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
  }
  // marks of split units
  const int marks = kLayerMaxCtas * min(a.T, kLayerRows) * kLayerUnit / 2;
  for (int i = e * kRouterThreads + threadIdx.x; i < marks; i += (a.E + a.T) * kRouterThreads)
    reinterpret_cast<uint4*>(a.part)[i] = make_uint4(0, 0, 0, 0);
  if (e < a.E) return;
  // token rows as operands (eight values at a time), and the columns behind the activations' H (weights there are zeros, these
  // must be finite)
  const int t = e - a.E;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + (int64_t)t * a.H);
  uint4* dst = reinterpret_cast<uint4*>(a.xh + (int64_t)t * a.Hp);
  float factor = 1.f;
  if constexpr (FP8) {
    uint32_t most = 0;
    for (int i = threadIdx.x; i < nvec; i += kRouterThreads) {
      const uint4 q = __ldg(xr + i);
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = (u[j] << 16) & 0x7fffffffu, hi = u[j] & 0x7fff0000u;
        if (lo < 0x7f800000u) most = max(most, lo);
        if (hi < 0x7f800000u) most = max(most, hi);
      }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) s_part[w] = __uint_as_float(most);
    __syncthreads();
    float top = 0.f, inverse;
    for (int i = 0; i < kRouterWarps; ++i) top = fmaxf(top, s_part[i]);
    layer_factor(__float_as_uint(top), factor, inverse);
    if (threadIdx.x == 0) a.x_scale[t] = inverse;
  } else if (threadIdx.x == 0) {
    a.x_scale[t] = 1.f;
  }
  for (int i = threadIdx.x; i < a.Hp / 8; i += kRouterThreads) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (i < nvec) {
      q = __ldg(xr + i);
      if constexpr (FP8) {
        uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = bf16x2_to_float2(u[j]);
          const __half2 h = __floats2half2_rn(f.x * factor, f.y * factor);
          u[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        q = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
    dst[i] = q;
  }
  const int pad = a.Hp - a.H, rows = a.T * a.K * 2;          // fp32 rows are as long as two of 16 bits
  for (int i = (e - a.E) * kRouterThreads + threadIdx.x; i < rows * pad; i += a.T * kRouterThreads) {
    const int r = i / pad, c = i - r * pad;
    if constexpr (FP8) a.act[(int64_t)(r >> 1) * 2 * a.Hp + 2 * a.H + (r & 1) * pad + c] = 0;
    else a.act[(int64_t)r * a.Hp + a.H + c] = 0;
  }
  if constexpr (FP8) {
    for (int i = (e - a.E) * kRouterThreads + threadIdx.x; i < a.T * a.K; i += a.T * kRouterThreads) a.act_max[i] = 0;
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// Half a tile of weights: e4m3 128 rows (output columns) of 128 reduction bytes; bf16 twice 64 reduction rows of 64 output
// columns.  The operands that a lane holds of the rows that it multiplies, 8 * NT of them, for one half: `row`, the
// shared memory address of the lane's row of the first eight at the half's first reduction index, the next eight 8 * pitch
// further.  Rows that do not exist are not defined, nor is what is computed of them.
template <bool FP8, bool F32, int NT>
__device__ __forceinline__ void layer_rows(uint32_t row, uint32_t pitch, int c, const float (&factor)[NT], uint4 (&b)[NT][FP8 ? 4 : 2]) {
  auto ld16 = [](uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const uint32_t at = row + n * 8 * pitch;
#pragma unroll
    for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
      if constexpr (F32) {                 // 16 neighbours out of each 64 reduction indices, eight at a time
        const uint4 u = ld16(at + (64 * (i >> 1) + 16 * c) * 4 + 32 * (i & 1)), v = ld16(at + (64 * (i >> 1) + 16 * c) * 4 + 32 * (i & 1) + 16);
        const float f = factor[n];
        const __half2 h[4] = {__floats2half2_rn(__uint_as_float(u.x) * f, __uint_as_float(u.y) * f),
                              __floats2half2_rn(__uint_as_float(u.z) * f, __uint_as_float(u.w) * f),
                              __floats2half2_rn(__uint_as_float(v.x) * f, __uint_as_float(v.y) * f),
                              __floats2half2_rn(__uint_as_float(v.z) * f, __uint_as_float(v.w) * f)};
        b[n][i] = *reinterpret_cast<const uint4*>(h);
      } else if constexpr (FP8) {
        b[n][i] = ld16(at + (64 * (i >> 1) + 16 * c) * 2 + 16 * (i & 1));
      } else {                             // four neighbours out of each 16
        uint2 lo, hi;
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(lo.x), "=r"(lo.y) : "r"(at + (32 * i + 4 * c) * 2));
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(hi.x), "=r"(hi.y) : "r"(at + (32 * i + 16 + 4 * c) * 2));
        b[n][i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  }
}

// acc += the warp's 16 output columns of half a tile times up to 8 * NT rows
template <bool FP8, int NT>
__device__ __forceinline__ void layer_tile(uint32_t tile, int w, int lane, const uint4 (&b)[NT][FP8 ? 4 : 2], float scale,
                                           float (&acc)[NT][4]) {
  if constexpr (FP8) {
    const int g = lane >> 2, c = lane & 3;
    uint32_t raw[2][2][4];                 // [row g, row g + 8][half of the reduction]
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = w * 16 + r * 8 + layer_m_row<true>(g);
        const uint32_t addr = tile + row * 128 + (((4 * h + c) ^ (row & 7)) << 4);
        uint32_t (&q)[4] = raw[r][h];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(addr));
      }
    float part[2][NT][4];                  // of either half: two chains of products
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[h][n][i] = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t lo = raw[0][h][s], hi = raw[1][h][s];
        const uint32_t a0 = e4m3x2_to_f16x2(lo & 0xffffu), a2 = e4m3x2_to_f16x2(lo >> 16);
        const uint32_t a1 = e4m3x2_to_f16x2(hi & 0xffffu), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 q = b[n][2 * h + (s >> 1)];
          mma_16816(part[h][n], a0, a1, a2, a3, (s & 1) ? q.z : q.x, (s & 1) ? q.w : q.y, true);
        }
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = fmaf(part[0][n][i] + part[1][n][i], scale, acc[n][i]);
  } else {
    uint32_t f[4][4];
    const int j = lane & 7, kh = lane >> 4, chunk = (w & 3) * 2 + ((lane >> 3) & 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = 16 * s + 4 * (j >> 1) + 2 * kh + (j & 1);
      const uint32_t addr = tile + (w >> 2) * 8192 + k * 128 + ((chunk ^ (k & 7)) << 4);
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(f[s][0]), "=r"(f[s][1]), "=r"(f[s][2]), "=r"(f[s][3]) : "r"(addr));
    }
    float part[NT][4];                     // the odd steps: two chains of products
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 x = b[n][s >> 1];
        mma_16816((s & 1) ? part[n] : acc[n], f[s][0], f[s][1], f[s][2], f[s][3], (s & 1) ? x.z : x.x, (s & 1) ? x.w : x.y, false);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] += part[n][i];
  }
}

// All CTAs of the (cooperative) grid have arrived here with their product warps; false when the wait was given up.
__device__ __forceinline__ bool layer_grid_barrier(int32_t* counter, int ctas, volatile int* outcome) {
  named_sync(1, 32 * kLayerWarps);
  if (threadIdx.x == 0) {
    int ok = 1;
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
    *outcome = ok;
  }
  named_sync(1, 32 * kLayerWarps);
  return *outcome != 0;
}

// A value and the mark that it is there, in one access of eight bytes
__device__ __forceinline__ void st_marked(uint2* p, float v) {
  asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p), "l"((1ull << 32) | __float_as_uint(v)) : "memory");
}
__device__ __forceinline__ bool ld_marked(const uint2* p, float& v) {
  uint64_t q;
  asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(q) : "l"(p) : "memory");
  v = __uint_as_float((uint32_t)q);
  return (q >> 32) != 0;
}

// A phase's tiles, dealt out in equal shares to the first `ctas` CTAs: at most kLayerParts - 1 for each unit, so that as many
// shares hold a unit's tiles and it has one owner more at most.  All below 2^31 (layer_shape_ok).
struct LayerPhase {
  int tiles, units_n, ctas, each, rest;      // of all units; units of an expert's matrix; tiles / ctas
  int parts;                                 // owners of a unit: 2 where there are as many units as CTAs, else kLayerParts
  __device__ __forceinline__ int begin(int c) const {
    return c >= ctas ? tiles : each * c + (int)((unsigned)rest * (unsigned)c / (unsigned)ctas);
  }
};

__device__ __forceinline__ float layer_key_value(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  const uint32_t b = key - 1u;
  return __uint_as_float((b >> 31) ? b & 0x7fffffffu : ~b);
}

// A token's K best experts, by one warp: lane k ends with the k-th and its logit.  NV * 32 >= E.
template <int NV>
__device__ __forceinline__ int layer_top_k(const float* logits, int E, int K, int lane, float& value) {
  uint32_t v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = lane + 32 * i < E ? layer_key(__ldcg(logits + lane + 32 * i)) : 0u;
  int mine = 0;
  for (int k = 0; k < K; ++k) {
    uint32_t best = v[0];
    int at = lane;
#pragma unroll
    for (int i = 1; i < NV; ++i)
      if (v[i] > best) { best = v[i]; at = lane + 32 * i; }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const int e = (int)__reduce_min_sync(0xffffffffu, (uint32_t)(best == top ? at : 0x7fffffff));
    if (lane == k) { mine = e; value = layer_key_value(top); }
    if ((e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == e >> 5) v[i] = 0;
    }
  }
  return mine;
}

// The same for more experts, with the keys in shared memory
__device__ __forceinline__ int layer_top_k_many(const float* logits, int E, int K, int lane, uint32_t* keys, float& value) {
  for (int e = lane; e < E; e += 32) keys[e] = layer_key(__ldcg(logits + e));
  int mine = 0;
  for (int k = 0; k < K; ++k) {
    uint32_t best = 0;
    int at = lane;
    for (int e = lane; e < E; e += 32) {
      const uint32_t v = keys[e];
      if (v > best) { best = v; at = e; }
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const int e = (int)__reduce_min_sync(0xffffffffu, (uint32_t)(best == top ? at : 0x7fffffff));
    if (lane == k) { mine = e; value = layer_key_value(top); }
    if ((e & 31) == lane) keys[e] = 0;
  }
  return mine;
}

template <bool FP8>
__global__ void __launch_bounds__(kLayerThreads, 1)
layer_experts_kernel(const __grid_constant__ CUtensorMap tm_gu, const __grid_constant__ CUtensorMap tm_dn, const LayerArgs a) {
  constexpr int kHalfK = FP8 ? 128 : 64, kTileK = 2 * kHalfK;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kLayerStages], bar_empty[kLayerStages], bar_act;
  __shared__ int16_t s_e[kLayerMaxS], s_sorted[kLayerMaxS], s_slot_e[kLayerMaxS], s_slot_first[kLayerMaxS + 1], s_slot[kLayerMaxS];
  __shared__ float s_w[kLayerMaxS], s_xs[kLayerMaxT];              
  __shared__ int s_scan[2][kLayerWarps + 1];
  __shared__ int abort_flag;
  __shared__ volatile int s_outcome;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* aligned = smem_raw + (ring - smem_u32(smem_raw));
  // ring space, before the first copy: by expert, the tokens that chose it, its first row and its first slot
  uint32_t* tokens_of = reinterpret_cast<uint32_t*>(aligned);
  int16_t* row_of = reinterpret_cast<int16_t*>(tokens_of + 1024);
  int16_t* slot_of = row_of + 1024;
  uint32_t* keys = tokens_of + 2048;         // [warps][1024]
  const int S = a.T * a.K;

  if (tid == 0) {
    for (int i = 0; i < kLayerStages; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), kLayerWarps);
    }
    mbar_init(smem_u32(&bar_act), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int e = tid; e < a.E; e += kLayerThreads) tokens_of[e] = 0;
  __syncthreads();
  // ---- top-k and softmax: a warp per token ----------------------------------------------------------------------------
  for (int t = w; t < a.T; t += kLayerWarps + 1) {
    const float* lg = a.logits + (int64_t)t * a.E;
    const float xs = __ldcg(a.x_scale + t);
    float v = 0.f;
    const int mine = a.E <= 64 ? layer_top_k<2>(lg, a.E, a.K, lane, v)
                     : a.E <= 128 ? layer_top_k<4>(lg, a.E, a.K, lane, v)
                     : layer_top_k_many(lg, a.E, a.K, lane, keys + w * 1024, v);
    const float v0 = __shfl_sync(0xffffffffu, v, 0);
    const float ex = lane < a.K ? expf(v - v0) : 0.f;
    float sum = ex;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < a.K) {
      s_e[t * a.K + lane] = (int16_t)mine;
      s_w[t * a.K + lane] = ex / sum;
      atomicOr(tokens_of + mine, 1u << t);
    }
    if (lane == 0) s_xs[t] = xs;
    if (t % ctas == cta) {                   // the dense row of scores, by one CTA
      __nv_bfloat16* row = a.scores + (int64_t)t * a.E;
      for (int e = lane; e < a.E; e += 32) row[e] = __float2bfloat16_rn(0.f);
      __syncwarp();
      if (lane < a.K) row[mine] = __float2bfloat16_rn(ex / sum);
    }
  }
  __syncthreads();
  // ---- rows of each expert, in ascending order; an expert with many takes several slots --------------------------------
  const int cap = (int)min(a.capacity, (int64_t)kLayerMaxT), per = (a.E + kLayerThreads - 1) / kLayerThreads;
  int rows_in = 0, slots_in = 0;             // of this thread's experts, then of all before them
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i, n = e < a.E ? min(__popc(tokens_of[e]), cap) : 0;
    rows_in += n;
    slots_in += (n + kLayerRows - 1) / kLayerRows;
  }
  int rows_sum = rows_in, slots_sum = slots_in;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, rows_sum, o), q = __shfl_up_sync(0xffffffffu, slots_sum, o);
    if (lane >= o) { rows_sum += r; slots_sum += q; }
  }
  if (lane == 31) { s_scan[0][w] = rows_sum; s_scan[1][w] = slots_sum; }
  __syncthreads();
  int rows_at = rows_sum - rows_in, slots_at = slots_sum - slots_in, slots = 0, kept = 0;
#pragma unroll
  for (int i = 0; i <= kLayerWarps; ++i) {
    if (i < w) { rows_at += s_scan[0][i]; slots_at += s_scan[1][i]; }
    kept += s_scan[0][i];
    slots += s_scan[1][i];
  }
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i, n = e < a.E ? min(__popc(tokens_of[e]), cap) : 0;
    if (n == 0) continue;
    row_of[e] = (int16_t)rows_at;
    slot_of[e] = (int16_t)slots_at;
    for (int r = 0; r < n; r += kLayerRows, ++slots_at) {
      s_slot_e[slots_at] = (int16_t)e;
      s_slot_first[slots_at] = (int16_t)(rows_at + r);
    }
    rows_at += n;
  }
  if (tid == 0) s_slot_first[slots] = (int16_t)kept;
  __syncthreads();
  if (tid < S) {
    const int e = s_e[tid], rank = __popc(tokens_of[e] & ((1u << (tid / a.K)) - 1u));
    s_slot[tid] = -1;                        // dropped
    if (rank < cap) {
      s_sorted[row_of[e] + rank] = (int16_t)tid;
      s_slot[tid] = (int16_t)(slot_of[e] + rank / kLayerRows);
    }
  }
  // what lay in the ring was written by ordinary stores, the copies come by another way
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();

  const int kt_n = (a.H + kTileK - 1) / kTileK;      // tiles of a unit, in either phase
  auto phase_of = [&](int columns) {
    LayerPhase p;
    p.units_n = (columns + kLayerUnit - 1) / kLayerUnit;
    const int units = slots * p.units_n;
    p.tiles = units * kt_n;
    p.ctas = max(min(ctas, min((kLayerParts - 1) * units, p.tiles)), 1);
    p.parts = units >= p.ctas ? 2 : kLayerParts;
    p.each = (int)((unsigned)p.tiles / (unsigned)p.ctas);
    p.rest = p.tiles - p.each * p.ctas;
    return p;
  };
  const LayerPhase up = phase_of(2 * a.H), dn = phase_of(a.H);
  const int b0 = up.begin(cta), e0 = up.begin(cta + 1), b1 = dn.begin(cta), e1 = dn.begin(cta + 1);
  if (w == kLayerWarps) {
    // ---- the copies, through both phases ----------------------------------------------------------------------------------
    auto copy = [&](const CUtensorMap& map, uint32_t dst, int n, int kt, int e, uint32_t bar) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kt * kTileK + h * kHalfK;
        if constexpr (FP8) {
          tma_load_3d(dst + h * (kLayerTileBytes / 2), &map, k, n * kLayerUnit, e, bar);
        } else {
          tma_load_3d(dst + h * (kLayerTileBytes / 2), &map, n * kLayerUnit, k, e, bar);
          tma_load_3d(dst + h * (kLayerTileBytes / 2) + kLayerTileBytes / 4, &map, n * kLayerUnit + 64, k, e, bar);
        }
      }
    };
    // The rows of slot `slot` that meet reduction tile kt, a lane's one or two of them, to the stage whose bytes they are part of
    auto row_bytes = [&](int i, int kt) { return (uint32_t)min(kTileK, a.Hp - kt * kTileK) * (FP8 && i == 1 ? 4u : 2u); };
    auto copy_rows = [&](int i, int slot, int kt, int stage) {
      const bool pairs = i == 1 && !FP8;
      const int first = s_slot_first[slot], n_rows = s_slot_first[slot + 1] - first, size = FP8 && i == 1 ? 4 : 2;
      if (lane < (pairs ? 2 * n_rows : n_rows)) {
        const int p = s_sorted[first + (pairs ? lane >> 1 : lane)];
        const uint16_t* row = i == 0 ? a.xh + (int64_t)(p / a.K) * a.Hp : a.act + (int64_t)(2 * p + (pairs ? lane & 1 : 0)) * a.Hp;
        const void* src = reinterpret_cast<const uint8_t*>(row) + (int64_t)kt * kTileK * size;
        const uint32_t dst = ring + kLayerStageRows + stage * kLayerRowBytes + lane * (kTileK * size + 16);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(dst), "l"(src), "r"(row_bytes(i, kt)), "r"(smem_u32(&bar_full[stage])) : "memory");
      }
    };
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < 2 && ok; ++i) {
      const int begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1;
      const int units_n = i == 0 ? up.units_n : dn.units_n, first_unit = begin / kt_n;
      int kt = begin - first_unit * kt_n, slot = first_unit / units_n, n = first_unit - slot * units_n;
      // of the second phase a ring of weights goes out before the activations are there, their rows after
      int r_kt = kt, r_slot = slot, r_n = n, r_stage = stage, behind = 0;
      auto step = [&](int& k, int& s_, int& n_) {
        if (++k == kt_n) {
          k = 0;
          if (++n_ == units_n) { n_ = 0; ++s_; }
        }
      };
      bool there = i == 0;
      for (int g = begin; g < end || (ok && behind > 0); ++g) {
        if (!there && (g >= end || behind == kLayerStages)) {
          ok = mbar_wait_warp(smem_u32(&bar_act), 0, &abort_flag);
          if (!ok) break;
          asm volatile("fence.proxy.async;" ::: "memory");       // written by ordinary stores, read by copies
          for (; behind > 0; --behind) {
            copy_rows(i, r_slot, r_kt, r_stage);
            step(r_kt, r_slot, r_n);
            if (++r_stage == kLayerStages) r_stage = 0;
          }
          there = true;
          if (g >= end) break;
        }
        ok = mbar_wait_warp(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag);
        if (!ok) break;
        const uint32_t bar = smem_u32(&bar_full[stage]), dst = ring + stage * kLayerTileBytes;
        const int rows = (s_slot_first[slot + 1] - s_slot_first[slot]) * (i == 1 && !FP8 ? 2 : 1);
        if (lane == 0) {
          mbar_expect_tx(bar, kLayerTileBytes + rows * row_bytes(i, kt));
          if (i == 0) copy(tm_gu, dst, n, kt, s_slot_e[slot], bar); else copy(tm_dn, dst, n, kt, s_slot_e[slot], bar);
        }
        __syncwarp();
        if (there) copy_rows(i, slot, kt, stage); else ++behind;
        step(kt, slot, n);
        if (++stage == kLayerStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicMax(a.header + kHdrStatus, (int)kStatusProducerTimeout);
    }
    __syncwarp();
  } else {
    // ---- products: warps 0 .. 7 -----------------------------------------------------------------------------------------------
    // Biases and scales of this CTA's units are asked for as early as the weights: behind those a load that misses L2 would queue for as
    // long as all tiles in flight take, some 4 us.
    for (int i = 0; i < 2; ++i) {
      const int begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1, N = i == 0 ? 2 * a.H : a.H;
      const int units_n = i == 0 ? up.units_n : dn.units_n, per_unit = 2 + (FP8 ? (a.H + 127) / 128 : 0);
      if (begin == end) continue;
      const int u0 = begin / kt_n, asks = ((end - 1) / kt_n - u0 + 1) * per_unit;
      for (int j = tid; j < asks; j += 32 * kLayerWarps) {
        const int q = j / per_unit, what = j - q * per_unit, unit = u0 + q, slot = unit / units_n;
        const int col0 = (unit - slot * units_n) * kLayerUnit, e = s_slot_e[slot];
        const void* at = (i == 0 ? a.bias_gu : a.bias_dn) + (int64_t)e * N + min(col0 + 64 * what, N - 1);
        if (what > 1)
          at = i == 0 ? a.scale_gu + e * a.gu_b + (col0 / 128) * a.gu_r + (what - 2) * a.gu_g
                      : a.scale_dn + e * a.dn_b + (col0 / 128) * a.dn_r + (what - 2) * a.dn_g;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      }
    }
    const int part_rows = min(a.T, kLayerRows), g8 = lane >> 2, c4 = lane & 3;
    bool ok = true;
    int stage = 0;
    uint32_t full_phase = 0;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      if (i == 1) {
        asm volatile("fence.proxy.async;" ::: "memory");
        if (!layer_grid_barrier(a.counters, ctas, &s_outcome) && tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
        if (tid == 0) mbar_arrive(smem_u32(&bar_act));
      }
      const int begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1;
      const int units_n = i == 0 ? up.units_n : dn.units_n, N = i == 0 ? 2 * a.H : a.H;
      const bool pairs = i == 1 && !FP8;         // a row takes two columns of N: value and rest
      int unit = begin / kt_n, slot = unit / units_n, un = unit - slot * units_n;
#pragma unroll 1
      for (int g = begin; g < end; ++unit) {
        const int unit_begin = unit * kt_n, seg_end = min(end, unit_begin + kt_n), tiles = seg_end - g;
        const int col0 = un * kLayerUnit, e = s_slot_e[slot];
        const int first = s_slot_first[slot], n_rows = s_slot_first[slot + 1] - first;
        const int cols = pairs ? 2 * n_rows : n_rows;
        // this lane's two output columns; their biases as loaded, so that nothing waits for them before the sums are there
        const int ca = col0 + w * 16 + layer_m_row<FP8>(g8), cb = ca + 8;
        const __nv_bfloat16* bias = (i == 0 ? a.bias_gu : a.bias_dn) + (int64_t)e * N;
        const uint16_t bias_a = ca < N ? __ldg(reinterpret_cast<const uint16_t*>(bias) + ca) : (uint16_t)0;
        const uint16_t bias_b = cb < N ? __ldg(reinterpret_cast<const uint16_t*>(bias) + cb) : (uint16_t)0;
        const float* scales = nullptr;
        int64_t scale_step = 0;
        if constexpr (FP8) {
          scales = i == 0 ? a.scale_gu + e * a.gu_b + un * a.gu_r : a.scale_dn + e * a.dn_b + un * a.dn_r;
          scale_step = i == 0 ? a.gu_g : a.dn_g;
        }
        // which part of a split unit this is, and, for the first, how many there are
        const LayerPhase& ph = i == 0 ? up : dn;
        int side = 0, owners = 1;
        if (g > unit_begin) {
          do ++side; while (ph.begin(cta - side) > unit_begin);
        } else {
          while (cta + owners < ph.ctas && ph.begin(cta + owners) < unit_begin + kt_n) ++owners;
        }
        const int kt0 = g - unit_begin;

        auto work = [&](auto NTC, auto F32C) {
          constexpr int NT = decltype(NTC)::value;
          constexpr bool F32 = decltype(F32C)::value;
          float factor[NT], inverse[NT];         // of fp32 rows
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            factor[n] = inverse[n] = 1.f;
            if constexpr (F32) {
              if (n * 8 + g8 < cols) layer_factor(__ldcg(a.act_max + s_sorted[first + n * 8 + g8]), factor[n], inverse[n]);
            }
          }
          const uint32_t pitch = kTileK * (F32 ? 4 : 2) + 16;
          float acc[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[n][r] = 0.f;
          float scale_next = FP8 ? __ldg(scales + 2 * kt0 * scale_step) : 1.f;      // asked for half a tile ahead
#pragma unroll 1
          for (int j = 0; j < tiles; ++j) {
            const int halves = (2 * (kt0 + j) + 1) * kHalfK < a.H ? 2 : 1;       // the last tile of a unit may have one
            if (ok) ok = mbar_wait_warp(smem_u32(&bar_full[stage]), full_phase, &abort_flag);
            const uint32_t row = ring + kLayerStageRows + stage * kLayerRowBytes + g8 * pitch;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h == halves) break;
              const float scale = scale_next;
              if (FP8 && (h + 1 < halves || j + 1 < tiles)) scale_next = __ldg(scales + (2 * (kt0 + j) + h + 1) * scale_step);
              if (ok) {
                uint4 b[NT][FP8 ? 4 : 2];
                layer_rows<FP8, F32, NT>(row + h * kHalfK * (F32 ? 4 : 2), pitch, c4, factor, b);
                layer_tile<FP8, NT>(ring + stage * kLayerTileBytes + h * (kLayerTileBytes / 2), w, lane, b, scale, acc);
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_empty[stage]));
            if (++stage == kLayerStages) { stage = 0; full_phase ^= 1u; }
          }
          // ---- the ends of a unit: acc[n][0], [1] column ca of rows 8 n + 2 c4 and the next, [2], [3] column cb ------------------
          if (i == 1) {
            const float ba = side == 0 ? __uint_as_float((uint32_t)bias_a << 16) : 0.f, bb = side == 0 ? __uint_as_float((uint32_t)bias_b << 16) : 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < (FP8 ? 2 : 1); ++r) {
                // the factor of a row is held by the lanes whose operand it was
                const float back = F32 ? __shfl_sync(0xffffffffu, inverse[n], 4 * (2 * c4 + r)) : 1.f;
                const int ci = 8 * n + 2 * c4 + r;
                if (ci >= cols) continue;
                const float va = FP8 ? acc[n][r] : acc[n][0] + acc[n][1], vb = FP8 ? acc[n][2 + r] : acc[n][2] + acc[n][3];
                float* dst = a.y + (int64_t)s_sorted[first + (pairs ? ci >> 1 : ci)] * dn.parts * a.H;
                if (ca < N) {
                  dst[side * a.H + ca] = fmaf(va, back, ba);
                  for (int q = owners; side == 0 && q < dn.parts; ++q) dst[q * a.H + ca] = 0.f;
                }
                if (cb < N) {
                  dst[side * a.H + cb] = fmaf(vb, back, bb);
                  for (int q = owners; side == 0 && q < dn.parts; ++q) dst[q * a.H + cb] = 0.f;
                }
              }
            return;
          }
          if (side > 0 || owners > 1) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int ci = 8 * n + 2 * c4 + (r & 1), at = w * 16 + layer_m_row<FP8>(g8) + 8 * (r >> 1);
                uint2* mine = a.part + ((int64_t)cta * part_rows + min(ci, cols - 1)) * kLayerUnit + at;
                if (side > 0) {
                  if (ci < cols) st_marked(mine, acc[n][r]);
                } else {
                  for (int q = 1; q < owners; ++q) {
                    const uint2* src = mine + (int64_t)q * part_rows * kLayerUnit;
                    float other = 0.f;
                    uint64_t since = 0;
                    for (uint32_t it = 1; ok; ++it) {
                      if (__all_sync(0xffffffffu, ld_marked(src, other))) break;
                      if ((it & 255u) == 0u) {
                        const uint64_t now = global_timer_ns();
                        if (since == 0) since = now;
                        ok = __all_sync(0xffffffffu, *(volatile int*)&abort_flag == 0 && now - since <= kWaitLimitNs);
                      }
                    }
                    acc[n][r] += other;
                  }
                }
              }
            if (side > 0) return;
          }
          // GLU: neighbouring columns are gate and up.  Their lanes exchange, so that the even column's finishes row 2 c4 and the odd one's
          // the next.
          constexpr int kPartner = FP8 ? 8 : 4;
          const bool odd = (lane & kPartner) != 0;
          const float ba = __uint_as_float((uint32_t)bias_a << 16), bb = __uint_as_float((uint32_t)bias_b << 16);
          const float oa = __shfl_xor_sync(0xffffffffu, ba, kPartner), ob = __shfl_xor_sync(0xffffffffu, bb, kPartner);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float ga = __shfl_xor_sync(0xffffffffu, odd ? acc[n][0] : acc[n][1], kPartner);
            const float gb = __shfl_xor_sync(0xffffffffu, odd ? acc[n][2] : acc[n][3], kPartner);
            const int ci = 8 * n + 2 * c4 + (odd ? 1 : 0);
            const bool real = ci < cols;
            const int p = s_sorted[first + min(ci, cols - 1)];
            const float xs = s_xs[p / a.K];
            const float act_a = odd ? glu_act(fmaf(ga, xs, oa), fmaf(acc[n][1], xs, ba)) : glu_act(fmaf(acc[n][0], xs, ba), fmaf(ga, xs, oa));
            const float act_b = odd ? glu_act(fmaf(gb, xs, ob), fmaf(acc[n][3], xs, bb)) : glu_act(fmaf(acc[n][2], xs, bb), fmaf(gb, xs, ob));
            if constexpr (FP8) {
              float* dst = reinterpret_cast<float*>(a.act) + (int64_t)p * a.Hp;
              uint32_t most = max(ca < N ? __float_as_uint(act_a) & 0x7fffffffu : 0u, cb < N ? __float_as_uint(act_b) & 0x7fffffffu : 0u);
              most = max(most, __shfl_xor_sync(0xffffffffu, most, 4));
              most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
              if (real) {
                if (ca < N) dst[ca >> 1] = act_a;
                if (cb < N) dst[cb >> 1] = act_b;
                if ((lane & 20) == 0) atomicMax(a.act_max + p, most);
              }
            } else if (real) {
              uint16_t* dst = a.act + (int64_t)2 * p * a.Hp;
              const __nv_bfloat16 ha = __float2bfloat16_rn(act_a), hb = __float2bfloat16_rn(act_b);
              if (ca < N) {
                dst[ca >> 1] = __bfloat16_as_ushort(ha);
                dst[a.Hp + (ca >> 1)] = __bfloat16_as_ushort(__float2bfloat16_rn(act_a - __bfloat162float(ha)));
              }
              if (cb < N) {
                dst[cb >> 1] = __bfloat16_as_ushort(hb);
                dst[a.Hp + (cb >> 1)] = __bfloat16_as_ushort(__float2bfloat16_rn(act_b - __bfloat162float(hb)));
              }
            }
          }
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        using Four = std::integral_constant<int, 4>;
        if constexpr (FP8) {
          if (i == 0) {
            if (cols <= 8) work(One(), std::false_type()); else work(Two(), std::false_type());
          } else {
            if (cols <= 8) work(One(), std::true_type()); else work(Two(), std::true_type());
          }
        } else {
          if (cols <= 8) work(One(), std::false_type());
          else if (cols <= 16) work(Two(), std::false_type());
          else work(Four(), std::false_type());
        }
        g = seg_end;
        if (++un == units_n) { un = 0; ++slot; }
      }
    }
    if (!ok) {
      abort_flag = 1;
      atomicMax(a.header + kHdrStatus, (int)kStatusProducerTimeout);
    }
    // ---- out[t] = sum over the kept slots k of w (y + bias); eight neighbours to a CTA, so that few outputs spread over all --
    if (!layer_grid_barrier(a.counters + 1, ctas, &s_outcome)) {
      if (tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
    }
    const int half = a.H / 2;
    for (int i0 = ((tid >> 3) * ctas + cta) * 8; i0 < a.T * half; i0 += ctas * 32 * kLayerWarps) {
      const int i = i0 + (tid & 7);
      if (i >= a.T * half) break;
      const int t = i / half, col = 2 * (i - t * half);
      float2 sum = make_float2(0.f, 0.f);
      for (int k0 = 0; k0 < a.K; k0 += 4) {      // the loads of four slots together
        float2 v[4][kLayerParts];
        float weight[4];
        bool have[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int p = t * a.K + min(k0 + k, a.K - 1);
          have[k] = k0 + k < a.K && s_slot[p] >= 0;
          weight[k] = s_w[p];
#pragma unroll
          for (int q = 0; q < kLayerParts; ++q) {
            v[k][q] = make_float2(0.f, 0.f);
            if (have[k] && q < dn.parts)
              v[k][q] = __ldcg(reinterpret_cast<const float2*>(a.y + ((int64_t)p * dn.parts + q) * a.H + col));
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (have[k]) {
            sum.x = fmaf(weight[k], ((v[k][0].x + v[k][1].x) + v[k][2].x) + v[k][3].x, sum.x);
            sum.y = fmaf(weight[k], ((v[k][0].y + v[k][1].y) + v[k][2].y) + v[k][3].y, sum.y);
          }
      }
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)t * a.H + col) = pack_bf16x2(sum.x, sum.y);
    }
  }
  __syncthreads();
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
  a.counters = reinterpret_cast<int32_t*>(take(256));
  a.logits = reinterpret_cast<float*>(take((size_t)a.T * a.E * 4));
  a.xh = reinterpret_cast<uint16_t*>(take((size_t)a.T * a.Hp * 2));
  a.x_scale = reinterpret_cast<float*>(take((size_t)a.T * 4));
  a.act = reinterpret_cast<uint16_t*>(take(S * a.Hp * 4));
  a.act_max = reinterpret_cast<uint32_t*>(take(S * 4));
  a.part = reinterpret_cast<uint2*>(take((size_t)kLayerMaxCtas * std::min(a.T, kLayerRows) * kLayerUnit * 8));
  a.y = reinterpret_cast<float*>(take(S * kLayerParts * a.H * 4));
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
  layer_router_kernel<FP8><<<(unsigned)(a.E + a.T), kRouterThreads, 0, st>>>(a);
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
