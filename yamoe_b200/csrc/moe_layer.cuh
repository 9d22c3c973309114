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
//    the whole reduction) may be split over two CTAs.  Of a split gate_up unit the CTA that has its end, and takes it up
//    first of all, leaves its sums in memory, each beside a mark; the other, which has its beginning last of all, finds them
//    there.  No fence: behind the weights in flight one took 5 us.
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
  int32_t* counters;                 // [2] grid barriers
  float* logits;                     // [T, E]
  uint16_t* xh;                      // [T, Hp] rows as operands (bf16 or f16)
  float* x_scale;                    // [T] what their products are multiplied by
  uint16_t* act;                     // [S, Hp] fp32 (e4m3 weights), or [2 S, Hp] bf16 (value, rest)
  uint32_t* act_max;                 // [S] largest magnitude of an activation row, as bits
  uint2* part;                       // [ctas][min(T, kLayerRows)][kLayerUnit] second halves of split gate_up units, marked
  float* y;                          // [S][2][H] down rows, the halves of a split unit (else the second is 0)
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
__global__ void __launch_bounds__(kLayerThreads)
layer_router_kernel(const LayerArgs a) {
  __shared__ float s_part[kLayerWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e = blockIdx.x, nvec = a.H / 8;
  pdl_trigger();
  if (e == a.E) {
    for (int i = threadIdx.x; i < 16; i += kLayerThreads) a.header[i] = 0;
    if (threadIdx.x < 2) a.counters[threadIdx.x] = 0;
  }
  if (e < a.E) {
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
    return;
  }
  // token rows as operands, and the columns behind the activations' H (weights there are zeros, these must be finite)
  const int t = e - a.E;
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
  const int pad = a.Hp - a.H, rows = a.T * a.K * 2;          // fp32 rows are as long as two of 16 bits
  for (int i = (e - a.E) * kLayerThreads + threadIdx.x; i < rows * pad; i += a.T * kLayerThreads) {
    const int r = i / pad, c = i - r * pad;
    if constexpr (FP8) a.act[(int64_t)(r >> 1) * 2 * a.Hp + 2 * a.H + (r & 1) * pad + c] = 0;
    else a.act[(int64_t)r * a.Hp + a.H + c] = 0;
  }
  const int marks = kLayerMaxCtas * min(a.T, kLayerRows) * kLayerUnit / 2;
  for (int i = (e - a.E) * kLayerThreads + threadIdx.x; i < marks; i += a.T * kLayerThreads)
    reinterpret_cast<uint4*>(a.part)[i] = make_uint4(0, 0, 0, 0);
  if constexpr (FP8) {
    for (int i = (e - a.E) * kLayerThreads + threadIdx.x; i < a.T * a.K; i += a.T * kLayerThreads) a.act_max[i] = 0;
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
  // fragments are loaded a step ahead of the products that use them
  if constexpr (FP8) {
    uint32_t raw[2][2][2][4];              // [step parity][row g, row g + 8][half of the reduction]
    auto load = [&](int m) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = m * 16 + r * 8 + layer_m_row<true>(g);
          const uint32_t addr = tile + row * 128 + (((4 * h + c) ^ (row & 7)) << 4);
          uint32_t (&q)[4] = raw[m & 1][r][h];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(addr));
        }
    };
    load(0);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < 3) load(m + 1);
      float part[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t lo = raw[m & 1][0][h][s], hi = raw[m & 1][1][h][s];
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
    uint32_t f[2][4][4];                   // [step parity][m]
    auto load = [&](int s) {
      const int j = lane & 7, kh = lane >> 4;
      const int k = 16 * s + 4 * (j >> 1) + 2 * kh + (j & 1);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int chunk = m * 2 + ((lane >> 3) & 1);
        const uint32_t addr = tile + k * 128 + ((chunk ^ (k & 7)) << 4);
        uint32_t (&q)[4] = f[s & 1][m];
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(addr));
      }
    };
    load(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s < 3) load(s + 1);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t (&q)[4] = f[s & 1][m];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 x = b[n][s >> 1];
          mma_16816(acc[n][m], q[0], q[1], q[2], q[3], (s & 1) ? x.z : x.x, (s & 1) ? x.w : x.y, false);
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

// A phase's tiles, dealt out in equal shares to the first `ctas` CTAs: no more than there are units, so that a unit has at most
// two owners.  All below 2^31 (layer_shape_ok).
struct LayerPhase {
  int tiles, kt, units_n, ctas, each, rest;      // of all units; tiles of a unit; units of an expert's matrix; tiles / ctas
  __device__ __forceinline__ int begin(int c) const {
    return c >= ctas ? tiles : each * c + (int)((unsigned)rest * (unsigned)c / (unsigned)ctas);
  }
};

// Where a warp is in its tiles of a phase: every eighth of the CTA's share
struct LayerCursor {
  int slot, n, kt, left;
  __device__ __forceinline__ void start(const LayerPhase& p, int begin, int end, int w) {
    left = end - begin > w ? (end - begin - w + kLayerWarps - 1) / kLayerWarps : 0;
    const unsigned tile = (unsigned)(begin + w), unit = tile / (unsigned)p.kt;
    kt = (int)(tile - unit * p.kt);
    slot = (int)(unit / (unsigned)p.units_n);
    n = (int)(unit - (unsigned)slot * p.units_n);
  }
  __device__ __forceinline__ void step(const LayerPhase& p) {
    --left;
    kt += kLayerWarps;
    while (kt >= p.kt) {
      kt -= p.kt;
      if (++n == p.units_n) { n = 0; ++slot; }
    }
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

template <bool FP8>
__global__ void __launch_bounds__(kLayerThreads, 1)
layer_experts_kernel(const __grid_constant__ CUtensorMap tm_gu, const __grid_constant__ CUtensorMap tm_dn, const LayerArgs a) {
  constexpr int kTileK = FP8 ? 128 : 64;
  constexpr int kNT = FP8 ? kLayerRows / 8 : kLayerRows / 4;        // most columns of N, in eights
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kLayerWarps][kLayerSlots];
  __shared__ int16_t s_e[kLayerMaxS], s_sorted[kLayerMaxS], s_slot_e[kLayerMaxS], s_slot_first[kLayerMaxS + 1], s_slot[kLayerMaxS];
  __shared__ float s_w[kLayerMaxS], s_xs[kLayerMaxT];              
  __shared__ int s_scan[2][kLayerWarps];
  __shared__ int s_arrived[2], abort_flag;
  __shared__ volatile int s_done;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + w * (kLayerSlots * kLayerTileBytes);
  uint8_t* aligned = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  float* red = reinterpret_cast<float*>(aligned + kLayerRingBytes);            // see below
  // ring space, before the first copy: by expert, the tokens that chose it, its first row and its first slot
  uint32_t* tokens_of = reinterpret_cast<uint32_t*>(aligned);
  int16_t* row_of = reinterpret_cast<int16_t*>(tokens_of + 1024);
  int16_t* slot_of = row_of + 1024;
  const int S = a.T * a.K;

  if (tid == 0) {
    for (int i = 0; i < kLayerWarps; ++i)
      for (int j = 0; j < kLayerSlots; ++j) mbar_init(smem_u32(&bar_full[i][j]), 1);
    abort_flag = 0;
    s_arrived[0] = s_arrived[1] = 0;
    s_done = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int e = tid; e < a.E; e += kLayerThreads) tokens_of[e] = 0;
  __syncthreads();
  pdl_wait();
  // ---- top-k and softmax: a warp per token ----------------------------------------------------------------------------
  for (int t = w; t < a.T; t += kLayerWarps) {
    const float* lg = a.logits + (int64_t)t * a.E;
    const float xs = __ldcg(a.x_scale + t);
    float v = 0.f;
    const int mine = a.E <= 64 ? layer_top_k<2>(lg, a.E, a.K, lane, v)
                     : a.E <= 128 ? layer_top_k<4>(lg, a.E, a.K, lane, v) : layer_top_k<32>(lg, a.E, a.K, lane, v);
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
  for (int i = 0; i < kLayerWarps; ++i) {
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

  LayerPhase ph[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ph[i].kt = (a.H + kTileK - 1) / kTileK;
    ph[i].units_n = ((i == 0 ? 2 * a.H : a.H) + kLayerUnit - 1) / kLayerUnit;
    const int units = slots * ph[i].units_n;
    ph[i].tiles = units * ph[i].kt;
    ph[i].ctas = max(min(ctas, units), 1);
    ph[i].each = (int)((unsigned)ph[i].tiles / (unsigned)ph[i].ctas);
    ph[i].rest = ph[i].tiles - ph[i].each * ph[i].ctas;
  }
  const int b0 = ph[0].begin(cta), e0 = ph[0].begin(cta + 1), b1 = ph[1].begin(cta), e1 = ph[1].begin(cta + 1);
  // this warp's tiles, one after the other through both phases
  LayerCursor next0, next1;
  next0.start(ph[0], b0, e0, w);
  next1.start(ph[1], b1, e1, w);
  int issued = 0;
  bool ok = true;
  auto issue = [&]() {                         // the next tile into slot issued % kLayerSlots
    const bool up = next0.left > 0;
    if ((!up && next1.left <= 0) || !ok) return;
    const LayerCursor& at = up ? next0 : next1;
    if (lane == 0) {
      const int slot = issued % kLayerSlots;
      const uint32_t bar = smem_u32(&bar_full[w][slot]), dst = ring + slot * kLayerTileBytes;
      const CUtensorMap* map = up ? &tm_gu : &tm_dn;
      mbar_expect_tx(bar, kLayerTileBytes);
      if constexpr (FP8) tma_load_3d(dst, map, at.kt * kTileK, at.n * kLayerUnit, s_slot_e[at.slot], bar);
      else tma_load_3d(dst, map, at.n * kLayerUnit, at.kt * kTileK, s_slot_e[at.slot], bar);
    }
    ++issued;
    if (up) next0.step(ph[0]); else next1.step(ph[1]);
  };
  // Biases and scales of this CTA's units, ahead of the weights: behind those a load that misses L2 would queue for as long
  // as all tiles in flight take, some 4 us.
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1, N = i == 0 ? 2 * a.H : a.H, per_unit = 1 + (FP8 ? ph[i].kt : 0);
    if (begin == end) continue;
    const int u0 = begin / ph[i].kt, asks = ((end - 1) / ph[i].kt - u0 + 1) * per_unit;
    for (int j = tid; j < asks; j += kLayerThreads) {
      const int q = j / per_unit, what = j - q * per_unit, unit = u0 + q, slot = unit / ph[i].units_n;
      const int col0 = (unit - slot * ph[i].units_n) * kLayerUnit, e = s_slot_e[slot];
      const void* at = (i == 0 ? a.bias_gu : a.bias_dn) + (int64_t)e * N + col0;
      if (what > 0)
        at = i == 0 ? a.scale_gu + e * a.gu_b + (col0 / 128) * a.gu_r + (what - 1) * a.gu_g
                    : a.scale_dn + e * a.dn_b + (col0 / 128) * a.dn_r + (what - 1) * a.dn_g;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
    }
  }
  for (int j = 0; j < kLayerSlots; ++j) issue();

  // The warps' sums of a unit (of eight columns of N at a time: an item) come together in `red`, and the warp that is last
  // to put its own there adds them up and finishes them, while the others go on with their next tiles.  Up to four
  // columns take half of `red`, so that two items can be on their way.
  const int part_rows = min(a.T, kLayerRows);
  int seq = 0, item = 0;                       // tiles of this warp, items of this CTA so far
  bool before_small = false;
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && !layer_grid_barrier(a.counters, ctas)) {
      if (tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
    }
    const int begin = i == 0 ? b0 : b1, end = i == 0 ? e0 : e1;
    const int kt_n = ph[0].kt, units_n = ph[i].units_n, N = i == 0 ? 2 * a.H : a.H;
    const bool pairs = i == 1 && !FP8;         // a row takes two columns: value and rest
    int next = begin + w;                      // this warp's next tile
    int unit = (int)((unsigned)begin / (unsigned)kt_n);
#pragma unroll 1
    for (int g = begin; g < end; ++unit) {
      const int unit_begin = unit * kt_n, seg_end = min(end, unit_begin + kt_n);
      const int slot = (int)((unsigned)unit / (unsigned)units_n), col0 = (unit - slot * units_n) * kLayerUnit, e = s_slot_e[slot];
      const int first = s_slot_first[slot], n_rows = s_slot_first[slot + 1] - first;
      const int cols = pairs ? 2 * n_rows : n_rows, nt = (cols + 7) / 8;
      const int my_col = col0 + 2 * lane;      // of the sums that a thread finishes
      uint32_t bias2 = 0;                      // as loaded, so that nothing waits for it before the sums are there
      if (my_col < N) bias2 = __ldg(reinterpret_cast<const uint32_t*>((i == 0 ? a.bias_gu : a.bias_dn) + (int64_t)e * N + my_col));
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
          const int kt = next - unit_begin, at = seq % kLayerSlots;
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
          issue();
        }
      };
      if (nt <= 1) tiles(std::integral_constant<int, 1>());
      else if (nt == 2 || kNT == 2) tiles(std::integral_constant<int, 2>());
      else tiles(std::integral_constant<int, kNT>());

      const bool whole = g == unit_begin && seg_end == unit_begin + kt_n;
      const int side = g == unit_begin ? 0 : 1;      // the part of a split unit: its beginning, its end
      auto finish_act = [&](int row, float2 v) {       // row of the slot; gate and up; by a whole warp
        const int p = s_sorted[first + row];
        const float xs = s_xs[p / a.K];
        const float2 bias = bf16x2_to_float2(bias2);
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
        const int have = min(8, cols - 8 * n);
        const bool small = have <= 4;
        const int need = small && before_small ? item - 1 : item;            // items that must be done
        uint64_t t0 = 0;
        for (uint32_t it = 1; ok && !__all_sync(0xffffffffu, s_done >= need); ++it)
          if ((it & 255u) == 0u) {
            const uint64_t now = global_timer_ns();
            if (t0 == 0) t0 = now;
            ok = __all_sync(0xffffffffu, *(volatile int*)&abort_flag == 0 && now - t0 <= kWaitLimitNs);
          }
        __syncwarp();
        const int stride = (small ? 4 : 8) * kLayerRedPitch;                 // of a warp's part
        float* buf = red + (small && (item & 1) ? kLayerWarps * 4 * kLayerRedPitch : 0);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int c = 2 * (lane & 3) + (r & 1);
            if (c < have)
              buf[w * stride + c * kLayerRedPitch + m * 16 + (r >> 1) * 8 + layer_m_row<FP8>(lane >> 2)] = acc[n][m][r];
          }
        __threadfence_block();
        __syncwarp();
        int order = 0;
        if (lane == 0) order = atomicAdd(&s_arrived[item & 1], 1);
        order = __shfl_sync(0xffffffffu, order, 0);
        if (order == kLayerWarps - 1) {
          __threadfence_block();
          for (int c = 0; c < have; c += pairs ? 2 : 1) {
            const int row = pairs ? (8 * n + c) >> 1 : 8 * n + c;
            float2 v = make_float2(0.f, 0.f);
#pragma unroll
            for (int q = 0; q < kLayerWarps; ++q) {
              const float* src = buf + q * stride + c * kLayerRedPitch + 2 * lane;
              const float2 u = *reinterpret_cast<const float2*>(src);
              v.x += u.x; v.y += u.y;
              if (pairs) {
                const float2 tail = *reinterpret_cast<const float2*>(src + kLayerRedPitch);
                v.x += tail.x; v.y += tail.y;
              }
            }
            if (i == 1) {
              const int p = s_sorted[first + row];
              const float back = __shfl_sync(0xffffffffu, inverse[n], 4 * c);      // the lanes of that column hold it
              if (my_col < N) {
                const float2 bias = side == 0 ? bf16x2_to_float2(bias2) : make_float2(0.f, 0.f);
                float* dst = a.y + (int64_t)p * 2 * a.H + my_col;
                *reinterpret_cast<float2*>(dst + side * a.H) = make_float2(fmaf(v.x, back, bias.x), fmaf(v.y, back, bias.y));
                if (whole) *reinterpret_cast<float2*>(dst + a.H) = make_float2(0.f, 0.f);
              }
            } else if (whole) {
              finish_act(row, v);
            } else if (side == 1) {
              uint2* dst = a.part + ((int64_t)cta * part_rows + row) * kLayerUnit + 2 * lane;
              st_marked(dst, v.x);
              st_marked(dst + 1, v.y);
            } else {
              const uint2* src = a.part + ((int64_t)(cta + 1) * part_rows + row) * kLayerUnit + 2 * lane;
              float2 u = make_float2(0.f, 0.f);
              uint64_t since = 0;
              for (uint32_t it = 1; ok; ++it) {
                const bool there = ld_marked(src, u.x) & ld_marked(src + 1, u.y);
                if (__all_sync(0xffffffffu, there)) break;
                if ((it & 255u) == 0u) {
                  const uint64_t now = global_timer_ns();
                  if (since == 0) since = now;
                  ok = __all_sync(0xffffffffu, *(volatile int*)&abort_flag == 0 && now - since <= kWaitLimitNs);
                }
              }
              finish_act(row, make_float2(v.x + u.x, v.y + u.y));
            }
          }
          __syncwarp();
          if (lane == 0) {
            s_arrived[item & 1] = 0;
            __threadfence_block();
            s_done = item + 1;
          }
        }
        __syncwarp();
        before_small = small;
        ++item;
      }
      g = seg_end;
    }
  }
  if (!ok) {
    abort_flag = 1;
    atomicMax(a.header + kHdrStatus, (int)kStatusProducerTimeout);
  }
  // ---- out[t] = sum over the kept slots k of w (y + bias); eight neighbours to a CTA, so that few outputs spread over all --
  if (!layer_grid_barrier(a.counters + 1, ctas)) {
    if (tid == 0) atomicMax(a.header + kHdrStatus, kLayerStatusBarrier);
  }
  const int half = a.H / 2;
  for (int i0 = ((tid >> 3) * ctas + cta) * 8; i0 < a.T * half; i0 += ctas * kLayerThreads) {
    const int i = i0 + (tid & 7);
    if (i >= a.T * half) break;
    const int t = i / half, col = 2 * (i - t * half);
    float2 sum = make_float2(0.f, 0.f);
    for (int k0 = 0; k0 < a.K; k0 += 4) {      // the loads of four slots together
      float2 v[4], u[4];
      float weight[4];
      bool have[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = t * a.K + min(k0 + k, a.K - 1);
        have[k] = k0 + k < a.K && s_slot[p] >= 0;
        weight[k] = s_w[p];
        v[k] = u[k] = make_float2(0.f, 0.f);
        if (have[k]) {
          const float* src = a.y + (int64_t)p * 2 * a.H + col;
          v[k] = __ldcg(reinterpret_cast<const float2*>(src));
          u[k] = __ldcg(reinterpret_cast<const float2*>(src + a.H));
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (have[k]) {
          sum.x = fmaf(weight[k], v[k].x + u[k].x, sum.x);
          sum.y = fmaf(weight[k], v[k].y + u[k].y, sum.y);
        }
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
  a.counters = reinterpret_cast<int32_t*>(take(256));
  a.logits = reinterpret_cast<float*>(take((size_t)a.T * a.E * 4));
  a.xh = reinterpret_cast<uint16_t*>(take((size_t)a.T * a.Hp * 2));
  a.x_scale = reinterpret_cast<float*>(take((size_t)a.T * 4));
  a.act = reinterpret_cast<uint16_t*>(take(S * a.Hp * 4));
  a.act_max = reinterpret_cast<uint32_t*>(take(S * 4));
  a.part = reinterpret_cast<uint2*>(take((size_t)kLayerMaxCtas * std::min(a.T, kLayerRows) * kLayerUnit * 8));
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
  layer_router_kernel<FP8><<<(unsigned)(a.E + a.T), kLayerThreads, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return YAMOE_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(umma_sm_count(), kLayerMaxCtas));
  cfg.blockDim = dim3(kLayerThreads);
  cfg.dynamicSmemBytes = kLayerSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;       // its CTAs wait for one another: all of them are resident or none
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled(true) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, gu, dn, a) != cudaSuccess) return YAMOE_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
