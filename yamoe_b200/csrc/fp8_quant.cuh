// Quantisation to e4m3 in groups of 128: the operands of the 8-bit products (fp8_gemm.cuh).
//
//   a = max |x| over the group, at least 2^-100 (a NaN among the values makes a NaN)
//   scale = a / 448,   q = e4m3(x * (448 / a))         448 is the largest e4m3 value; nearest, ties to even
//
// with 32-bit divisions and products, so that every value has one definite code: a value equal to the largest becomes
// +-448 whatever way the two divisions are rounded.  A group is 128 neighbours in a row (activations, gradients) or
// 128 x 128 values (weights), the last ones of a matrix being smaller.
//
// Bound by HBM: a value is read once and its code written once, 3 bytes for bf16.  Rows (groups of 1 x 128) need no
// exchange beyond 16 lanes, which hold a group; blocks and transposed outputs go by tiles of 128 x 128 values held in
// the registers of a CTA, codes turned around in shared memory.
#pragma once
#include "common.cuh"

namespace yb {

constexpr int kFp8Group = 128;
constexpr float kFp8Max = 448.0f;
constexpr uint32_t kFp8LeastBits = 0x0d800000u;    // 2^-100

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// largest magnitude of a group, as bits: NaN ranks above everything there
__device__ __forceinline__ float fp8_group_max(uint32_t bits) { return __uint_as_float(max(bits, kFp8LeastBits)); }
__device__ __forceinline__ float fp8_scale(float a) { return __fdiv_rn(a, kFp8Max); }
__device__ __forceinline__ float fp8_inverse(float a) { return __fdiv_rn(kFp8Max, a); }

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// Eight neighbouring values of a row, of which `n` exist (the others 0); VEC: 16-byte loads, rows being aligned to them.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  if (VEC && n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p) + j);
        v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? DT<T>::ld(p + j) : 0.f;
  }
}

// ---- rows: groups of 1 x 128 --------------------------------------------------------------------------------------
// A half warp holds a group, eight values to a lane; a warp takes kQuantRows pairs of groups, whose loads are in flight
// together.  With `flat_row` a row is a token and goes to the rows of its K assignments (negative: dropped), read once.
constexpr int kQuantWarps = 8, kQuantPairs = 4;

struct QuantRows {
  uint8_t* q;          // [.., ldq]
  float* scale;        // (row, group) at row * scale_row + group * scale_group within its matrix
  int64_t ldq, scale_row, scale_group, scale_batch;
  const int32_t* flat_row;
  int slots;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32)
quantize_rows_kernel(const T* __restrict__ x, const QuantRows d, int64_t rows, int64_t rows_per_matrix, int K) {
  pdl_trigger();
  const int lane = threadIdx.x & 31, l16 = lane & 15;
  const int pairs = (K + 2 * kFp8Group - 1) / (2 * kFp8Group);
  const int64_t total = rows * pairs;
  const int64_t first = ((int64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5)) * kQuantPairs;
  float v[kQuantPairs][8];
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) {
    const int64_t u = first + i, row = u / pairs;
    const int k = (int)(u - row * pairs) * 2 * kFp8Group + lane * 8;
    load8<T, VEC>(x + row * K + k, u < total ? K - k : 0, v[i]);
  }
  pdl_wait();
  const int32_t* flat_row = d.flat_row != nullptr ? after_wait(d.flat_row) : nullptr;
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) {
    const int64_t u = first + i, row = u / pairs;
    const int k = (int)(u - row * pairs) * 2 * kFp8Group + lane * 8;
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[i][j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (u >= total || k >= K) continue;
    const float a = fp8_group_max(most), inv = fp8_inverse(a);
    uint2 out;
    out.x = e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
    out.y = e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
    const float s = fp8_scale(a);
    if (flat_row == nullptr) {
      *reinterpret_cast<uint2*>(d.q + row * d.ldq + k) = out;
      if (l16 == 0) {
        const int64_t b = row / rows_per_matrix, m = row - b * rows_per_matrix;
        d.scale[b * d.scale_batch + m * d.scale_row + (k / kFp8Group) * d.scale_group] = s;
      }
    } else {
      for (int j = 0; j < d.slots; ++j) {
        const int64_t r = flat_row[row * d.slots + j];
        if (r < 0) continue;
        *reinterpret_cast<uint2*>(d.q + r * d.ldq + k) = out;
        if (l16 == 0) d.scale[r * d.scale_row + (k / kFp8Group) * d.scale_group] = s;
      }
    }
  }
}

// ---- tiles: blocks of 128 x 128, transposed outputs ---------------------------------------------------------------
// One output of a tile kernel: codes [rows, ld] per matrix and scales (see QuantRows); q null: not wanted.
struct QuantOut {
  uint8_t* q;
  float* scale;
  int64_t ld, q_batch, scale_row, scale_group, scale_batch;
};

// A CTA holds 128 x 128 values of x: thread (rg, cg) rows 8 rg .. 8 rg + 7 of columns 8 cg .. 8 cg + 7.
// BLOCK: one scale for the tile, else one per row (`out`) and per column (`turned`).  `turned` gets the codes of x^T.
// Codes are turned around in shared memory with the 8-byte units of a row permuted (unit rg of row k lies at
// rg ^ (k / 8)), so that neither the writing by columns nor the reading by rows meets bank conflicts.
template <typename T, bool VEC, bool BLOCK>
__global__ void __launch_bounds__(256)
quantize_tile_kernel(const T* __restrict__ x, int64_t batch_stride, int M, int K, const QuantOut out, const QuantOut turned) {
  __shared__ __align__(16) uint8_t s_codes[128 * 128];
  __shared__ uint32_t s_max[8][128];
  pdl_trigger();
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m0 = blockIdx.y * 128, k0 = blockIdx.x * 128;
  const int64_t b = blockIdx.z;
  const int m = m0 + 8 * rg, k = k0 + 8 * cg;
  float v[8][8];
  pdl_wait();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load8<T, VEC>(x + b * batch_stride + (int64_t)(m + i) * K + k, m + i < M ? K - k : 0, v[i]);

  float inv_block = 0.f;
  [[maybe_unused]] uint2 codes_t[8];
  if constexpr (BLOCK) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[i][j]));
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) s_max[0][warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, s_max[0][w]);
    const float a = fp8_group_max(most);
    inv_block = fp8_inverse(a);
    if (threadIdx.x == 0) {
      if (out.q != nullptr) out.scale[b * out.scale_batch + blockIdx.y * out.scale_row + blockIdx.x * out.scale_group] = fp8_scale(a);
      if (turned.q != nullptr)
        turned.scale[b * turned.scale_batch + blockIdx.x * turned.scale_row + blockIdx.y * turned.scale_group] = fp8_scale(a);
    }
  }
  if (out.q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float inv = inv_block;
      if constexpr (!BLOCK) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[i][j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float a = fp8_group_max(most);
        inv = fp8_inverse(a);
        if (cg == 0 && m + i < M)
          out.scale[b * out.scale_batch + (int64_t)(m + i) * out.scale_row + blockIdx.x * out.scale_group] = fp8_scale(a);
      }
      if (m + i < M && k < K) {
        uint2 c;
        c.x = e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        c.y = e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv);
        *reinterpret_cast<uint2*>(out.q + b * out.q_batch + (int64_t)(m + i) * out.ld + k) = c;
      }
    }
  }
  if (turned.q == nullptr) return;
  float inv_col[8];
  if constexpr (!BLOCK) {
    uint32_t most[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      most[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most[j] = max(most[j], abs_bits(v[i][j]));
      most[j] = max(most[j], __shfl_xor_sync(0xffffffffu, most[j], 16));     // the other row group of this warp
      if (lane < 16) s_max[warp][8 * cg + j] = most[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int w = 0; w < 8; ++w) most[j] = max(most[j], s_max[w][8 * cg + j]);
      const float a = fp8_group_max(most[j]);
      inv_col[j] = fp8_inverse(a);
      if (rg == 0 && k + j < K)
        turned.scale[b * turned.scale_batch + (int64_t)(k + j) * turned.scale_row + blockIdx.y * turned.scale_group] = fp8_scale(a);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) inv_col[j] = inv_block;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint2 c;
    c.x = e4m3x4(v[0][j] * inv_col[j], v[1][j] * inv_col[j], v[2][j] * inv_col[j], v[3][j] * inv_col[j]);
    c.y = e4m3x4(v[4][j] * inv_col[j], v[5][j] * inv_col[j], v[6][j] * inv_col[j], v[7][j] * inv_col[j]);
    *reinterpret_cast<uint2*>(s_codes + (8 * cg + j) * 128 + ((rg ^ cg) << 3)) = c;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kk = 32 * i + (threadIdx.x >> 3), u = threadIdx.x & 7;      // 16 bytes: columns m0 + 16 u ...
    uint4 c = *reinterpret_cast<const uint4*>(s_codes + kk * 128 + ((u ^ (kk >> 4)) << 4));
    if ((kk >> 3) & 1) c = make_uint4(c.z, c.w, c.x, c.y);
    if (k0 + kk < K && m0 + 16 * u < M)
      *reinterpret_cast<uint4*>(turned.q + b * turned.q_batch + (int64_t)(k0 + kk) * turned.ld + m0 + 16 * u) = c;
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------
template <typename T>
inline bool rows_of_16_bytes(const void* x, int64_t K) {
  return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && K * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T>
inline int launch_quantize_rows(const T* x, const QuantRows& d, int64_t rows, int64_t rows_per_matrix, int K, bool pdl,
                                cudaStream_t st) {
  const int64_t work = ceil_div(rows * ceil_div(K, 2 * kFp8Group), kQuantPairs);
  const int64_t ctas = ceil_div(work, kQuantWarps);
  if (ctas == 0) return YAMOE_OK;
  if (ctas > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  auto kern = rows_of_16_bytes<T>(x, K) ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
  const cudaError_t rc =
      launch_pdl_opt(pdl, kern, dim3((unsigned)ctas), dim3(kQuantWarps * 32), 0, st, x, d, rows, rows_per_matrix, K);
  return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

template <typename T>
inline int launch_quantize_tiles(const T* x, int64_t B, int64_t M, int64_t K, bool block, const QuantOut& out,
                                 const QuantOut& turned, cudaStream_t st) {
  if (B == 0 || M == 0 || K == 0) return YAMOE_OK;
  const int64_t my = ceil_div(M, 128);
  if (my > 65535 || B > 65535) return YAMOE_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)ceil_div(K, 128), (unsigned)my, (unsigned)B);
  const bool vec = rows_of_16_bytes<T>(x, K);
  auto kern = block ? (vec ? quantize_tile_kernel<T, true, true> : quantize_tile_kernel<T, false, true>)
                    : (vec ? quantize_tile_kernel<T, true, false> : quantize_tile_kernel<T, false, false>);
  kern<<<grid, 256, 0, st>>>(x, M * K, (int)M, (int)K, out, turned);
  return cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
