// Quantisation to 8-bit integers with one scale per row (a token, an output channel): the operands of int8_gemm.cuh.
//
//   a = max |x| over the row, at least 2^-100;   scale = a / 127,   q = x * (127 / a) to the nearest integer, ties to even
//
// with 32-bit divisions and products, so that every value has one definite code.  Integers hold no NaN: a row with a NaN or an infinity gets
// codes 0 and the scale NaN, so that whatever is computed from it is NaN.
//
// Bound by HBM: a value is read once and its code written once, 3 bytes for bf16.  Rows: 1 to 8 warps hold one in registers; a longer one is read
// twice.  A row of one warp needs no barrier between its loads and its stores (11520 x 1024: 5.3 TB/s), one of two or four waits for the others (5760 x
// 2048, 2880 x 4096: 4.7, 4.8), and places that it does not fill are loads that are not under way (4096 x 2880, 70 % of four warps' places: 4.2).  Transposed (the codes of x^T, a scale per column of x): a cluster has a strip of 64 columns, reads it for the largest
// magnitudes and, but for its last rows, once more for the codes, which it turns around in shared memory.
#pragma once
#include <algorithm>

#include "fp8_quant.cuh"

namespace yb {

constexpr float kInt8Max = 127.0f;

__device__ __forceinline__ bool int8_bad(uint32_t most) { return most >= 0x7f800000u; }      // NaN or infinity
__device__ __forceinline__ float int8_scale(uint32_t most) {
  return int8_bad(most) ? __uint_as_float(0x7fc00000u) : __fdiv_rn(fp8_group_max(most), kInt8Max);
}
__device__ __forceinline__ float int8_inverse(uint32_t most) { return __fdiv_rn(kInt8Max, fp8_group_max(most)); }
// x * inverse lies in [-127, 127]: added to 1.5 * 2^23 its nearest integer is the low byte of the sum.  (One value at a time: two, by mul.rn.f32x2 and
// add.rn.f32x2, came out as one fma, which does not round the product.)
__device__ __forceinline__ uint32_t int8_code(float x, float inverse) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inverse), 12582912.f)); }
// Eight neighbouring values of a row; VEC: rows are multiples of eight, so that all of them exist or none.
template <bool VEC, typename T>
__device__ __forceinline__ void load_eight(Eight<T>& v, const T* p, int n) {
  if (VEC && n <= 0) v.template load<false>(p, 0);
  else v.template load<VEC>(p, VEC ? 8 : n);
}
__device__ __forceinline__ uint32_t int8x4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

struct Int8Out {
  uint8_t* q;            // codes of (matrix b, row r) at b * q_batch + r * ld
  float* scale;          // of (matrix b, row r) at b * scale_batch + r * scale_row
  int64_t ld, q_batch, scale_row, scale_batch;
};

constexpr int kInt8Pieces = 4;         // of 8 values that a lane holds
constexpr int kInt8RowWarps = 8;

// 2^log_wpr warps (1, 2, 4, 8) per row of x [batch, M, K]
template <typename T, bool VEC>
__global__ void __launch_bounds__(kInt8RowWarps * 32)
int8_rows_quantize_kernel(const T* x, const Int8Out d, int64_t M, int K, int log_wpr) {
  __shared__ uint32_t s_most[kInt8RowWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, wpr = 1 << log_wpr, sub = w & (wpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (kInt8RowWarps >> log_wpr) + (w >> log_wpr);
  const bool there = row < M;
  pdl_trigger();
  pdl_wait();
  const T* src = after_wait(x) + ((int64_t)blockIdx.y * M + (there ? row : 0)) * K;
  // (unsigned, as the step behind the last value may pass 31 bits)
  const unsigned step = wpr * 256, first = (sub * 32 + lane) * 8, end = there ? K : 0;
  Eight<T> v[kInt8Pieces];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kInt8Pieces; ++i) {
    const unsigned k = first + i * step;
    load_eight<VEC>(v[i], src + k, k < end ? (int)min(8u, end - k) : 0);
  }
#pragma unroll
  for (int i = 0; i < kInt8Pieces; ++i) most = max(most, v[i].most());
  for (unsigned k = first + kInt8Pieces * step; k < end; k += step) {
    Eight<T> more;
    load_eight<VEC>(more, src + k, (int)min(8u, end - k));
    most = max(most, more.most());
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (wpr > 1) {
    if (lane == 0) s_most[w] = most;
    __syncthreads();
    for (int i = 0; i < wpr; ++i) most = max(most, s_most[w - sub + i]);
  }
  if (!there) return;
  const float inv = int8_inverse(most);
  const bool bad = int8_bad(most);
  if (sub == 0 && lane == 0) d.scale[blockIdx.y * d.scale_batch + row * d.scale_row] = int8_scale(most);
  uint8_t* dst = d.q + blockIdx.y * d.q_batch + row * d.ld;
  auto put = [&](const Eight<T>& e, unsigned k) {
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = int8_code(e.value(j), inv);
    const uint2 out = make_uint2(int8x4(c[0], c[1], c[2], c[3]), int8x4(c[4], c[5], c[6], c[7]));
    *reinterpret_cast<uint2*>(dst + k) = bad ? make_uint2(0, 0) : out;
  };
#pragma unroll
  for (int i = 0; i < kInt8Pieces; ++i)
    if (first + i * step < end) put(v[i], first + i * step);
  for (unsigned k = first + kInt8Pieces * step; k < end; k += step) {
    Eight<T> more;
    load_eight<VEC>(more, src + k, (int)min(8u, end - k));
    put(more, k);
  }
}

// Codes of x^T [K, M] of x [M, K].  A cluster of `parts` CTAs has 64 columns and shares out the rows; each keeps the last 256 of its own in
// registers, thread (rg, cg) rows 8 rg .. 8 rg + 7 of each 256 and columns 8 cg .. 8 cg + 7, and reads what is before them twice, from L2 the
// second time: four CTAs to a strip, since of one to a strip what all have under way is more than L2 holds (2880 x 5760 of 32 experts: 410 us,
// two 379, four 344, eight 539; 512 rows each in registers, clusters of six: 373).
// Codes are parked as [64 columns][256 rows] with the 8-byte units of a column permuted (unit rg lies at rg ^ 4 cg), so that the eight
// columns that a warp writes at a time fall on different banks.
constexpr int kInt8MaxParts = 4;
inline int int8_parts(int64_t M) { return (int)std::max<int64_t>(1, std::min<int64_t>(kInt8MaxParts, ceil_div(M, 256))); }      // (x without rows: scales alone)
__host__ __device__ constexpr int64_t int8_part_rows(int64_t M, int parts) { return ((M + parts - 1) / parts + 15) & ~(int64_t)15; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(256, VEC && sizeof(T) == 2 ? 4 : 2)
int8_columns_quantize_kernel(const T* x, const Int8Out d, int64_t M, int64_t K, int parts) {
  constexpr int kWords = sizeof(T) == 2 ? 4 : 8;      // largest magnitudes of eight columns: bf16 two to a word
  __shared__ __align__(16) uint8_t s_parked[2][64 * 256];
  __shared__ uint32_t s_max[8][8 * kWords];
  __shared__ uint32_t s_top[64];
  __shared__ float s_inv[64];
  __shared__ uint32_t s_keep[64];
  const int cg = threadIdx.x & 7, rg = threadIdx.x >> 3, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned part = cluster_ctarank();
  const int64_t rows = int8_part_rows(M, parts), first = part * rows, end = min(M, first + rows);
  const int64_t held = first + (rows - 1) / 256 * 256;         // rows from here on stay in registers
  const int64_t c0 = (int64_t)(blockIdx.x / parts) * 64, k = c0 + 8 * cg;
  const int columns = (int)max((int64_t)0, min((int64_t)8, K - k));
  pdl_trigger();
  pdl_wait();
  const T* src = after_wait(x) + (int64_t)blockIdx.y * M * K + k;
  Eight<T> v[8];
  auto load = [&](int64_t m) {
    const T* p = src + m * K;
#pragma unroll
    for (int i = 0; i < 8; ++i, p += K) load_eight<VEC>(v[i], p, m + i < end ? columns : 0);
  };
  uint32_t most[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j) most[j] = 0;
  for (int64_t m0 = first; m0 <= held; m0 += 256) {
    load(m0 + 8 * rg);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].most_by_column(most);
  }
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, most[j], o);
      most[j] = sizeof(T) == 2 ? __vmaxu2(most[j], other) : max(most[j], other);
    }
    if (lane < 8) s_max[warp][kWords * cg + j] = most[j];
  }
  __syncthreads();
  const int c = threadIdx.x;               // (below 64: a column)
  if (c < 64) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t two = s_max[w][c >> 1];
        top = max(top, (c & 1) ? two & 0xffff0000u : two << 16);
      } else {
        top = max(top, s_max[w][c]);
      }
    }
    s_top[c] = top;
  }
  cluster_sync_all();
  if (c < 64) {
    const uint32_t at = smem_addr_u32(s_top + c);
    uint32_t top = 0;
    for (int o = 0; o < parts; ++o) top = max(top, __float_as_uint(ld_shared_cluster_f32(mapa_u32(at, (uint32_t)o))));
    s_inv[c] = int8_inverse(top);
    s_keep[c] = int8_bad(top) ? 0u : 0xffffffffu;
    if (part == 0 && c0 + c < K) d.scale[blockIdx.y * d.scale_batch + (c0 + c) * d.scale_row] = int8_scale(top);
  }
  cluster_sync_all();                      // (also: no CTA ends before the others have read its maxima)
  uint8_t* dst = d.q + blockIdx.y * d.q_batch;
  int turn = 0;
  auto put = [&](int64_t m0) {
    uint8_t* s_codes = s_parked[turn];
    turn ^= 1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = s_inv[8 * cg + j];
      const uint32_t keep = s_keep[8 * cg + j];
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = int8_code(v[i].value(j), f);
      *reinterpret_cast<uint2*>(s_codes + (8 * cg + j) * 256 + ((rg ^ (cg << 2)) << 3)) =
          make_uint2(int8x4(q[0], q[1], q[2], q[3]) & keep, int8x4(q[4], q[5], q[6], q[7]) & keep);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 16 * i + (threadIdx.x >> 4), u = threadIdx.x & 15;      // 16 bytes: rows m0 + 16 u ...
      const uint4 q = *reinterpret_cast<const uint4*>(s_codes + col * 256 + (((2 * u) ^ ((col >> 3) << 2)) << 3));
      if (c0 + col < K && m0 + 16 * u < end) __stcs(reinterpret_cast<uint4*>(dst + (c0 + col) * d.ld + m0 + 16 * u), q);
    }
  };
  put(held);
  for (int64_t m0 = held - 256; m0 >= first; m0 -= 256) {      // backwards: L2 holds the last ones best
    load(m0 + 8 * rg);
    put(m0);
  }
}

constexpr int64_t kMostGridRows = 65535;
template <typename T>
inline int launch_int8_quantize(const T* x, Int8Out d, int64_t B, int64_t M, int64_t K, bool transpose, cudaStream_t st) {
  for (; B > kMostGridRows; B -= kMostGridRows) {      // a matrix is a row of the grid
    const int rc = launch_int8_quantize(x, d, kMostGridRows, M, K, transpose, st);
    if (rc) return rc;
    x += kMostGridRows * M * K;
    d.q += kMostGridRows * d.q_batch;
    d.scale += kMostGridRows * d.scale_batch;
  }
  const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (transpose) {
    const int64_t strips = ceil_div(K, 64);
    if (strips * kInt8MaxParts > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
    auto kern = vec ? int8_columns_quantize_kernel<T, true> : int8_columns_quantize_kernel<T, false>;
    const int parts = int8_parts(M);
    return launch_clusters(kern, parts, true, dim3((unsigned)(strips * parts), (unsigned)B), dim3(256), 0, st, x, d, M, K, parts);
  }
  int log_wpr = 0;
  while ((1 << log_wpr) < kInt8RowWarps && K > (kInt8Pieces * 256) << log_wpr) ++log_wpr;
  const int64_t ctas = ceil_div(M, kInt8RowWarps >> log_wpr);
  if (ctas > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  auto kern = vec ? int8_rows_quantize_kernel<T, true> : int8_rows_quantize_kernel<T, false>;
  return launch_behind(kern, dim3((unsigned)ctas, (unsigned)B), dim3(kInt8RowWarps * 32), 0, st, x, d, M, (int)K, log_wpr);
}

}  // namespace yb
