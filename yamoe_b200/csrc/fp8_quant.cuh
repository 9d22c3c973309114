// Quantisation to e4m3 in groups of 128: the operands of the 8-bit products (fp8_gemm.cuh).
//
//   a = max |x| over the group, at least 2^-100 (a NaN among the values makes a NaN)
//   scale = a / 448,   q = e4m3(x * (448 / a))         448 is the largest e4m3 value; nearest, ties to even
//
// with 32-bit divisions and products, so that every value has one definite code: a value equal to the largest becomes
// +-448 whatever way the two divisions are rounded.  A group is 128 neighbours in a row (activations, gradients) or
// 128 x 128 values (weights), the last ones of a matrix being smaller.
//
// The kernels may start before what writes x has ended: x is read by ordinary loads behind the wait for it.  The one exception
// is the gather of the expert pass, which reads the token rows before its wait: the kernel before it is the routing's, a
// plain launch, which began when all that went before it had ended; only its tables are waited for.
//
// Bound by HBM: a value is read once and its code written once, 3 bytes for bf16.  Rows (groups of 1 x 128) need no
// exchange beyond 16 lanes, which hold a group; blocks and transposed outputs go by tiles of 128 x 128 values held in
// the registers of a CTA, codes turned around in shared memory.
// Rows: 4096 x 2880 of bf16 8.6 us (4.1 TB/s, 3 us of it the launch).  Tiles: the transposed codes of the bf16 weights of
// 32 experts (2880 x 5760), 1.6 GB read and written, 246 us (6.5 TB/s).
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

// Eight neighbouring values of a row as loaded, of which `n` exist (the others 0); VEC: 16-byte loads, rows being aligned to them.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
  uint4 q;
  template <bool VEC>
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n) {
    if (VEC && n >= 8) {
      q = ld_written(reinterpret_cast<const uint4*>(p));
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (2 * j < n ? (uint32_t)h[2 * j] : 0u) | (2 * j + 1 < n ? (uint32_t)h[2 * j + 1] << 16 : 0u);
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ uint32_t word(int j) const { return j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w; }
  __device__ __forceinline__ float value(int j) const {
    const uint32_t w = word(j >> 1);
    return __uint_as_float((j & 1) ? w & 0xffff0000u : w << 16);
  }
  // two magnitudes at a time: as 16-bit numbers they are ordered like the values, NaN above all
  __device__ __forceinline__ uint32_t most() const {
    const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu), __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu));
    return max(m & 0xffff0000u, m << 16);
  }
  __device__ __forceinline__ void most_by_column(uint32_t (&m)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = __vmaxu2(m[j], word(j) & 0x7fff7fffu);
  }
};
template <> struct Eight<float> {
  float4 q[2];
  template <bool VEC>
  __device__ __forceinline__ void load(const float* p, int n) {
    if (VEC && n >= 8) {
      q[0] = *reinterpret_cast<const float4*>(p);
      q[1] = *(reinterpret_cast<const float4*>(p) + 1);
    } else {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
  __device__ __forceinline__ float value(int j) const {
    const float4& r = q[j >> 2];
    return (j & 3) == 0 ? r.x : (j & 3) == 1 ? r.y : (j & 3) == 2 ? r.z : r.w;
  }
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(value(j)));
    return m;
  }
  __device__ __forceinline__ void most_by_column(uint32_t (&m)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = max(m[j], abs_bits(value(j)));
  }
};
template <class E>
__device__ __forceinline__ uint2 fp8_codes(const E& e, float inv) {
  return make_uint2(e4m3x4(e.value(0) * inv, e.value(1) * inv, e.value(2) * inv, e.value(3) * inv),
                    e4m3x4(e.value(4) * inv, e.value(5) * inv, e.value(6) * inv, e.value(7) * inv));
}

// ---- rows: groups of 1 x 128 --------------------------------------------------------------------------------------
// A half warp holds a group, eight values to a lane; a warp takes up to kQuantPairs neighbouring pairs of groups of one row, whose loads
// are in flight together.  With `flat_row` a row is a token and goes to the rows of its K assignments (negative: dropped),
// read once.
constexpr int kQuantWarps = 8, kQuantPairs = 4;
// What a warp takes of a row.  A row may have up to 2^31 - 1 values: rounding up passes 31 bits.
constexpr int kQuantPiece = 2 * kQuantPairs * kFp8Group;
__host__ __device__ constexpr unsigned quant_pieces(int K) { return ((unsigned)K + kQuantPiece - 1) / kQuantPiece; }
static_assert(quant_pieces(0x7fffffff) == 1u << 21 && quant_pieces(1) == 1, "");

struct QuantRows {
  uint8_t* q;          // [.., ldq]
  float* scale;        // (matrix, row, group) at matrix * scale_batch + row * scale_row + group * scale_group
  int64_t ldq, q_batch, scale_row, scale_group, scale_batch;
  const int32_t* flat_row;
  int slots;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32)
quantize_rows_kernel(const T* x, const QuantRows d, int64_t rows, int K) {
  pdl_trigger();
  const int lane = threadIdx.x & 31, l16 = lane & 15;
  // the pieces of a row are neighbours in the grid
  const unsigned pieces = quant_pieces(K);
  const unsigned unit = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  const int64_t row = unit / pieces;
  const int k0 = (int)(unit - (unsigned)row * pieces) * kQuantPiece + lane * 8;
  if (row >= rows) return;
  // Of the expert pass only the tables come from the kernel before this one, a plain launch: x was there when that one began.
  if (d.flat_row == nullptr) pdl_wait();
  const T* src = after_wait(x) + ((int64_t)blockIdx.y * rows + row) * K;
  Eight<T> v[kQuantPairs];
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) v[i].template load<VEC>(src + k0 + i * 2 * kFp8Group, K - k0 - i * 2 * kFp8Group);
  if (d.flat_row != nullptr) pdl_wait();
  const int32_t* flat_row = d.flat_row != nullptr ? after_wait(d.flat_row) : nullptr;
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) {
    const int k = k0 + i * 2 * kFp8Group;
    if (k - lane * 8 >= K) break;
    uint32_t most = v[i].most();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (k >= K) continue;
    const float a = fp8_group_max(most), s = fp8_scale(a);
    const uint2 out = fp8_codes(v[i], fp8_inverse(a));
    if (flat_row == nullptr) {
      *reinterpret_cast<uint2*>(d.q + blockIdx.y * d.q_batch + row * d.ldq + k) = out;
      if (l16 == 0) d.scale[blockIdx.y * d.scale_batch + row * d.scale_row + (k / kFp8Group) * d.scale_group] = s;
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
__global__ void __launch_bounds__(256, sizeof(T) == 2 && VEC ? 4 : 2)
quantize_tile_kernel(const T* x, int64_t batch_stride, int M, int K, const QuantOut out, const QuantOut turned) {
  constexpr int kWords = sizeof(T) == 2 ? 4 : 8;           // largest magnitudes of eight columns: bf16 two to a word
  __shared__ __align__(16) uint8_t s_codes[128 * 128];
  __shared__ uint32_t s_max[8][16 * kWords];
  __shared__ float s_inv[128];
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m0 = blockIdx.y * 128, k0 = blockIdx.x * 128;
  const int64_t b = blockIdx.z;
  const int m = m0 + 8 * rg, k = k0 + 8 * cg;
  pdl_trigger();
  pdl_wait();
  x = after_wait(x);
  Eight<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i].template load<VEC>(x + b * batch_stride + (int64_t)(m + i) * K + k, m + i < M ? K - k : 0);

  float inv_block = 0.f;
  if constexpr (BLOCK) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, v[i].most());
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) s_max[0][warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, s_max[0][w]);
    const float a = fp8_group_max(most);
    inv_block = fp8_inverse(a);
    if (threadIdx.x == 0) {
      const float s = fp8_scale(a);
      if (out.q != nullptr) out.scale[b * out.scale_batch + blockIdx.y * out.scale_row + blockIdx.x * out.scale_group] = s;
      if (turned.q != nullptr)
        turned.scale[b * turned.scale_batch + blockIdx.x * turned.scale_row + blockIdx.y * turned.scale_group] = s;
    }
  } else if (turned.q != nullptr) {
    uint32_t most[kWords];
#pragma unroll
    for (int j = 0; j < kWords; ++j) most[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].most_by_column(most);
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, most[j], 16);       // the other row group of this warp
      most[j] = sizeof(T) == 2 ? __vmaxu2(most[j], other) : max(most[j], other);
      if (lane < 16) s_max[warp][kWords * cg + j] = most[j];
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      const int c = threadIdx.x;
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
      const float a = fp8_group_max(top);
      s_inv[c] = fp8_inverse(a);
      if (k0 + c < K)
        turned.scale[b * turned.scale_batch + (int64_t)(k0 + c) * turned.scale_row + blockIdx.y * turned.scale_group] = fp8_scale(a);
    }
  }
  if (out.q != nullptr) {
    float inv = inv_block;
    if constexpr (!BLOCK) {
      // lane cg of the sixteen that hold a row takes up row cg's division
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t most = v[i].most();
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (cg == i) mine = most;
      }
      const float a = fp8_group_max(mine);
      inv = fp8_inverse(a);
      if (cg < 8 && m + cg < M)
        out.scale[b * out.scale_batch + (int64_t)(m + cg) * out.scale_row + blockIdx.x * out.scale_group] = fp8_scale(a);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = BLOCK ? inv : __shfl_sync(0xffffffffu, inv, (lane & 16) + i);
      if (m + i < M && k < K) *reinterpret_cast<uint2*>(out.q + b * out.q_batch + (int64_t)(m + i) * out.ld + k) = fp8_codes(v[i], f);
    }
  }
  if (turned.q == nullptr) return;
  if constexpr (!BLOCK) __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = BLOCK ? inv_block : s_inv[8 * cg + j];
    uint2 c;
    c.x = e4m3x4(v[0].value(j) * f, v[1].value(j) * f, v[2].value(j) * f, v[3].value(j) * f);
    c.y = e4m3x4(v[4].value(j) * f, v[5].value(j) * f, v[6].value(j) * f, v[7].value(j) * f);
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

// `batch` matrices of `rows` rows
template <typename T>
inline int launch_quantize_rows(const T* x, const QuantRows& d, int64_t batch, int64_t rows, int K, cudaStream_t st) {
  const int64_t ctas = ceil_div(rows * quant_pieces(K), kQuantWarps);
  if (ctas == 0 || batch == 0) return YAMOE_OK;
  if (ctas * kQuantWarps > 0x7fffffff || batch > 65535) return YAMOE_ERR_UNSUPPORTED;
  auto kern = rows_of_16_bytes<T>(x, K) ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
  const cudaError_t rc = launch_early(kern, dim3((unsigned)ctas, (unsigned)batch), dim3(kQuantWarps * 32), st, x, d, rows, K);
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
  const cudaError_t rc = launch_early(kern, grid, dim3(256), st, x, M * K, (int)M, (int)K, out, turned);
  return rc == cudaSuccess && cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
