// The clamped GLU of the expert pass as an operator of its own, whose backward pass keeps its inputs in 8 bits.
//
//   g = min(gate, 7), u = clamp(up, -7, 7), s = 1 / (1 + exp(-1.702 g)):   y = (u + 1) g s         gate, up: even and odd columns
//   d_gate = dy (u + 1) s (1 + 1.702 g (1 - s)), 0 where gate > 7;   d_up = dy g s, 0 where |up| > 7
//
// The checkpoint is the e4m3 codes of the pre-activations in groups of 1 x 128 with an fp32 scale each (fp8_quant.cuh has the definition):
// 2 N + 8 N / 128 ... bytes per row instead of 4 N (bf16) or 8 N (fp32).  The backward pass takes the GLU's derivative at the values
// that the codes stand for.  Scales lie with a row's groups side by side, since only rows are ever read.
//
// Bound by HBM: one pass each way.  Half a warp holds a group, four gate / up pairs to a lane, four such pairs of groups per warp on
// their way together, as in the quantisation of rows.  fp32 calls exp and divides as IEEE has it; for bf16 results the approximate
// forms (2^-21) are far below half a step.
#pragma once
#include "int8_quant.cuh"

namespace yb {

template <typename T>
__device__ __forceinline__ float glu_sigmoid(float g) {
  if constexpr (sizeof(T) == 4) return __fdiv_rn(1.f, 1.f + expf(-kAlpha * g));
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * (-kAlpha * 1.4426950408889634f)));      // exp(x) = 2^(x log2 e)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}

struct GluSaved {
  uint8_t* q;            // [M, ld]; null: not kept
  float* scale;          // [M, groups]
  int64_t ld;
};

// four results to a row of N, of which `n` exist (VEC: all)
template <typename T, bool VEC>
__device__ __forceinline__ void put_four(T* p, const float (&v)[4], int n) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) DT<T>::st(p + j, v[j]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void get_four(const T* p, float (&v)[4], int n) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 2) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(q.x << 16);
      v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16);
      v[3] = __uint_as_float(q.y & 0xffff0000u);
    } else {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? DT<T>::ld(p + j) : 0.f;
  }
}

// pre [M, W], W = 2 N; out [M, N]
template <typename T, bool VEC, bool SAVE>
__global__ void __launch_bounds__(kQuantWarps * 32)
glu_forward_kernel(const T* pre, T* out, const GluSaved saved, int64_t M, int W) {
  pdl_trigger();
  const int lane = threadIdx.x & 31, l16 = lane & 15;
  const unsigned pieces = quant_pieces(W);
  const unsigned unit = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  const int64_t row = unit / pieces;
  const int k0 = (int)(unit - (unsigned)row * pieces) * kQuantPiece + lane * 8;
  if (row >= M) return;
  pdl_wait();
  const T* src = after_wait(pre) + row * W;
  T* dst = out + row * (W / 2);
  Eight<T> v[kQuantPairs];
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) load_eight<VEC>(v[i], src + k0 + i * 2 * kFp8Group, W - k0 - i * 2 * kFp8Group);
  float inv = 0.f;
  if constexpr (SAVE) {
    // lane i of the sixteen that hold a group takes up the divisions of their i-th
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kQuantPairs; ++i) {
      uint32_t most = v[i].most();
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (l16 == i) mine = most;
    }
    const float a = fp8_group_max(mine);
    const int group = k0 / kFp8Group + 2 * l16, groups = (W + kFp8Group - 1) / kFp8Group;      // (k0 / 128 is that of the half warp's first)
    inv = fp8_inverse(a);
    if (l16 < kQuantPairs && group < groups) saved.scale[row * groups + group] = fp8_scale(a);
  }
#pragma unroll
  for (int i = 0; i < kQuantPairs; ++i) {
    const int k = k0 + i * 2 * kFp8Group;
    const float f = SAVE ? __shfl_sync(0xffffffffu, inv, (lane & 16) + i) : 0.f;
    if (k >= W) continue;
    if constexpr (SAVE) *reinterpret_cast<uint2*>(saved.q + row * saved.ld + k) = fp8_codes(v[i], f);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float g = clamp_gate(v[i].value(2 * j)), u = clamp_up(v[i].value(2 * j + 1));
      y[j] = (u + 1.f) * (g * glu_sigmoid<T>(g));
    }
    put_four<T, VEC>(dst + k / 2, y, (W - k) / 2);
  }
}

__device__ __forceinline__ void e4m3x2_values(uint32_t two, float& lo, float& hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}

// What a warp of the backward pass takes of a row: two pairs of groups, with which eight CTAs fit an SM (32768 x 5760 bf16: 148 us, four
// pairs 161, one 165).
constexpr int kGluBackPairs = 2, kGluBackPiece = 2 * kGluBackPairs * kFp8Group;
__host__ __device__ constexpr unsigned glu_back_pieces(int W) { return ((unsigned)W + kGluBackPiece - 1) / kGluBackPiece; }

// dy [M, N], d_pre [M, W]
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32, sizeof(T) == 2 ? 8 : 4)
glu_backward_kernel(const T* dy, const uint8_t* q, const float* scale, int64_t ld, T* d_pre, int64_t M, int W) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const unsigned pieces = glu_back_pieces(W);
  const unsigned unit = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
  const int64_t row = unit / pieces;
  const int k0 = (int)(unit - (unsigned)row * pieces) * kGluBackPiece + lane * 8;
  if (row >= M) return;
  pdl_wait();
  const T* dsrc = after_wait(dy) + row * (W / 2);
  const uint8_t* qsrc = after_wait(q) + row * ld;
  const float* ssrc = after_wait(scale) + row * ((W + kFp8Group - 1) / kFp8Group);
  T* dst = d_pre + row * W;
  uint2 code[kGluBackPairs];
  float s[kGluBackPairs], d[kGluBackPairs][4];
#pragma unroll
  for (int i = 0; i < kGluBackPairs; ++i) {
    const int k = k0 + i * 2 * kFp8Group;
    if (k >= W) break;
    code[i] = *reinterpret_cast<const uint2*>(qsrc + k);
    s[i] = ssrc[k / kFp8Group];
    get_four<T, VEC>(dsrc + k / 2, d[i], (W - k) / 2);
  }
#pragma unroll
  for (int i = 0; i < kGluBackPairs; ++i) {
    const int k = k0 + i * 2 * kFp8Group;
    if (k >= W) break;
    float out[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float gate, up;
      e4m3x2_values((j < 2 ? code[i].x : code[i].y) >> (16 * (j & 1)), gate, up);
      gate *= s[i];
      up *= s[i];
      const float g = clamp_gate(gate), u = clamp_up(up), sig = glu_sigmoid<T>(g), y = g * sig;
      out[2 * j] = gate > kLimit ? 0.f : d[i][j] * (u + 1.f) * (sig + kAlpha * y * (1.f - sig));
      out[2 * j + 1] = fabsf(up) > kLimit ? 0.f : d[i][j] * y;
    }
    if constexpr (VEC) {
      if constexpr (sizeof(T) == 2) {
        uint32_t two[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(out[2 * j], out[2 * j + 1]);
          two[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(dst + k) = make_uint4(two[0], two[1], two[2], two[3]);
      } else {
        *reinterpret_cast<float4*>(dst + k) = make_float4(out[0], out[1], out[2], out[3]);
        *reinterpret_cast<float4*>(dst + k + 4) = make_float4(out[4], out[5], out[6], out[7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < W) DT<T>::st(dst + k + j, out[j]);
    }
  }
}

template <typename T>
inline int launch_glu_forward(const T* pre, T* out, const GluSaved& saved, int64_t M, int W, cudaStream_t st) {
  const int64_t units = M * quant_pieces(W), ctas = ceil_div(units, kQuantWarps);
  if (units > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  const bool vec = W % 8 == 0 && ((reinterpret_cast<uintptr_t>(pre) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto kern = saved.q != nullptr ? (vec ? glu_forward_kernel<T, true, true> : glu_forward_kernel<T, false, true>)
                                 : (vec ? glu_forward_kernel<T, true, false> : glu_forward_kernel<T, false, false>);
  return launch_behind(kern, dim3((unsigned)ctas), dim3(kQuantWarps * 32), 0, st, pre, out, saved, M, W);
}

template <typename T>
inline int launch_glu_backward(const T* dy, const uint8_t* q, const float* scale, int64_t ld, T* d_pre, int64_t M, int W, cudaStream_t st) {
  const int64_t units = M * glu_back_pieces(W), ctas = ceil_div(units, kQuantWarps);
  if (units > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  const bool vec = W % 8 == 0 && ((reinterpret_cast<uintptr_t>(d_pre) | reinterpret_cast<uintptr_t>(dy)) & 15) == 0;
  auto kern = vec ? glu_backward_kernel<T, true> : glu_backward_kernel<T, false>;
  return launch_behind(kern, dim3((unsigned)ctas), dim3(kQuantWarps * 32), 0, st, dy, q, scale, ld, d_pre, M, W);
}

}  // namespace yb
