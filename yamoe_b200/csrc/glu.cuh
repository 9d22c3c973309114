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

// 1 / (1 + exp(-1.702 g)) as IEEE has it
__device__ __forceinline__ float glu_sigmoid(float g) { return __fdiv_rn(1.f, 1.f + expf(-kAlpha * g)); }
// Two of them by the approximate forms
__device__ __forceinline__ uint64_t glu_sigmoid_f32x2(uint64_t g) {
  constexpr float kLog2 = -kAlpha * 1.4426950408889634f;             // exp(x) = 2^(x log2 e)
  float x, y;
  unpack_f32x2(mul_f32x2(g, pack_f32x2(kLog2, kLog2)), x, y);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
  unpack_f32x2(add_f32x2(pack_f32x2(x, y), pack_f32x2(1.f, 1.f)), x, y);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(y));
  return pack_f32x2(x, y);
}

// The GLU of two gate / up pairs
template <typename T>
__device__ __forceinline__ void glu_two(const float (&gate)[2], const float (&up)[2], float (&y)[2]) {
  const float g[2] = {clamp_gate(gate[0]), clamp_gate(gate[1])}, u[2] = {clamp_up(up[0]), clamp_up(up[1])};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) y[i] = (u[i] + 1.f) * (g[i] * glu_sigmoid(g[i]));
  } else {
    const uint64_t gg = pack_f32x2(g[0], g[1]), v = add_f32x2(pack_f32x2(u[0], u[1]), pack_f32x2(1.f, 1.f));
    unpack_f32x2(mul_f32x2(v, mul_f32x2(gg, glu_sigmoid_f32x2(gg))), y[0], y[1]);
  }
}
// Its gradients, d those of the results
template <typename T>
__device__ __forceinline__ void glu_two_backward(const float (&gate)[2], const float (&up)[2], const float (&d)[2], float (&d_gate)[2],
                                                 float (&d_up)[2]) {
  const float g[2] = {clamp_gate(gate[0]), clamp_gate(gate[1])}, u[2] = {clamp_up(up[0]), clamp_up(up[1])};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float s = glu_sigmoid(g[i]), y = g[i] * s;
      d_gate[i] = d[i] * (u[i] + 1.f) * (s + kAlpha * y * (1.f - s));
      d_up[i] = d[i] * y;
    }
  } else {
    const uint64_t one = pack_f32x2(1.f, 1.f), gg = pack_f32x2(g[0], g[1]), s = glu_sigmoid_f32x2(gg), y = mul_f32x2(gg, s),
                   dd = pack_f32x2(d[0], d[1]), v = add_f32x2(pack_f32x2(u[0], u[1]), one);
    const uint64_t rest = fma_f32x2(s, pack_f32x2(-1.f, -1.f), one), slope = fma_f32x2(mul_f32x2(y, rest), pack_f32x2(kAlpha, kAlpha), s);
    unpack_f32x2(mul_f32x2(mul_f32x2(dd, v), slope), d_gate[0], d_gate[1]);
    unpack_f32x2(mul_f32x2(dd, y), d_up[0], d_up[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (gate[i] > kLimit) d_gate[i] = 0.f;
    if (fabsf(up[i]) > kLimit) d_up[i] = 0.f;
  }
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
    for (int j = 0; j < 4; j += 2) {
      const float gate[2] = {v[i].value(2 * j), v[i].value(2 * j + 2)}, up[2] = {v[i].value(2 * j + 1), v[i].value(2 * j + 3)};
      float two[2];
      glu_two<T>(gate, up, two);
      y[j] = two[0];
      y[j + 1] = two[1];
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
    for (int j = 0; j < 4; j += 2) {
      float gate[2], up[2], d_gate[2], d_up[2];
      const uint32_t word = j < 2 ? code[i].x : code[i].y;
      e4m3x2_values(word, gate[0], up[0]);
      e4m3x2_values(word >> 16, gate[1], up[1]);
      const uint64_t scale = pack_f32x2(s[i], s[i]);
      unpack_f32x2(mul_f32x2(pack_f32x2(gate[0], up[0]), scale), gate[0], up[0]);
      unpack_f32x2(mul_f32x2(pack_f32x2(gate[1], up[1]), scale), gate[1], up[1]);
      const float two[2] = {d[i][j], d[i][j + 1]};
      glu_two_backward<T>(gate, up, two, d_gate, d_up);
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        out[2 * (j + o)] = d_gate[o];
        out[2 * (j + o) + 1] = d_up[o];
      }
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
