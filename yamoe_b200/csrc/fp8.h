// 8-bit kernels as the other translation unit calls them (host side).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/yamoe_b200.h"

namespace yb {

// A matrix that the calls of this library read or write: pitches and alignment as the header asks
bool fp8_matrix_ok(const yamoe_fp8_matrix_t* m, int64_t batch, int64_t cols);
// The same as tensor maps want it besides: the matrices of `rows` rows one behind the other, a whole number of pitches apart
bool fp8_maps_ok(const yamoe_fp8_matrix_t* m, int64_t batch, int64_t rows);

// hidden [T, H] -> codes [rows, ld] and scales [groups, scale_group] at the rows of each token's K assignments
template <typename T>
int fp8_gather(const T* hidden, uint8_t* q, float* scale, int64_t ld, int64_t scale_group, const int32_t* flat_row, int64_t tokens,
               int H, int K, cudaStream_t st);

// The two grouped products of the expert pass over rows in the padded, expert-sorted layout.
struct Fp8Rows {
  const int32_t* pad_off;
  const int32_t* header;        // row tiles, status
  const int32_t* row_token;
  const float* row_weight;
  int64_t max_rows, max_tiles;
};
template <typename T>
int fp8_gate_up(const Fp8Rows& r, const uint8_t* x, const float* x_scale, int64_t ld, const yamoe_fp8_matrix_t& w, const T* bias,
                uint8_t* act, float* act_scale, int H, int E, cudaStream_t st);
template <typename T>
int fp8_down(const Fp8Rows& r, const uint8_t* act, const float* act_scale, int64_t ld, const yamoe_fp8_matrix_t& w, const T* bias,
             float* y, int H, int E, cudaStream_t st);

}  // namespace yb
