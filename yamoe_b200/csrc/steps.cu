// The steps of the expert layer as operators of their own: tokens sorted by expert and back, products of 8-bit integers, the GLU with
// an 8-bit checkpoint.  C entry points.
#include "glu.cuh"
#include "int8_gemm.cuh"
#include "int8_quant.cuh"
#include "token_sort.cuh"

namespace yb {

static bool known_dtype(int dtype) { return dtype == YAMOE_F32 || dtype == YAMOE_BF16; }
static size_t size_of(int dtype) { return dtype == YAMOE_F32 ? 4 : 2; }
static bool at_boundary(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
static bool workspace_ok(const void* ws, size_t bytes, size_t needed) {
  return needed == 0 || (ws != nullptr && at_boundary(ws, 256) && bytes >= needed);
}
constexpr int64_t kMaxAssignments = (int64_t)1 << 30, kMaxRows = ((int64_t)1 << 31) - 1, kMaxExtent = (int64_t)1 << 40;
// T tokens of K assignments
static bool countable(int64_t T, int K) { return T <= kMaxRows && T * K < kMaxAssignments; }

static bool int8_matrix_ok(const yamoe_int8_matrix_t* m, int64_t batch, int64_t cols) {
  if (m == nullptr || m->q == nullptr || m->scale == nullptr || !at_boundary(m->q, 16) || !at_boundary(m->scale, 4)) return false;
  if (m->ld < cols || m->ld % 16 != 0 || m->ld >= kMaxExtent) return false;
  return batch <= 1 || (m->q_batch > 0 && m->q_batch % 16 == 0 && m->q_batch < kMaxExtent);
}
// as tensor maps want it besides
static bool int8_maps_ok(const yamoe_int8_matrix_t* m, int64_t batch, int64_t rows) {
  return batch <= 1 || (m->q_batch % m->ld == 0 && m->q_batch / m->ld >= rows);
}

// What the combine and its gradients have in common, of one pair of types.
struct CombineCall {
  const void *rows, *weights;
  const int32_t* row_of;
  const int64_t* indices;
  int64_t T, n_rows, H;
  int E, K;
  template <typename TT, typename TW>
  CombineArgs<TT, TW> args() const {
    return CombineArgs<TT, TW>{reinterpret_cast<const TT*>(rows), row_of, reinterpret_cast<const TW*>(weights), indices, T, n_rows, (int)H, K, E};
  }
};

template <typename T, typename TW>
static int combine_impl(const CombineCall& c, void* out, cudaStream_t st) {
  const auto a = c.args<T, TW>();
  T* o = reinterpret_cast<T*>(out);
  if (pieces_of(16, c.H * sizeof(T), {c.rows, out})) return launch_combine_tokens_ve<T, TW, 16 / sizeof(T)>(a, o, st);
  if constexpr (sizeof(T) == 2)
    if (pieces_of(4, c.H * sizeof(T), {c.rows, out})) return launch_combine_tokens_ve<T, TW, 2>(a, o, st);
  return launch_combine_tokens_ve<T, TW, 1>(a, o, st);
}
template <typename T, typename TW>
static int combine_backward_impl(const CombineCall& c, const void* d_out, void* d_rows, void* d_weights, int32_t* head, int32_t* next,
                                 cudaStream_t st) {
  const auto a = c.args<T, TW>();
  const T* g = reinterpret_cast<const T*>(d_out);
  T* dr = reinterpret_cast<T*>(d_rows);
  TW* dw = reinterpret_cast<TW*>(d_weights);
  if (pieces_of(16, c.H * sizeof(T), {c.rows, d_out, d_rows}))
    return launch_combine_backward_ve<T, TW, 16 / sizeof(T)>(a, g, dr, dw, head, next, st);
  if constexpr (sizeof(T) == 2)
    if (pieces_of(4, c.H * sizeof(T), {c.rows, d_out, d_rows})) return launch_combine_backward_ve<T, TW, 2>(a, g, dr, dw, head, next, st);
  return launch_combine_backward_ve<T, TW, 1>(a, g, dr, dw, head, next, st);
}

// the arguments that both have
static int check_combine(const CombineCall& c, int weight_dtype, int dtype) {
  if (!known_dtype(dtype) || (c.weights != nullptr && weight_dtype != dtype && weight_dtype != YAMOE_F32)) return YAMOE_ERR_DTYPE;
  if (c.T < 0 || c.n_rows < 0 || c.H < 0 || c.K < 0 || c.E < 0) return YAMOE_ERR_BAD_ARG;
  if (!countable(c.T, c.K) || c.H > kMaxRows || c.n_rows > kMaxRows) return YAMOE_ERR_UNSUPPORTED;
  const int64_t S = c.T * c.K;
  if (S > 0 && (c.row_of == nullptr || !at_boundary(c.row_of, 4))) return YAMOE_ERR_BAD_ARG;
  if (S > 0 && c.n_rows > 0 && c.H > 0 && (c.rows == nullptr || !at_boundary(c.rows, size_of(dtype)))) return YAMOE_ERR_BAD_ARG;
  if (c.weights != nullptr && !at_boundary(c.weights, size_of(weight_dtype))) return YAMOE_ERR_BAD_ARG;
  return at_boundary(c.indices, 8) ? YAMOE_OK : YAMOE_ERR_BAD_ARG;
}

template <typename T>
static int int8_mm_impl(const yamoe_int8_matrix_t& a, const yamoe_int8_matrix_t& b, const int32_t* offsets, void* out, int64_t batch,
                        int64_t M, int64_t N, int64_t K, int32_t* status, cudaStream_t st) {
  Int8Params<T> p{};
  p.M = M; p.N = (int)N; p.K = (int)K; p.B = (int)batch;
  p.sa = a.scale; p.sa_b = a.scale_batch; p.sa_m = a.scale_row;
  p.sb = b.scale; p.sb_b = b.scale_batch; p.sb_n = b.scale_row;
  p.offsets = offsets;
  p.out = reinterpret_cast<T*>(out);
  p.wide = sizeof(T) == 2 && N % 8 == 0 && at_boundary(out, 16);
  p.status = status;
  p.splits = 1;
  return launch_int8_mm(Int8Operand{a.q, M, a.ld, a.q_batch}, Int8Operand{b.q, N, b.ld, b.q_batch}, p, st);
}

}  // namespace yb

using namespace yb;

extern "C" {

size_t yamoe_b200_sort_tokens_workspace_bytes(int64_t T, int E, int K) {
  if (T < 0 || E <= 0 || E > kSortMaxExperts || K < 0 || !countable(T, K)) return 0;
  return 256 + sort_counts_bytes(T * K, E);
}

int yamoe_b200_sort_tokens(const void* hidden_states, const int64_t* router_indices, void* rows, int32_t* row_of, int32_t* offsets,
                           int64_t T, int64_t H, int E, int K, int64_t capacity, int dtype, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (!known_dtype(dtype)) return YAMOE_ERR_DTYPE;
  if (T < 0 || H < 0 || K < 0 || E <= 0) return YAMOE_ERR_BAD_ARG;
  if (E > kSortMaxExperts || H >= kMaxExtent || !countable(T, K)) return YAMOE_ERR_UNSUPPORTED;
  if (capacity > kMaxRows || (capacity >= 0 && capacity * E > kMaxRows)) return YAMOE_ERR_UNSUPPORTED;
  const int64_t S = T * K, R = capacity < 0 ? S : capacity * E;
  const size_t size = size_of(dtype);
  if (offsets == nullptr || !at_boundary(offsets, 4) || !at_boundary(row_of, 4) || !at_boundary(router_indices, 8)) return YAMOE_ERR_BAD_ARG;
  if (S > 0 && (router_indices == nullptr || row_of == nullptr)) return YAMOE_ERR_BAD_ARG;
  if (R > 0 && H > 0 && (rows == nullptr || !at_boundary(rows, size))) return YAMOE_ERR_BAD_ARG;
  if (S > 0 && H > 0 && (hidden_states == nullptr || !at_boundary(hidden_states, size))) return YAMOE_ERR_BAD_ARG;
  if (!workspace_ok(workspace, workspace_bytes, yamoe_b200_sort_tokens_workspace_bytes(T, E, K))) return YAMOE_ERR_WORKSPACE;
  SortArgs a{};
  a.indices = router_indices;
  a.hidden = reinterpret_cast<const uint8_t*>(hidden_states);
  a.rows = reinterpret_cast<uint8_t*>(rows);
  a.row_of = row_of;
  a.offsets = offsets;
  a.T = K > 0 ? T : 0; a.R = R; a.row_bytes = H * (int64_t)size;
  a.S = (int)S; a.E = E; a.K = K;
  while ((1 << a.bits) < E) ++a.bits;
  a.capacity = capacity < 0 ? -1 : (int)capacity;
  a.counts = reinterpret_cast<int32_t*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(hidden_states) | reinterpret_cast<uintptr_t>(rows) | (uintptr_t)a.row_bytes;
  return (bits & 15) == 0 ? launch_sort<uint4>(a, st) : (bits & 3) == 0 ? launch_sort<uint32_t>(a, st) : launch_sort<uint16_t>(a, st);
}

int yamoe_b200_combine_tokens(const void* rows, int64_t n_rows, const int32_t* row_of, const void* weights, int weight_dtype,
                              const int64_t* router_indices, void* out, int64_t T, int64_t H, int E, int K, int dtype, void* stream) {
  const CombineCall c{rows, weights, row_of, weights != nullptr ? router_indices : nullptr, T, n_rows, H, E, K};
  if (const int rc = check_combine(c, weight_dtype, dtype)) return rc;
  if (T == 0 || H == 0) return YAMOE_OK;
  if (out == nullptr || !at_boundary(out, size_of(dtype))) return YAMOE_ERR_BAD_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == YAMOE_F32) return combine_impl<float, float>(c, out, st);
  return weights != nullptr && weight_dtype == YAMOE_F32 ? combine_impl<__nv_bfloat16, float>(c, out, st)
                                                         : combine_impl<__nv_bfloat16, __nv_bfloat16>(c, out, st);
}

size_t yamoe_b200_combine_tokens_backward_workspace_bytes(int64_t n_rows, int64_t T, int K) {
  if (n_rows < 0 || T < 0 || K < 0 || n_rows > kMaxRows || !countable(T, K)) return 0;
  return 512 + (size_t)round_up(n_rows * 4, 256) + (size_t)(T * K) * 4;
}

int yamoe_b200_combine_tokens_backward(const void* d_out, const void* rows, int64_t n_rows, const int32_t* row_of, const void* weights,
                                       int weight_dtype, const int64_t* router_indices, void* d_rows, void* d_weights, int64_t T,
                                       int64_t H, int E, int K, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const CombineCall c{rows, weights, row_of, weights != nullptr ? router_indices : nullptr, T, n_rows, H, E, K};
  // (the rows themselves are read for the gradient of the weights only)
  CombineCall needed = c;
  if (d_weights == nullptr) needed.n_rows = 0;
  if (const int rc = check_combine(needed, weight_dtype, dtype)) return rc;
  if (n_rows < 0 || (d_weights != nullptr && (weights == nullptr || !at_boundary(d_weights, size_of(weight_dtype))))) return YAMOE_ERR_BAD_ARG;
  if (n_rows > kMaxRows || K > 1024) return YAMOE_ERR_UNSUPPORTED;
  if ((d_rows != nullptr && !at_boundary(d_rows, size_of(dtype))) || (T > 0 && H > 0 && (d_out == nullptr || !at_boundary(d_out, size_of(dtype)))))
    return YAMOE_ERR_BAD_ARG;
  if (!workspace_ok(workspace, workspace_bytes, yamoe_b200_combine_tokens_backward_workspace_bytes(n_rows, T, K))) return YAMOE_ERR_WORKSPACE;
  if (d_rows == nullptr && d_weights == nullptr) return YAMOE_OK;
  int32_t* head = reinterpret_cast<int32_t*>(workspace);
  int32_t* next = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(workspace) + 256 + round_up(n_rows * 4, 256));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == YAMOE_F32) return combine_backward_impl<float, float>(c, d_out, d_rows, d_weights, head, next, st);
  return weights != nullptr && weight_dtype == YAMOE_F32
             ? combine_backward_impl<__nv_bfloat16, float>(c, d_out, d_rows, d_weights, head, next, st)
             : combine_backward_impl<__nv_bfloat16, __nv_bfloat16>(c, d_out, d_rows, d_weights, head, next, st);
}

int yamoe_b200_int8_quantize(const void* x, const yamoe_int8_matrix_t* out, int64_t batch, int64_t M, int64_t K, int transpose, int dtype,
                             void* stream) {
  if (!known_dtype(dtype)) return YAMOE_ERR_DTYPE;
  if (batch < 0 || M < 0 || K < 0) return YAMOE_ERR_BAD_ARG;
  const int64_t rows = transpose ? K : M, cols = transpose ? M : K;
  if (batch == 0 || rows == 0) return YAMOE_OK;
  if (cols > 0 && (x == nullptr || !at_boundary(x, size_of(dtype)))) return YAMOE_ERR_BAD_ARG;
  if (!int8_matrix_ok(out, batch, cols)) return YAMOE_ERR_BAD_ARG;
  if (batch > kMaxRows || M > kMaxRows || K > kMaxRows) return YAMOE_ERR_UNSUPPORTED;
  const Int8Out d{reinterpret_cast<uint8_t*>(out->q), out->scale, out->ld, out->q_batch, out->scale_row, out->scale_batch};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == YAMOE_BF16 ? launch_int8_quantize(reinterpret_cast<const __nv_bfloat16*>(x), d, batch, M, K, transpose != 0, st)
                             : launch_int8_quantize(reinterpret_cast<const float*>(x), d, batch, M, K, transpose != 0, st);
}

size_t yamoe_b200_int8_mm_workspace_bytes(int64_t batch, int64_t M, int64_t N, int64_t K) {
  if (batch < 0 || M < 0 || N < 0 || K < 0) return 0;
  return 256;
}

int yamoe_b200_int8_mm(const yamoe_int8_matrix_t* a, const yamoe_int8_matrix_t* b, const int32_t* offsets, void* out, int64_t batch,
                       int64_t M, int64_t N, int64_t K, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!known_dtype(out_dtype)) return YAMOE_ERR_DTYPE;
  if (batch < 0 || M < 0 || N < 0 || K < 0 || !at_boundary(offsets, 4)) return YAMOE_ERR_BAD_ARG;
  const bool grouped = offsets != nullptr;
  if (M == 0 || N == 0 || (batch == 0 && !grouped)) return YAMOE_OK;
  const size_t size = size_of(out_dtype);
  if (out == nullptr || !at_boundary(out, size)) return YAMOE_ERR_BAD_ARG;
  // sums of 2^17 products of codes of -128 pass 31 bits; coordinates and tile counts are 32-bit numbers
  if (M >= (int64_t)1 << 30 || N >= (int64_t)1 << 30 || K >= (int64_t)1 << 17 || batch >= (int64_t)1 << 30) return YAMOE_ERR_UNSUPPORTED;
  if (grouped && batch > kInt8MaxExperts) return YAMOE_ERR_UNSUPPORTED;
  if (!workspace_ok(workspace, workspace_bytes, yamoe_b200_int8_mm_workspace_bytes(batch, M, N, K))) return YAMOE_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (K == 0 || batch == 0) {
    YB_CUDA_OK(cudaMemsetAsync(workspace, 0, 256, st));
    YB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)(grouped ? 1 : batch) * M * N * size, st));
    return YAMOE_OK;
  }
  const int64_t a_batch = grouped ? 1 : batch;
  if (!int8_matrix_ok(a, a_batch, K) || !int8_matrix_ok(b, batch, K) || !int8_maps_ok(a, a_batch, M) || !int8_maps_ok(b, batch, N))
    return YAMOE_ERR_BAD_ARG;
  int32_t* status = reinterpret_cast<int32_t*>(workspace) + 4;
  return out_dtype == YAMOE_BF16 ? int8_mm_impl<__nv_bfloat16>(*a, *b, offsets, out, batch, M, N, K, status, st)
                                 : int8_mm_impl<float>(*a, *b, offsets, out, batch, M, N, K, status, st);
}

int yamoe_b200_glu_forward(const void* pre, void* out, void* codes, float* scales, int64_t ld, int64_t M, int64_t N, int dtype,
                           void* stream) {
  if (!known_dtype(dtype)) return YAMOE_ERR_DTYPE;
  if (M < 0 || N < 0) return YAMOE_ERR_BAD_ARG;
  if (M == 0 || N == 0) return YAMOE_OK;
  if (M >= kMaxExtent || N >= (int64_t)1 << 30) return YAMOE_ERR_UNSUPPORTED;
  const size_t size = size_of(dtype);
  if (pre == nullptr || out == nullptr || !at_boundary(pre, size) || !at_boundary(out, size)) return YAMOE_ERR_BAD_ARG;
  if (codes != nullptr && (scales == nullptr || !at_boundary(codes, 16) || !at_boundary(scales, 4) || ld % 16 != 0 || ld < 2 * N || ld >= kMaxExtent))
    return YAMOE_ERR_BAD_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const GluSaved saved{reinterpret_cast<uint8_t*>(codes), scales, ld};
  using bf = __nv_bfloat16;
  return dtype == YAMOE_BF16
             ? launch_glu_forward(reinterpret_cast<const bf*>(pre), reinterpret_cast<bf*>(out), saved, M, (int)(2 * N), st)
             : launch_glu_forward(reinterpret_cast<const float*>(pre), reinterpret_cast<float*>(out), saved, M, (int)(2 * N), st);
}

int yamoe_b200_glu_backward(const void* d_out, const void* codes, const float* scales, int64_t ld, void* d_pre, int64_t M, int64_t N,
                            int dtype, void* stream) {
  if (!known_dtype(dtype)) return YAMOE_ERR_DTYPE;
  if (M < 0 || N < 0) return YAMOE_ERR_BAD_ARG;
  if (M == 0 || N == 0) return YAMOE_OK;
  if (M >= kMaxExtent || N >= (int64_t)1 << 30) return YAMOE_ERR_UNSUPPORTED;
  const size_t size = size_of(dtype);
  if (d_out == nullptr || d_pre == nullptr || !at_boundary(d_out, size) || !at_boundary(d_pre, size)) return YAMOE_ERR_BAD_ARG;
  if (codes == nullptr || scales == nullptr || !at_boundary(codes, 16) || !at_boundary(scales, 4) || ld % 16 != 0 || ld < 2 * N || ld >= kMaxExtent)
    return YAMOE_ERR_BAD_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t* q = reinterpret_cast<const uint8_t*>(codes);
  using bf = __nv_bfloat16;
  return dtype == YAMOE_BF16
             ? launch_glu_backward(reinterpret_cast<const bf*>(d_out), q, scales, ld, reinterpret_cast<bf*>(d_pre), M, (int)(2 * N), st)
             : launch_glu_backward(reinterpret_cast<const float*>(d_out), q, scales, ld, reinterpret_cast<float*>(d_pre), M, (int)(2 * N), st);
}

}  // extern "C"
