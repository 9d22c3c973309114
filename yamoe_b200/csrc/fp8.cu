// 8-bit operands: quantisation, products, and the grouped products of the expert pass; the layer for a few tokens.
// C entry points but that of the expert pass, which is put together in yamoe_b200.cu.
#include "fp8.h"

#include "fp8_gemm.cuh"
#include "moe_layer.cuh"

namespace yb {

bool fp8_matrix_ok(const yamoe_fp8_matrix_t* m, int64_t batch, int64_t cols) {
  if (m->q == nullptr || m->scale == nullptr) return false;
  if ((reinterpret_cast<uintptr_t>(m->q) & 15) != 0 || (reinterpret_cast<uintptr_t>(m->scale) & 3) != 0) return false;
  if (m->ld < cols || m->ld % 16 != 0 || m->ld >= (int64_t)1 << 40) return false;
  return batch <= 1 || (m->q_batch > 0 && m->q_batch % 16 == 0 && m->q_batch < (int64_t)1 << 40);
}

bool fp8_maps_ok(const yamoe_fp8_matrix_t* m, int64_t batch, int64_t rows) {
  return batch <= 1 || (m->q_batch % m->ld == 0 && m->q_batch / m->ld >= rows);
}

static QuantOut quant_out(const yamoe_fp8_matrix_t* m) {
  if (m == nullptr) return QuantOut{};
  return QuantOut{reinterpret_cast<uint8_t*>(m->q), m->scale, m->ld, m->q_batch, m->scale_row, m->scale_group, m->scale_batch};
}

template <typename T>
static int quantize_impl(const T* x, const yamoe_fp8_matrix_t* out, const yamoe_fp8_matrix_t* turned, int64_t B, int64_t M,
                         int64_t K, int block_rows, cudaStream_t st) {
  if (block_rows == 1 && turned == nullptr) {
    const QuantRows d{reinterpret_cast<uint8_t*>(out->q), out->scale, out->ld, out->q_batch, out->scale_row, out->scale_group,
                      out->scale_batch, nullptr, 0};
    return launch_quantize_rows<T>(x, d, B, M, (int)K, st);
  }
  return launch_quantize_tiles<T>(x, B, M, K, block_rows == 128, quant_out(out), quant_out(turned), st);
}

template <typename T>
int fp8_gather(const T* hidden, uint8_t* q, float* scale, int64_t ld, int64_t scale_group, const int32_t* flat_row, int64_t tokens,
               int H, int K, cudaStream_t st) {
  const QuantRows d{q, scale, ld, 0, 1, scale_group, 0, flat_row, K};
  return launch_quantize_rows<T>(hidden, d, 1, tokens, H, st);
}
template int fp8_gather<float>(const float*, uint8_t*, float*, int64_t, int64_t, const int32_t*, int64_t, int, int, cudaStream_t);
template int fp8_gather<__nv_bfloat16>(const __nv_bfloat16*, uint8_t*, float*, int64_t, int64_t, const int32_t*, int64_t, int, int,
                                       cudaStream_t);

template <class Epi>
static int grouped(const Fp8Rows& r, const uint8_t* a, const float* a_scale, int64_t ld, const yamoe_fp8_matrix_t& w, int N, int K,
                   int E, const Fp8Out& o, const Epi& epi, cudaStream_t st) {
  Fp8Params p{};
  p.M = r.max_rows; p.N = N; p.K = K; p.B = E;
  p.sa = a_scale; p.sa_m = 1; p.sa_k = r.max_rows;
  p.sb = w.scale; p.sb_b = w.scale_batch; p.sb_n = w.scale_row; p.sb_k = w.scale_group;
  p.pad_off = r.pad_off;
  p.n_tiles = r.header + kHdrRowTiles;
  p.status = const_cast<int32_t*>(r.header) + kHdrStatus;
  const Fp8Operand A{a, r.max_rows, ld, 0}, B{w.q, N, w.ld, w.q_batch};
  return launch_fp8_gemm<256, false, true>(A, B, o, p, epi, r.max_tiles, st);
}

template <typename T>
int fp8_gate_up(const Fp8Rows& r, const uint8_t* x, const float* x_scale, int64_t ld, const yamoe_fp8_matrix_t& w, const T* bias,
                uint8_t* act, float* act_scale, int H, int E, cudaStream_t st) {
  return grouped(r, x, x_scale, ld, w, 2 * H, H, E, Fp8Out{}, Fp8GluQuant<T>{bias, act, act_scale, ld, r.max_rows}, st);
}
template <typename T>
int fp8_down(const Fp8Rows& r, const uint8_t* act, const float* act_scale, int64_t ld, const yamoe_fp8_matrix_t& w, const T* bias,
             float* y, int H, int E, cudaStream_t st) {
  return grouped(r, act, act_scale, ld, w, H, H, E, Fp8Out{y, r.max_rows, H, 1, 4}, Fp8WeightedRows<T>{bias, r.row_token, r.row_weight, H}, st);
}
#define YB_INSTANTIATE(T)                                                                                                  \
  template int fp8_gate_up<T>(const Fp8Rows&, const uint8_t*, const float*, int64_t, const yamoe_fp8_matrix_t&, const T*,   \
                              uint8_t*, float*, int, int, cudaStream_t);                                                    \
  template int fp8_down<T>(const Fp8Rows&, const uint8_t*, const float*, int64_t, const yamoe_fp8_matrix_t&, const T*,      \
                           float*, int, int, cudaStream_t);
YB_INSTANTIATE(float)
YB_INSTANTIATE(__nv_bfloat16)
#undef YB_INSTANTIATE

// Tiles of a product: estimated clocks of each kind, the least of them.  A block takes a 128 x 256 tile some 1020 clocks, a
// 128 x 128 one 640; a tile's beginning and end 2300; meeting in shared memory 1500 more.  Clusters come in as many waves as
// the GPU's groups of SMs hold of them at a time: 48 clusters of three took 26.2 us in two waves, 48 of two 18.8 in one.
struct Fp8Choice { int bn, splits; };
template <bool BROWS, class Epi>
static Fp8Choice choose_tiles(int64_t B, int64_t M, int64_t N, int64_t K) {
  const int64_t kb = ceil_div(K, kFp8Group), rows = B * ceil_div(M, 128);
  Fp8Choice best{256, 1};
  double least = (double)ceil_div(rows * ceil_div(N, 256), kSMs) * (double)(kb * 1020 + 2300);
  for (int s = 1; s <= kFp8MaxSplits && s <= kb; ++s) {
    const double t =
        (double)ceil_div(rows * ceil_div(N, 128), s > 1 ? fp8_clusters<BROWS, Epi>(s) : kSMs) * (double)(ceil_div(kb, s) * 640 + 2300 + (s > 1 ? 1500 : 0));
    if (t < least) { least = t; best = Fp8Choice{128, s}; }
  }
  return best;
}

template <typename T, bool BROWS>
static int mm_impl(const Fp8Operand& A, const Fp8Operand& B, Fp8Params p, T* out, cudaStream_t st) {
  const int vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && p.N * (int64_t)sizeof(T) % 16 == 0;
  const Fp8Store<T> epi{out, p.N, p.M * p.N, vec};
  const Fp8Choice c = choose_tiles<BROWS, Fp8Store<T>>(p.B, p.M, p.N, p.K);
  p.MT = (int)ceil_div(p.M, 128);
  p.splits = c.splits;
  const int64_t tiles = (int64_t)p.B * p.MT;
  const Fp8Out o{vec ? out : nullptr, p.M, p.N, p.B, (int)sizeof(T)};
  return c.bn == 256 ? launch_fp8_gemm<256, BROWS, false>(A, B, o, p, epi, tiles, st)
                     : launch_fp8_gemm<128, BROWS, false>(A, B, o, p, epi, tiles, st);
}

}  // namespace yb

using namespace yb;

extern "C" {

int yamoe_b200_fp8_quantize(const void* x, const yamoe_fp8_matrix_t* out, const yamoe_fp8_matrix_t* transposed, int64_t batch,
                            int64_t M, int64_t K, int block_rows, int dtype, void* stream) {
  if (dtype != YAMOE_F32 && dtype != YAMOE_BF16) return YAMOE_ERR_DTYPE;
  if (batch < 0 || M < 0 || K < 0 || (block_rows != 1 && block_rows != 128)) return YAMOE_ERR_BAD_ARG;
  if (out == nullptr && transposed == nullptr) return YAMOE_ERR_BAD_ARG;
  if (batch == 0 || M == 0 || K == 0) return YAMOE_OK;
  if (x == nullptr || (reinterpret_cast<uintptr_t>(x) & (dtype == YAMOE_F32 ? 3 : 1)) != 0) return YAMOE_ERR_BAD_ARG;
  if ((out != nullptr && !fp8_matrix_ok(out, batch, K)) || (transposed != nullptr && !fp8_matrix_ok(transposed, batch, M)))
    return YAMOE_ERR_BAD_ARG;
  if (M >= (int64_t)1 << 31 || K >= (int64_t)1 << 31) return YAMOE_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == YAMOE_BF16
             ? quantize_impl(reinterpret_cast<const __nv_bfloat16*>(x), out, transposed, batch, M, K, block_rows, st)
             : quantize_impl(reinterpret_cast<const float*>(x), out, transposed, batch, M, K, block_rows, st);
}

size_t yamoe_b200_fp8_mm_workspace_bytes(int64_t batch, int64_t M, int64_t N, int64_t K) {
  if (batch < 0 || M < 0 || N < 0 || K < 0) return 0;
  return 256;
}

int yamoe_b200_fp8_mm(const yamoe_fp8_matrix_t* a, const yamoe_fp8_matrix_t* b, int b_block_rows, void* out, int64_t batch,
                      int64_t M, int64_t N, int64_t K, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (out_dtype != YAMOE_F32 && out_dtype != YAMOE_BF16) return YAMOE_ERR_DTYPE;
  if (batch < 0 || M < 0 || N < 0 || K < 0 || (b_block_rows != 1 && b_block_rows != 128)) return YAMOE_ERR_BAD_ARG;
  if (batch == 0 || M == 0 || N == 0) return YAMOE_OK;
  const size_t size = out_dtype == YAMOE_F32 ? 4 : 2;
  if (out == nullptr || (reinterpret_cast<uintptr_t>(out) & (size - 1)) != 0) return YAMOE_ERR_BAD_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (K == 0) {
    YB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)batch * M * N * size, st));
    return YAMOE_OK;
  }
  if (a == nullptr || b == nullptr || !fp8_matrix_ok(a, batch, K) || !fp8_matrix_ok(b, batch, K)) return YAMOE_ERR_BAD_ARG;
  // coordinates and tile counts are 32-bit numbers
  if (M >= (int64_t)1 << 30 || N >= (int64_t)1 << 30 || K >= (int64_t)1 << 30 || batch >= (int64_t)1 << 30)
    return YAMOE_ERR_UNSUPPORTED;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < yamoe_b200_fp8_mm_workspace_bytes(batch, M, N, K))
    return YAMOE_ERR_WORKSPACE;
  if (!fp8_maps_ok(a, batch, M) || !fp8_maps_ok(b, batch, N)) return YAMOE_ERR_BAD_ARG;
  Fp8Params p{};
  p.M = M; p.N = N; p.K = (int)K; p.B = (int)batch;
  p.sa = a->scale; p.sa_b = a->scale_batch; p.sa_m = a->scale_row; p.sa_k = a->scale_group;
  p.sb = b->scale; p.sb_b = b->scale_batch; p.sb_n = b->scale_row; p.sb_k = b->scale_group;
  p.status = reinterpret_cast<int32_t*>(workspace) + kHdrStatus;
  p.clear_status = 1;
  const Fp8Operand A{a->q, M, a->ld, a->q_batch}, B{b->q, N, b->ld, b->q_batch};
  const bool rows = b_block_rows == 1;
  if (out_dtype == YAMOE_BF16) {
    auto o = reinterpret_cast<__nv_bfloat16*>(out);
    return rows ? mm_impl<__nv_bfloat16, true>(A, B, p, o, st) : mm_impl<__nv_bfloat16, false>(A, B, p, o, st);
  }
  auto o = reinterpret_cast<float*>(out);
  return rows ? mm_impl<float, true>(A, B, p, o, st) : mm_impl<float, false>(A, B, p, o, st);
}

size_t yamoe_b200_moe_layer_workspace_bytes(int64_t T, int H, int E, int K) {
  if (!layer_shape_ok(T, H, E, K)) return 0;
  LayerArgs a{};
  a.T = (int)T; a.H = H; a.E = E; a.K = K;
  return layer_workspace(a, nullptr);
}

int yamoe_b200_moe_layer(const void* hidden_states, const void* router_weight, const void* router_bias, const void* gate_up,
                         const yamoe_fp8_matrix_t* gate_up_fp8, const void* gate_up_bias, const void* down,
                         const yamoe_fp8_matrix_t* down_fp8, const void* down_bias, void* out, void* router_scores, int64_t T, int H,
                         int E, int K, int64_t expert_capacity, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != YAMOE_BF16) return YAMOE_ERR_DTYPE;
  if (T < 0 || H <= 0 || E <= 0 || K <= 0 || H % 8 != 0 || K > E || expert_capacity < 0) return YAMOE_ERR_BAD_ARG;
  if (!layer_shape_ok(T, H, E, K)) return YAMOE_ERR_UNSUPPORTED;
  const bool fp8 = gate_up_fp8 != nullptr;
  if (fp8 ? down_fp8 == nullptr : (gate_up == nullptr || down == nullptr || down_fp8 != nullptr)) return YAMOE_ERR_BAD_ARG;
  if (T > 0 && (!hidden_states || !out || !router_scores)) return YAMOE_ERR_BAD_ARG;
  if (!router_weight || !gate_up_bias || !down_bias) return YAMOE_ERR_BAD_ARG;
  const void* wide[] = {hidden_states, router_weight, gate_up, down, out};
  for (const void* q : wide)
    if (reinterpret_cast<uintptr_t>(q) & 15) return YAMOE_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(gate_up_bias) | reinterpret_cast<uintptr_t>(down_bias)) & 3) return YAMOE_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(router_bias) | reinterpret_cast<uintptr_t>(router_scores)) & 1) return YAMOE_ERR_BAD_ARG;
  if (fp8 && (!fp8_matrix_ok(gate_up_fp8, E, H) || !fp8_matrix_ok(down_fp8, E, H))) return YAMOE_ERR_BAD_ARG;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < yamoe_b200_moe_layer_workspace_bytes(T, H, E, K))
    return YAMOE_ERR_WORKSPACE;
  if (T == 0) return YAMOE_OK;
  if (fp8 && (!fp8_maps_ok(gate_up_fp8, E, 2 * (int64_t)H) || !fp8_maps_ok(down_fp8, E, H))) return YAMOE_ERR_BAD_ARG;
  if (!umma_available()) return YAMOE_ERR_UNSUPPORTED;
  using bf = __nv_bfloat16;
  LayerArgs a{};
  a.T = (int)T; a.H = H; a.E = E; a.K = K; a.capacity = expert_capacity;
  layer_workspace(a, reinterpret_cast<char*>(workspace));
  a.x = reinterpret_cast<const bf*>(hidden_states);
  a.router = reinterpret_cast<const bf*>(router_weight);
  a.router_bias = reinterpret_cast<const bf*>(router_bias);
  a.bias_gu = reinterpret_cast<const bf*>(gate_up_bias);
  a.bias_dn = reinterpret_cast<const bf*>(down_bias);
  a.out = reinterpret_cast<bf*>(out);
  a.scores = reinterpret_cast<bf*>(router_scores);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  CUtensorMap gu, dn;
  const uint64_t h = (uint64_t)H, n = (uint64_t)E;
  if (fp8) {
    const yamoe_fp8_matrix_t &g = *gate_up_fp8, &d = *down_fp8;
    a.scale_gu = g.scale; a.gu_b = g.scale_batch; a.gu_r = g.scale_row; a.gu_g = g.scale_group;
    a.scale_dn = d.scale; a.dn_b = d.scale_batch; a.dn_r = d.scale_row; a.dn_g = d.scale_group;
    const uint64_t dg[3] = {h, 2 * h, n}, dd[3] = {h, h, n};
    const uint64_t sg[2] = {(uint64_t)g.ld, E > 1 ? (uint64_t)g.q_batch : 2 * h * g.ld}, sd[2] = {(uint64_t)d.ld, E > 1 ? (uint64_t)d.q_batch : h * d.ld};
    const uint32_t box[3] = {128, kLayerUnit, 1};
    if (!encode_map(&gu, g.q, 3, dg, sg, box, kMapU8) || !encode_map(&dn, d.q, 3, dd, sd, box, kMapU8)) return YAMOE_ERR_CUDA;
    return launch_moe_layer<true>(a, gu, dn, st);
  }
  const uint64_t dg[3] = {2 * h, h, n}, dd[3] = {h, h, n};
  const uint64_t sg[2] = {4 * h, 4 * h * h}, sd[2] = {2 * h, 2 * h * h};
  const uint32_t box[3] = {64, 64, 1};
  if (!encode_map(&gu, gate_up, 3, dg, sg, box, kMapBf16) || !encode_map(&dn, down, 3, dd, sd, box, kMapBf16)) return YAMOE_ERR_CUDA;
  return launch_moe_layer<false>(a, gu, dn, st);
}

}  // extern "C"
