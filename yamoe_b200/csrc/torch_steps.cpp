// Torch binding of the expert layer's steps: `sort_tokens`, `combine_tokens`, `quantize_int8`, `int8_mm` and `glu_fp8` over the C ABI, with
// the gradients of the three that have one and a refusal of those of the integers.
#include <ATen/cuda/EmptyTensor.h>

#include <optional>
#include <tuple>
#include <vector>

#include "torch_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(std::initializer_list<at::Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// A new tensor on the device of `like`, without the dispatcher (which takes as long as the smallest kernels do)
at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}
at::Tensor scratch(size_t bytes, const at::Tensor& like) { return empty_on(like, {(int64_t)bytes}, at::kByte); }

at::Tensor as_int64(const at::Tensor& t) { return !t.defined() || t.scalar_type() == at::kLong ? t : t.to(at::kLong); }

void check_float(const char* op, const char* name, const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be on CUDA");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, op, ": ", name, " must be float32 or bfloat16, got ",
              t.scalar_type());
}

// ---- tokens sorted by expert and back ------------------------------------------------------------------------------------------

at::Tensor combine(const at::Tensor& rows, const at::Tensor& row_of, const at::Tensor& weights, const at::Tensor& indices) {
  const at::Tensor r = rows.contiguous(), of = row_of.contiguous(), w = weights.defined() ? weights.contiguous() : weights,
                   idx = indices.defined() ? indices.contiguous() : indices;
  const int64_t T = of.size(0), K = of.size(1), H = r.size(-1);
  at::Tensor out = empty_on(r, {T, H}, r.scalar_type());
  int64_t n_rows = 1;                                  // (H may be 0)
  for (int64_t i = 0; i + 1 < r.dim(); ++i) n_rows *= r.size(i);
  check(yamoe_b200_combine_tokens(r.data_ptr(), n_rows, of.data_ptr<int32_t>(), w.defined() ? w.data_ptr() : nullptr,
                                  w.defined() ? dtype_of(w) : YAMOE_F32, idx.defined() ? idx.data_ptr<int64_t>() : nullptr, out.data_ptr(), T,
                                  H, idx.defined() ? (int)w.size(1) : 0, (int)K, dtype_of(r), current_stream()),
        "combine_tokens");
  return out;
}

struct Sorted {
  at::Tensor rows, row_of, offsets;
};

Sorted sort_tokens(const at::Tensor& hidden_states, const at::Tensor& router_indices, int64_t num_experts,
                   std::optional<int64_t> expert_capacity) {
  check_float("sort_tokens", "hidden_states", hidden_states);
  TORCH_CHECK(hidden_states.dim() == 2, "sort_tokens: hidden_states must be 2D [T, H]");
  TORCH_CHECK(router_indices.device() == hidden_states.device(), "sort_tokens: router_indices must be on the device of hidden_states");
  TORCH_CHECK(router_indices.scalar_type() == at::kLong || router_indices.scalar_type() == at::kInt, "sort_tokens: router_indices must be int64");
  const int64_t T = hidden_states.size(0), H = hidden_states.size(1), E = num_experts;
  TORCH_CHECK(router_indices.dim() == 2 && router_indices.size(0) == T, "sort_tokens: router_indices must be [T, K]");
  TORCH_CHECK(E >= 1 && E <= 1024, "sort_tokens: num_experts must be between 1 and 1024, got ", E);
  TORCH_CHECK(!expert_capacity.has_value() || *expert_capacity >= 0, "sort_tokens: expert_capacity must not be negative");
  const int64_t K = router_indices.size(1), C = expert_capacity.value_or(-1);
  TORCH_CHECK(C < (int64_t)1 << 31 && E * std::max<int64_t>(C, 0) < (int64_t)1 << 31, "sort_tokens: too many rows");
  TORCH_CHECK(T * K < (int64_t)1 << 30, "sort_tokens: fewer than 2^30 assignments expected, got ", T * K);
  const c10::cuda::CUDAGuard guard(hidden_states.device());
  const at::Tensor hs = hidden_states.contiguous(), ri = as_int64(router_indices).contiguous();
  Sorted s;
  s.rows = C < 0 ? empty_on(hs, {T * K, H}, hs.scalar_type()) : empty_on(hs, {E, C, H}, hs.scalar_type());
  s.row_of = empty_on(hs, {T, K}, at::kInt);
  s.offsets = empty_on(hs, {E + 1}, at::kInt);
  const at::Tensor ws = scratch(yamoe_b200_sort_tokens_workspace_bytes(T, (int)E, (int)K), hs);
  check(yamoe_b200_sort_tokens(hs.data_ptr(), ri.data_ptr<int64_t>(), s.rows.data_ptr(), s.row_of.data_ptr<int32_t>(),
                               s.offsets.data_ptr<int32_t>(), T, H, (int)E, (int)K, C, dtype_of(hs), ws.data_ptr(), (size_t)ws.numel(),
                               current_stream()),
        "sort_tokens");
  return s;
}

struct SortTokens : torch::autograd::Function<SortTokens> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& hidden_states, const at::Tensor& router_indices, int64_t num_experts,
                               std::optional<int64_t> expert_capacity) {
    const at::AutoDispatchBelowADInplaceOrView below;
    const Sorted s = sort_tokens(hidden_states, router_indices, num_experts, expert_capacity);
    ctx->mark_non_differentiable({s.row_of, s.offsets});
    ctx->set_materialize_grads(false);                 // (zeros for the integers would be two launches)
    ctx->save_for_backward({s.row_of});
    return {s.rows, s.row_of, s.offsets};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor d_rows = grads[0], row_of = ctx->get_saved_variables()[0];
    variable_list out(4);
    if (!d_rows.defined()) return out;
    const c10::cuda::CUDAGuard guard(d_rows.device());
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      out[0] = combine(d_rows, row_of, at::Tensor(), at::Tensor());
    }
    if (at::GradMode::is_enabled()) differentiate_no_further("sort_tokens", {d_rows}, {&out[0]});
    return out;
  }
};

using ThreeTensors = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
ThreeTensors sort_tokens_cuda(const at::Tensor& hidden_states, const at::Tensor& router_indices, int64_t num_experts,
                              std::optional<int64_t> expert_capacity) {
  const Sorted s = sort_tokens(hidden_states, router_indices, num_experts, expert_capacity);
  return {s.rows, s.row_of, s.offsets};
}
ThreeTensors sort_tokens_autograd(const at::Tensor& hidden_states, const at::Tensor& router_indices, int64_t num_experts,
                                  std::optional<int64_t> expert_capacity) {
  check_no_tangent("sort_tokens", hidden_states);
  if (wants_grad({hidden_states})) {
    const variable_list s = SortTokens::apply(hidden_states, router_indices, num_experts, expert_capacity);
    return {s[0], s[1], s[2]};
  }
  const at::AutoDispatchBelowAutograd below;
  return sort_tokens_cuda(hidden_states, router_indices, num_experts, expert_capacity);
}

void check_combine(const at::Tensor& rows, const at::Tensor& row_of, const at::Tensor& weights, const at::Tensor& indices) {
  check_float("combine_tokens", "rows", rows);
  TORCH_CHECK(rows.dim() >= 2, "combine_tokens: rows must be [R, H] or [E, C, H]");
  TORCH_CHECK(row_of.device() == rows.device(), "combine_tokens: row_of must be on the device of rows");
  TORCH_CHECK(row_of.dim() == 2 && row_of.scalar_type() == at::kInt, "combine_tokens: row_of must be int32 [T, K]");
  const int64_t T = row_of.size(0), K = row_of.size(1);
  TORCH_CHECK(K <= 1024, "combine_tokens: at most 1024 rows per token, got ", K);
  TORCH_CHECK(weights.defined() || !indices.defined(), "combine_tokens: router_indices belong to routing_weights");
  if (!weights.defined()) return;
  TORCH_CHECK(weights.device() == rows.device(), "combine_tokens: routing_weights must be on the device of rows");
  TORCH_CHECK(weights.scalar_type() == rows.scalar_type() || weights.scalar_type() == at::kFloat,
              "combine_tokens: routing_weights must have the dtype of rows (", rows.scalar_type(), ") or float32, got ", weights.scalar_type());
  TORCH_CHECK(weights.dim() == 2 && weights.size(0) == T, "combine_tokens: routing_weights must be [T, K], or [T, E] with router_indices");
  if (indices.defined()) {
    TORCH_CHECK(indices.device() == rows.device(), "combine_tokens: router_indices must be on the device of rows");
    TORCH_CHECK(indices.scalar_type() == at::kLong || indices.scalar_type() == at::kInt, "combine_tokens: router_indices must be int64");
    TORCH_CHECK(indices.sizes() == row_of.sizes(), "combine_tokens: router_indices must be [T, K]");
  } else {
    TORCH_CHECK(weights.size(1) == K, "combine_tokens: routing_weights must be [T, K], or [T, E] with router_indices");
  }
}

// arguments as the kernels take them
at::Tensor or_none(const std::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }

struct CombineTokens : torch::autograd::Function<CombineTokens> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows, const at::Tensor& row_of,
                            const std::optional<at::Tensor>& routing_weights, const std::optional<at::Tensor>& router_indices) {
    const at::Tensor weights = or_none(routing_weights), indices = as_int64(or_none(router_indices));
    const c10::cuda::CUDAGuard guard(rows.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    // the rows themselves are needed for the gradient of the weights only
    ctx->save_for_backward({weights.defined() && weights.requires_grad() ? rows : at::Tensor(), row_of, weights, indices});
    ctx->saved_data["shape"] = rows.sizes().vec();
    return combine(rows, row_of, weights, indices);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    const at::Tensor d = grads[0];
    if (!d.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &rows = saved[0], &row_of = saved[1], &weights = saved[2], &indices = saved[3];
    const bool want_rows = ctx->needs_input_grad(0), want_weights = rows.defined() && ctx->needs_input_grad(2);
    if (!want_rows && !want_weights) return out;
    const c10::cuda::CUDAGuard guard(d.device());
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor g = d.contiguous(), of = row_of.contiguous(), r = rows.defined() ? rows.contiguous() : rows,
                       w = weights.defined() ? weights.contiguous() : weights, idx = indices.defined() ? indices.contiguous() : indices;
      const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
      int64_t n_rows = 1;
      for (size_t i = 0; i + 1 < shape.size(); ++i) n_rows *= shape[i];
      const int64_t T = of.size(0), K = of.size(1), H = shape.back();
      if (want_rows) out[0] = empty_on(g, shape, g.scalar_type());
      // (indices without elements have no address: dense weights of tokens without slots)
      if (want_weights) out[2] = K > 0 ? at::empty_like(w) : at::zeros_like(w);
      const at::Tensor ws = scratch(yamoe_b200_combine_tokens_backward_workspace_bytes(n_rows, T, (int)K), g);
      check(yamoe_b200_combine_tokens_backward(g.data_ptr(), r.defined() ? r.data_ptr() : nullptr, n_rows, of.data_ptr<int32_t>(),
                                               w.defined() ? w.data_ptr() : nullptr, w.defined() ? dtype_of(w) : YAMOE_F32,
                                               idx.defined() ? idx.data_ptr<int64_t>() : nullptr, want_rows ? out[0].data_ptr() : nullptr,
                                               want_weights ? out[2].data_ptr() : nullptr, T, H, idx.defined() ? (int)w.size(1) : 0, (int)K,
                                               dtype_of(g), ws.data_ptr(), (size_t)ws.numel(), current_stream()),
            "combine_tokens (backward)");
    }
    if (at::GradMode::is_enabled()) differentiate_no_further("combine_tokens", {d}, {&out[0], &out[2]});
    return out;
  }
};

at::Tensor combine_tokens_cuda(const at::Tensor& rows, const at::Tensor& row_of, const std::optional<at::Tensor>& routing_weights,
                               const std::optional<at::Tensor>& router_indices) {
  const at::Tensor w = or_none(routing_weights), idx = or_none(router_indices);
  check_combine(rows, row_of, w, idx);
  const c10::cuda::CUDAGuard guard(rows.device());
  return combine(rows, row_of, w, as_int64(idx));
}
at::Tensor combine_tokens_autograd(const at::Tensor& rows, const at::Tensor& row_of, const std::optional<at::Tensor>& routing_weights,
                                   const std::optional<at::Tensor>& router_indices) {
  const at::Tensor w = or_none(routing_weights), idx = or_none(router_indices);
  check_no_tangent("combine_tokens", rows);
  if (w.defined()) check_no_tangent("combine_tokens", w);
  if (wants_grad({rows, w})) {
    check_combine(rows, row_of, w, idx);
    const c10::cuda::CUDAGuard guard(rows.device());
    return CombineTokens::apply(rows, row_of, routing_weights, router_indices);
  }
  const at::AutoDispatchBelowAutograd below;
  return combine_tokens_cuda(rows, row_of, routing_weights, router_indices);
}

// ---- 8-bit integers --------------------------------------------------------------------------------------------------------------

struct Integers {
  at::Tensor q, scale;          // [.., rows, cols] and [.., rows]
};

yamoe_int8_matrix_t matrix_of(const Integers& m) {
  const bool batched = m.q.dim() == 3, several = batched && m.q.size(0) > 1;
  yamoe_int8_matrix_t r{};
  r.q = m.q.data_ptr();
  r.scale = m.scale.data_ptr<float>();
  // (one row: its pitch is that of the matrices)
  r.ld = m.q.size(-2) > 1 ? m.q.stride(-2) : several ? m.q.stride(0) : ceil_div(m.q.size(-1), 16) * 16;
  r.q_batch = several ? m.q.stride(0) : m.q.size(-2) * r.ld;
  r.scale_row = m.scale.stride(-1);
  r.scale_batch = batched ? m.scale.stride(0) : 0;
  return r;
}

// Codes with rows of 16-byte multiples, the bytes behind them included that the kernels may write.
at::Tensor empty_codes(at::IntArrayRef shape, const at::Tensor& like) {
  std::vector<int64_t> held = shape.vec();
  held.back() = ceil_div(held.back(), 16) * 16;
  const at::Tensor q = empty_on(like, held, at::kChar);
  return held.back() == shape.back() ? q : q.narrow(-1, 0, shape.back());
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_cuda(const at::Tensor& x, bool transpose) {
  check_float("quantize_int8", "x", x);
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "quantize_int8: x must be 2D [M, K] or 3D [B, M, K]");
  const c10::cuda::CUDAGuard guard(x.device());
  // a transposed view is quantised from what it is a view of
  const bool turned = x.size(-2) > 1 && x.size(-1) > 1 && !x.is_contiguous() && x.transpose(-1, -2).is_contiguous();
  const at::Tensor held = turned ? x.transpose(-1, -2) : x.contiguous();
  std::vector<int64_t> shape = x.sizes().vec();
  if (transpose) std::swap(shape[shape.size() - 1], shape[shape.size() - 2]);
  Integers m{empty_codes(shape, x), at::Tensor()};
  shape.pop_back();
  m.scale = empty_on(x, shape, at::kFloat);
  if (x.numel() == 0) {                                 // rows without values
    m.scale.fill_(0x1p-100f / 127.f);
    return {m.q, m.scale};
  }
  const yamoe_int8_matrix_t out = matrix_of(m);
  check(yamoe_b200_int8_quantize(held.data_ptr(), &out, x.dim() == 3 ? x.size(0) : 1, held.size(-2), held.size(-1), turned != transpose,
                                 dtype_of(x), current_stream()),
        "quantize_int8");
  return {m.q, m.scale};
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_autograd(const at::Tensor& x, bool transpose) {
  check_no_tangent("quantize_int8", x);
  std::tuple<at::Tensor, at::Tensor> codes;
  {
    const at::AutoDispatchBelowAutograd below;
    codes = quantize_int8_cuda(x, transpose);
  }
  if (wants_grad({x})) no_gradient("quantize_int8", {x}, std::get<1>(codes));
  return codes;
}

// Checks a pair of codes and scales and brings codes whose rows the kernels cannot address into a layout of their own.
Integers operand(const char* name, const at::Tensor& q, const at::Tensor& scale, int64_t dim) {
  TORCH_CHECK(q.scalar_type() == at::kChar, "int8_mm: ", name, " must be int8, got ", q.scalar_type());
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "int8_mm: the scale of ", name, " must be float32, got ", scale.scalar_type());
  TORCH_CHECK(q.dim() == dim && scale.dim() == dim - 1, "int8_mm: ", name, " must be ", dim, "D and its scale ", dim - 1, "D");
  TORCH_CHECK(scale.sizes() == q.sizes().slice(0, dim - 1), "int8_mm: the scale of ", name, " must hold one value per row");
  const int64_t rows = q.size(-2);
  const bool ok = q.stride(-1) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 &&
                  (rows <= 1 || (q.stride(-2) % 16 == 0 && q.stride(-2) >= q.size(-1))) &&
                  (dim == 2 || q.size(0) <= 1 ||
                   (rows <= 1 ? q.stride(0) % 16 == 0 && q.stride(0) >= q.size(-1)
                              : q.stride(-2) > 0 && q.stride(0) % q.stride(-2) == 0 && q.stride(0) / q.stride(-2) >= rows));
  if (ok || q.numel() == 0) return {q, scale};
  const Integers m{empty_codes(q.sizes(), q), scale};
  m.q.copy_(q);
  return m;
}

at::Tensor int8_mm_cuda(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                        at::ScalarType out_dtype, const std::optional<at::Tensor>& offsets) {
  const bool grouped = offsets.has_value();
  TORCH_CHECK(out_dtype == at::kFloat || out_dtype == at::kBFloat16, "int8_mm: out_dtype must be float32 or bfloat16");
  TORCH_CHECK(a.is_cuda() && b.device() == a.device() && a_scale.device() == a.device() && b_scale.device() == a.device() &&
                  (!grouped || offsets->device() == a.device()),
              "int8_mm: tensors must be on one CUDA device");
  TORCH_CHECK(grouped ? a.dim() == 2 : a.dim() == 2 || a.dim() == 3, "int8_mm: a must be 2D [M, K]", grouped ? "" : " or 3D [B, M, K]");
  const c10::cuda::CUDAGuard guard(a.device());
  const Integers ma = operand("a", a, a_scale, a.dim()), mb = operand("b", b, b_scale, grouped ? 3 : a.dim());
  const int64_t M = a.size(-2), N = b.size(-2), K = a.size(-1), B = b.dim() == 3 ? b.size(0) : 1;
  TORCH_CHECK(b.size(-1) == K, "int8_mm: a is [.., M, K] and b [.., N, K]: K is ", K, " and ", b.size(-1));
  TORCH_CHECK(K < (int64_t)1 << 17, "int8_mm: sums of fewer than 2^17 products expected, got ", K);
  at::Tensor first;
  if (grouped) {
    TORCH_CHECK(B <= 1024, "int8_mm: at most 1024 experts, got ", B);
    TORCH_CHECK(offsets->dim() == 1 && offsets->size(0) == B + 1 && (offsets->scalar_type() == at::kInt || offsets->scalar_type() == at::kLong),
                "int8_mm: offsets must be int32 [E + 1]");
    // 64 bits are kept within the rows before they become 32, as the kernels keep 32
    first = (offsets->scalar_type() == at::kInt ? *offsets : offsets->clamp(0, M).to(at::kInt)).contiguous();
  } else {
    TORCH_CHECK(a.dim() == 2 || a.size(0) == B, "int8_mm: a and b must hold the same number of matrices");
  }
  const at::Tensor out = a.dim() == 3 ? empty_on(a, {B, M, N}, out_dtype) : empty_on(a, {M, N}, out_dtype);
  if (out.numel() == 0) return out;
  if (K == 0 || B == 0) return out.zero_();
  const yamoe_int8_matrix_t x = matrix_of(ma), w = matrix_of(mb);
  const at::Tensor ws = scratch(yamoe_b200_int8_mm_workspace_bytes(B, M, N, K), a);
  check(yamoe_b200_int8_mm(&x, &w, grouped ? first.data_ptr<int32_t>() : nullptr, out.data_ptr(), B, M, N, K,
                           out_dtype == at::kFloat ? YAMOE_F32 : YAMOE_BF16, ws.data_ptr(), (size_t)ws.numel(), current_stream()),
        "int8_mm");
  check_device_status(ws, current_stream(), "int8_mm");
  return out;
}

at::Tensor int8_mm_autograd(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                            at::ScalarType out_dtype, const std::optional<at::Tensor>& offsets) {
  check_no_tangent("int8_mm", a_scale);
  check_no_tangent("int8_mm", b_scale);
  at::Tensor out;
  {
    const at::AutoDispatchBelowAutograd below;
    out = int8_mm_cuda(a, a_scale, b, b_scale, out_dtype, offsets);
  }
  if (wants_grad({a_scale, b_scale})) no_gradient("int8_mm", {a_scale, b_scale}, out);
  return out;
}

// ---- GLU -------------------------------------------------------------------------------------------------------------------------

struct Checkpoint {
  at::Tensor q, scale;          // codes [M, ld], scales [M, groups]
};

at::Tensor glu(const at::Tensor& pre, Checkpoint* keep) {
  const at::Tensor x = pre.contiguous();
  std::vector<int64_t> shape = x.sizes().vec();
  const int64_t W = shape.back();
  int64_t M = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) M *= shape[i];
  shape.back() = W / 2;
  const at::Tensor out = empty_on(x, shape, x.scalar_type());
  const int64_t ld = ceil_div(W, 16) * 16;
  if (keep) {
    keep->q = empty_on(x, {M, ld}, at::kFloat8_e4m3fn);
    keep->scale = empty_on(x, {M, ceil_div(W, 128)}, at::kFloat);
  }
  check(yamoe_b200_glu_forward(x.data_ptr(), out.data_ptr(), keep ? keep->q.data_ptr() : nullptr,
                               keep ? keep->scale.data_ptr<float>() : nullptr, ld, M, W / 2, dtype_of(x), current_stream()),
        "glu_fp8");
  return out;
}

void check_glu(const at::Tensor& pre) {
  check_float("glu_fp8", "pre", pre);
  TORCH_CHECK(pre.dim() >= 1 && pre.size(-1) % 2 == 0, "glu_fp8: pre must be [.., 2 * N], gate and up in turn");
  TORCH_CHECK(pre.size(-1) < (int64_t)1 << 31, "glu_fp8: rows of fewer than 2^31 values expected");
}

struct GluFp8 : torch::autograd::Function<GluFp8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& pre) {
    const c10::cuda::CUDAGuard guard(pre.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    Checkpoint kept;
    const at::Tensor out = glu(pre, &kept);
    ctx->save_for_backward({kept.q, kept.scale});
    ctx->saved_data["shape"] = pre.sizes().vec();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor dy = grads[0];
    at::Tensor d_pre;
    if (!dy.defined()) return {d_pre};
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(dy.device());
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      // hooks on saved tensors may give the codes back at another address
      const at::Tensor g = dy.contiguous(), q = aligned(saved[0]), scale = saved[1].contiguous();
      d_pre = empty_on(g, ctx->saved_data["shape"].toIntVector(), g.scalar_type());
      check(yamoe_b200_glu_backward(g.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), q.size(1), d_pre.data_ptr(), q.size(0),
                                    d_pre.size(-1) / 2, dtype_of(g), current_stream()),
            "glu_fp8 (backward)");
    }
    if (at::GradMode::is_enabled()) differentiate_no_further("glu_fp8", {dy}, {&d_pre});
    return {d_pre};
  }
};

at::Tensor glu_fp8_cuda(const at::Tensor& pre) {
  check_glu(pre);
  const c10::cuda::CUDAGuard guard(pre.device());
  return glu(pre, nullptr);
}
at::Tensor glu_fp8_autograd(const at::Tensor& pre) {
  check_no_tangent("glu_fp8", pre);
  if (wants_grad({pre})) {
    check_glu(pre);
    return GluFp8::apply(pre);
  }
  const at::AutoDispatchBelowAutograd below;
  return glu_fp8_cuda(pre);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(yamoe_b200, m) {
  m.def(
      "sort_tokens(Tensor hidden_states, Tensor router_indices, int num_experts, int? expert_capacity=None) -> (Tensor, Tensor, Tensor)");
  m.def("combine_tokens(Tensor rows, Tensor row_of, Tensor? routing_weights=None, Tensor? router_indices=None) -> Tensor");
  m.def("quantize_int8(Tensor x, bool transpose=False) -> (Tensor, Tensor)");
  m.def(
      "int8_mm(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType out_dtype=bfloat16, Tensor? offsets=None) -> Tensor");
  m.def("glu_fp8(Tensor pre) -> Tensor");
}

TORCH_LIBRARY_IMPL(yamoe_b200, AutogradCUDA, m) {
  m.impl("sort_tokens", &sort_tokens_autograd);
  m.impl("combine_tokens", &combine_tokens_autograd);
  m.impl("quantize_int8", &quantize_int8_autograd);
  m.impl("int8_mm", &int8_mm_autograd);
  m.impl("glu_fp8", &glu_fp8_autograd);
}

TORCH_LIBRARY_IMPL(yamoe_b200, CUDA, m) {
  m.impl("sort_tokens", &sort_tokens_cuda);
  m.impl("combine_tokens", &combine_tokens_cuda);
  m.impl("quantize_int8", &quantize_int8_cuda);
  m.impl("int8_mm", &int8_mm_cuda);
  m.impl("glu_fp8", &glu_fp8_cuda);
}
