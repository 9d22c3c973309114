// Thin torch binding over the C ABI: the operators `yamoe_b200::experts` and
// `yamoe_b200::experts_backward` with the reference's schemas
// (torch-ext/torch_binding.cpp:58-83), implemented as argument checks, output / workspace
// allocation through torch, and one call into libyamoe_b200.so with raw pointers and torch's
// current stream.  Takes the place of torch-ext/torch_binding.cpp + csrc/moe.cpp:45-136 of the
// reference; the preconditions and their messages follow csrc/moe.cpp:58-96.
//
// Built separately from the CUDA library (host compiler only) and loaded with
// torch.ops.load_library; when it is absent the same operators are registered from Python
// (yamoe_b200/ops.py), which costs some tens of microseconds more per call.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cstdlib>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/yamoe_b200.h"

namespace {

struct Shape {
  int64_t T;
  int H, E, K, dtype;
};

Shape validate(const at::Tensor& hidden_states, const at::Tensor& router_indices, const at::Tensor& routing_weights,
               const at::Tensor& gate_up_proj, const at::Tensor& gate_up_proj_bias, const at::Tensor& down_proj,
               const at::Tensor& down_proj_bias, int64_t num_experts, int64_t top_k) {
  const at::Tensor* tensors[] = {&hidden_states, &router_indices, &routing_weights, &gate_up_proj,
                                 &gate_up_proj_bias, &down_proj, &down_proj_bias};
  const char* names[] = {"hidden_states", "router_indices", "routing_weights", "gate_up_proj",
                         "gate_up_proj_bias", "down_proj", "down_proj_bias"};
  for (int i = 0; i < 7; ++i) TORCH_CHECK(tensors[i]->is_cuda(), names[i], " must be on CUDA");
  TORCH_CHECK(hidden_states.dim() == 2, "hidden_states must be 2D [T, H]");
  TORCH_CHECK(router_indices.dim() == 2, "router_indices must be 2D [T, K]");
  TORCH_CHECK(routing_weights.dim() == 2, "routing_weights must be 2D [T, K]");
  TORCH_CHECK(gate_up_proj.dim() == 3, "gate_up_proj must be 3D [E, H, 2*H]");
  TORCH_CHECK(gate_up_proj_bias.dim() == 2, "gate_up_proj_bias must be 2D [E, 2*H]");
  TORCH_CHECK(down_proj.dim() == 3, "down_proj must be 3D [E, H, H]");
  TORCH_CHECK(down_proj_bias.dim() == 2, "down_proj_bias must be 2D [E, H]");
  const int64_t T = hidden_states.size(0), H = hidden_states.size(1), E = num_experts, K = top_k;
  TORCH_CHECK(router_indices.size(0) == T && router_indices.size(1) == K, "router_indices must be [T, K]");
  TORCH_CHECK(routing_weights.size(0) == T && (routing_weights.size(1) == K || routing_weights.size(1) == E),
              "routing_weights must be [T, K] or [T, E]");
  TORCH_CHECK(gate_up_proj.size(0) == E && gate_up_proj.size(1) == H && gate_up_proj.size(2) == 2 * H,
              "gate_up_proj must be [E, H, 2*H]");
  TORCH_CHECK(gate_up_proj_bias.size(0) == E && gate_up_proj_bias.size(1) == 2 * H,
              "gate_up_proj_bias must be [E, 2*H]");
  TORCH_CHECK(down_proj.size(0) == E && down_proj.size(1) == H && down_proj.size(2) == H, "down_proj must be [E, H, H]");
  TORCH_CHECK(down_proj_bias.size(0) == E && down_proj_bias.size(1) == H, "down_proj_bias must be [E, H]");
  const auto dt = hidden_states.scalar_type();
  TORCH_CHECK(dt == at::kFloat || dt == at::kBFloat16, "yamoe_b200 supports float32 and bfloat16, got ", dt);
  for (int i = 2; i < 7; ++i)
    TORCH_CHECK(tensors[i]->scalar_type() == dt, names[i], " must have the dtype of hidden_states (", dt, "), got ",
                tensors[i]->scalar_type());
  TORCH_CHECK(router_indices.scalar_type() == at::kLong || router_indices.scalar_type() == at::kInt,
              "router_indices must be int64");
  return Shape{T, (int)H, (int)E, (int)K, dt == at::kBFloat16 ? YAMOE_BF16 : YAMOE_F32};
}

void check(int status, const char* what) {
  TORCH_CHECK(status == YAMOE_OK, "yamoe_b200: ", what, " failed: ", yamoe_b200_status_string(status), " (status ",
              status, ")");
}

// YAMOE_B200_CHECK_STATUS=1: read the device status word after the call (one stream synchronisation)
void check_device_status(const at::Tensor& ws, cudaStream_t st, const char* what) {
  static const bool on = []() {
    const char* env = std::getenv("YAMOE_B200_CHECK_STATUS");
    return env != nullptr && env[0] != '\0' && !(env[0] == '0' && env[1] == '\0');
  }();
  if (!on) return;
  int32_t status = 0;
  check(yamoe_b200_device_status(ws.data_ptr(), st, &status), what);
  TORCH_CHECK(status == 0, "yamoe_b200: ", what, " failed: ", yamoe_b200_status_string(YAMOE_ERR_DEVICE_TIMEOUT),
              " (device status ", status, ")");
}

at::Tensor workspace(size_t nbytes, const at::Tensor& like) {
  return at::empty({(int64_t)(nbytes > 256 ? nbytes : 256)}, like.options().dtype(at::kByte));
}

at::Tensor experts_cuda(const at::Tensor& hidden_states, const at::Tensor& router_indices,
                        const at::Tensor& routing_weights, const at::Tensor& gate_up_proj,
                        const at::Tensor& gate_up_proj_bias, const at::Tensor& down_proj,
                        const at::Tensor& down_proj_bias, int64_t expert_capacity, int64_t num_experts,
                        int64_t top_k) {
  const Shape s = validate(hidden_states, router_indices, routing_weights, gate_up_proj, gate_up_proj_bias, down_proj,
                           down_proj_bias, num_experts, top_k);
  const c10::cuda::CUDAGuard guard(hidden_states.device());
  const at::Tensor hs = hidden_states.contiguous(), ri = router_indices.to(at::kLong).contiguous(),
                   rw = routing_weights.contiguous(), wgu = gate_up_proj.contiguous(),
                   bgu = gate_up_proj_bias.contiguous(), wd = down_proj.contiguous(), bd = down_proj_bias.contiguous();
  at::Tensor out = at::empty_like(hs);
  const size_t nbytes = yamoe_b200_forward_workspace_bytes(s.T, s.H, s.E, s.K, s.dtype);
  TORCH_CHECK(nbytes > 0, "yamoe_b200: unsupported shape (H must be a positive multiple of 8, E <= 1024)");
  const at::Tensor ws = workspace(nbytes, hs);
  cudaStream_t st = at::cuda::getCurrentCUDAStream().stream();
  check(yamoe_b200_experts_forward(hs.data_ptr(), ri.data_ptr<int64_t>(), rw.data_ptr(), (int)rw.size(1),
                                   wgu.data_ptr(), bgu.data_ptr(), wd.data_ptr(), bd.data_ptr(), out.data_ptr(), s.T,
                                   s.H, s.E, s.K, expert_capacity, s.dtype, ws.data_ptr(), (size_t)ws.numel(), st),
        "experts");
  check_device_status(ws, st, "experts");
  return out;
}

std::vector<at::Tensor> experts_backward_cuda(const at::Tensor& grad_out, const at::Tensor& hidden_states,
                                              const at::Tensor& router_indices, const at::Tensor& routing_weights,
                                              const at::Tensor& gate_up_proj, const at::Tensor& gate_up_proj_bias,
                                              const at::Tensor& down_proj, const at::Tensor& down_proj_bias,
                                              int64_t expert_capacity, int64_t num_experts, int64_t top_k) {
  TORCH_CHECK(grad_out.is_cuda(), "grad_out must be CUDA");
  const Shape s = validate(hidden_states, router_indices, routing_weights, gate_up_proj, gate_up_proj_bias, down_proj,
                           down_proj_bias, num_experts, top_k);
  TORCH_CHECK(grad_out.numel() == s.T * s.H || grad_out.numel() == s.T * s.K * s.H,
              "grad_out numel must be T*H or T*K*H");
  TORCH_CHECK(grad_out.scalar_type() == hidden_states.scalar_type(), "grad_out must have the dtype of hidden_states");
  const int per_slot = (grad_out.numel() == s.T * s.K * s.H && s.K != 1) ? 1 : 0;
  const c10::cuda::CUDAGuard guard(hidden_states.device());
  const at::Tensor go = grad_out.contiguous(), hs = hidden_states.contiguous(),
                   ri = router_indices.to(at::kLong).contiguous(), rw = routing_weights.contiguous(),
                   wgu = gate_up_proj.contiguous(), bgu = gate_up_proj_bias.contiguous(), wd = down_proj.contiguous(),
                   bd = down_proj_bias.contiguous();
  at::Tensor d_hidden = at::empty_like(hs), d_routing = at::empty_like(rw), d_wgu = at::empty_like(wgu),
             d_bgu = at::empty_like(bgu), d_wd = at::empty_like(wd), d_bd = at::empty_like(bd);
  const size_t nbytes = yamoe_b200_backward_workspace_bytes(s.T, s.H, s.E, s.K, s.dtype);
  TORCH_CHECK(nbytes > 0, "yamoe_b200: unsupported shape (H must be a positive multiple of 8, E <= 1024)");
  const at::Tensor ws = workspace(nbytes, hs);
  cudaStream_t st = at::cuda::getCurrentCUDAStream().stream();
  check(yamoe_b200_experts_backward(go.data_ptr(), per_slot, hs.data_ptr(), ri.data_ptr<int64_t>(), rw.data_ptr(),
                                    (int)rw.size(1), wgu.data_ptr(), bgu.data_ptr(), wd.data_ptr(), bd.data_ptr(),
                                    d_hidden.data_ptr(), d_routing.data_ptr(), d_wgu.data_ptr(), d_bgu.data_ptr(),
                                    d_wd.data_ptr(), d_bd.data_ptr(), s.T, s.H, s.E, s.K, expert_capacity, s.dtype,
                                    ws.data_ptr(), (size_t)ws.numel(), st),
        "experts_backward");
  check_device_status(ws, st, "experts_backward");
  return std::vector<at::Tensor>{d_hidden, d_routing, d_wgu, d_bgu, d_wd, d_bd};
}

// ---- 8-bit operands --------------------------------------------------------------------------------------------------

constexpr int64_t kGroup = 128;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? YAMOE_BF16 : YAMOE_F32; }
cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// A quantised operand: codes [B, rows, cols] or [rows, cols] with scales [.., rows or row blocks, groups].
struct Quantised {
  at::Tensor q, scale;
  bool defined() const { return q.defined(); }
};

yamoe_fp8_matrix_t matrix_of(const Quantised& m) {
  const bool batched = m.q.dim() == 3;
  yamoe_fp8_matrix_t r{};
  r.q = m.q.data_ptr();
  r.scale = m.scale.data_ptr<float>();
  const bool several = batched && m.q.size(0) > 1;
  // (one row: its pitch is that of the matrices)
  r.ld = m.q.size(-2) > 1 ? m.q.stride(-2) : several ? m.q.stride(0) : ceil_div(m.q.size(-1), 16) * 16;
  r.q_batch = several ? m.q.stride(0) : m.q.size(-2) * r.ld;
  r.scale_row = m.scale.stride(-2);
  r.scale_group = m.scale.stride(-1);
  r.scale_batch = batched ? m.scale.stride(0) : 0;
  return r;
}

// Codes with rows of 16-byte multiples (those that the kernels may fill up included) and scales with the rows side by side.
Quantised empty_quantised(bool batched, int64_t B, int64_t rows, int64_t cols, int64_t block_rows, const at::Tensor& like) {
  const int64_t ld = ceil_div(cols, 16) * 16, r = ceil_div(rows, block_rows), g = ceil_div(cols, kGroup);
  const auto codes = like.options().dtype(at::kFloat8_e4m3fn).requires_grad(false);
  const auto floats = like.options().dtype(at::kFloat).requires_grad(false);
  Quantised m;
  if (batched) {
    m.q = at::empty({B, rows, ld}, codes);
    m.scale = at::empty_strided({B, r, g}, {r * g, 1, r}, floats);
  } else {
    m.q = at::empty({rows, ld}, codes);
    m.scale = at::empty_strided({r, g}, {1, r}, floats);
  }
  if (ld != cols) m.q = m.q.narrow(-1, 0, cols);
  return m;
}

// x [B, M, K] or [M, K], contiguous -> codes of x and/or of its transpose
void quantise(const at::Tensor& x, int64_t block_rows, Quantised* out, Quantised* turned) {
  const bool batched = x.dim() == 3;
  const int64_t B = batched ? x.size(0) : 1, M = x.size(-2), K = x.size(-1);
  yamoe_fp8_matrix_t m{}, t{};
  if (out) {
    *out = empty_quantised(batched, B, M, K, block_rows, x);
    m = matrix_of(*out);
  }
  if (turned) {
    *turned = empty_quantised(batched, B, K, M, block_rows, x);
    t = matrix_of(*turned);
  }
  check(yamoe_b200_fp8_quantize(x.data_ptr(), out ? &m : nullptr, turned ? &t : nullptr, B, M, K, (int)block_rows, dtype_of(x),
                                current_stream()),
        "quantize_fp8");
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8_cuda(const at::Tensor& x, int64_t block_rows, bool transpose) {
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "quantize_fp8: x must be 2D [M, K] or 3D [B, M, K]");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16,
              "quantize_fp8: float32 or bfloat16 expected, got ", x.scalar_type());
  TORCH_CHECK(block_rows == 1 || block_rows == kGroup, "quantize_fp8: block_rows must be 1 or 128");
  const c10::cuda::CUDAGuard guard(x.device());
  Quantised m;
  // a transposed view is quantised from what it is a view of
  if (x.size(-2) > 1 && x.size(-1) > 1 && !x.is_contiguous() && x.transpose(-1, -2).is_contiguous()) {
    quantise(x.transpose(-1, -2), block_rows, transpose ? &m : nullptr, transpose ? nullptr : &m);
  } else {
    quantise(x.contiguous(), block_rows, transpose ? nullptr : &m, transpose ? &m : nullptr);
  }
  return {m.q, m.scale};
}

// Checks a pair of codes and scales and brings codes whose rows the kernels cannot address into a layout of their own.
Quantised operand(const char* op, const char* name, const at::Tensor& q, const at::Tensor& scale, int dim, bool blocks_only) {
  TORCH_CHECK(q.is_cuda() && scale.is_cuda(), op, ": ", name, " and its scale must be on CUDA");
  TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn, op, ": ", name, " must be float8_e4m3fn, got ", q.scalar_type());
  TORCH_CHECK(scale.scalar_type() == at::kFloat, op, ": the scale of ", name, " must be float32, got ", scale.scalar_type());
  TORCH_CHECK(q.dim() == dim && scale.dim() == dim, op, ": ", name, " and its scale must be ", dim, "D");
  const int64_t rows = q.size(-2), r = scale.size(-2);
  TORCH_CHECK(scale.size(-1) == ceil_div(q.size(-1), kGroup) && (r == ceil_div(rows, kGroup) || (!blocks_only && r == rows)) &&
                  (dim == 2 || scale.size(0) == q.size(0)),
              op, ": the scale of ", name, " must hold one value per group of ", blocks_only ? "128 x 128" : "1 or 128 x 128");
  const bool ok = q.stride(-1) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 &&
                  (rows <= 1 || (q.stride(-2) % 16 == 0 && q.stride(-2) >= q.size(-1))) &&
                  (dim == 2 || q.size(0) <= 1 ||
                   (rows <= 1 ? q.stride(0) % 16 == 0 && q.stride(0) >= q.size(-1)
                              : q.stride(-2) > 0 && q.stride(0) % q.stride(-2) == 0 && q.stride(0) / q.stride(-2) >= rows));
  // one row of a width that is no multiple of 16 may end where its memory ends
  if (ok || q.numel() == 0) return {q, scale};
  Quantised m = empty_quantised(dim == 3, dim == 3 ? q.size(0) : 1, rows, q.size(-1), kGroup, q);
  m.q.copy_(q);
  m.scale = scale;
  return m;
}

at::Tensor mm(const Quantised& a, const Quantised& b, at::ScalarType out_dtype) {
  const bool batched = a.q.dim() == 3;
  const int64_t B = batched ? a.q.size(0) : 1, M = a.q.size(-2), N = b.q.size(-2), K = a.q.size(-1);
  const auto options = a.scale.options().dtype(out_dtype);
  at::Tensor out = batched ? at::empty({B, M, N}, options) : at::empty({M, N}, options);
  if (out.numel() == 0) return out;
  const yamoe_fp8_matrix_t ma = matrix_of(a), mb = matrix_of(b);
  const at::Tensor ws = workspace(yamoe_b200_fp8_mm_workspace_bytes(B, M, N, K), a.scale);
  const int block = b.scale.size(-2) == ceil_div(N, kGroup) ? (int)kGroup : 1;
  check(yamoe_b200_fp8_mm(&ma, &mb, block, out.data_ptr(), B, M, N, K, out_dtype == at::kFloat ? YAMOE_F32 : YAMOE_BF16,
                          ws.data_ptr(), (size_t)ws.numel(), current_stream()),
        "fp8_mm");
  if (K > 0) check_device_status(ws, current_stream(), "fp8_mm");
  return out;
}

at::Tensor fp8_mm_cuda(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale,
                       at::ScalarType out_dtype) {
  TORCH_CHECK(a.dim() == 2 || a.dim() == 3, "fp8_mm: a must be 2D [M, K] or 3D [B, M, K]");
  TORCH_CHECK(out_dtype == at::kFloat || out_dtype == at::kBFloat16, "fp8_mm: out_dtype must be float32 or bfloat16");
  TORCH_CHECK(b.device() == a.device() && a_scale.device() == a.device() && b_scale.device() == a.device(),
              "fp8_mm: tensors must be on one device");
  const c10::cuda::CUDAGuard guard(a.device());
  const Quantised qa = operand("fp8_mm", "a", a, a_scale, a.dim(), false), qb = operand("fp8_mm", "b", b, b_scale, a.dim(), false);
  TORCH_CHECK(a_scale.size(-2) == a.size(-2), "fp8_mm: a must have a scale per row and group of 128");
  TORCH_CHECK(a.size(-1) == b.size(-1), "fp8_mm: a is [.., M, K] and b [.., N, K]: K is ", a.size(-1), " and ", b.size(-1));
  TORCH_CHECK(a.dim() == 2 || a.size(0) == b.size(0), "fp8_mm: a and b must hold the same number of matrices");
  return mm(qa, qb, out_dtype);
}

void check_linear(const at::Tensor& x, const at::Tensor& w) {
  TORCH_CHECK(x.is_cuda() && w.is_cuda() && x.device() == w.device(), "fp8_linear: x and weight must be on one CUDA device");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16,
              "fp8_linear: float32 or bfloat16 expected, got ", x.scalar_type());
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "fp8_linear: weight must have the dtype of x (", x.scalar_type(), "), got ",
              w.scalar_type());
  TORCH_CHECK((w.dim() == 2 && x.dim() >= 1) || (w.dim() == 3 && x.dim() == 3 && x.size(0) == w.size(0)),
              "fp8_linear: weight must be [N, K], or [B, N, K] with x [B, M, K]");
  TORCH_CHECK(x.size(-1) == w.size(-1), "fp8_linear: x is [.., K] and weight [.., N, K]: K is ", x.size(-1), " and ", w.size(-1));
}

// x (or dy) as the matrices that a weight of this rank multiplies
at::Tensor as_matrices(const at::Tensor& x, int64_t rank) {
  if (rank == 3 || x.dim() == 2) return x.contiguous();
  int64_t rows = 1;                        // (reshape cannot tell it where a row has no values)
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  return x.reshape({rows, x.size(-1)}).contiguous();
}
std::vector<int64_t> linear_shape(const at::Tensor& x, const at::Tensor& w) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = w.size(-2);
  return s;
}

at::Tensor fp8_linear_cuda(const at::Tensor& x, const at::Tensor& weight) {
  check_linear(x, weight);
  const c10::cuda::CUDAGuard guard(x.device());
  Quantised xq, wq;
  quantise(as_matrices(x, weight.dim()), 1, &xq, nullptr);
  quantise(weight.contiguous(), kGroup, &wq, nullptr);
  return mm(xq, wq, x.scalar_type()).view(linear_shape(x, weight));
}

// Backward computes on codes, below the autograd layer: what it returns has no derivative.  Where a graph of it is asked for
// (create_graph), it leads through a node that raises when it is differentiated, on to all that it depends on.
void differentiate_no_further(const at::Tensor& dy, at::Tensor& dx, at::Tensor& dw) {
  torch::autograd::edge_list on = torch::autograd::get_current_node()->next_edges();
  for (const torch::autograd::Edge& e : torch::autograd::collect_next_edges(dy)) on.push_back(e);
  const auto node = std::make_shared<torch::autograd::Error>("fp8_linear can be differentiated once only", std::move(on));
  for (at::Tensor* t : {&dx, &dw})
    if (t->defined()) torch::autograd::create_gradient_edge(*t, node);
}

// y = Q(x) Q(w)^T with dx = Q(dy) Q(w) and dw = Q(dy^T) Q(x^T)^T; what backward needs of x and w is kept as codes.
struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight) {
    check_linear(x, weight);
    const c10::cuda::CUDAGuard guard(x.device());
    const at::AutoDispatchBelowADInplaceOrView below;      // of what is made here nothing is recorded
    const bool dx = x.requires_grad(), dw = weight.requires_grad();
    Quantised xq, wq, xt, wt;
    quantise(as_matrices(x, weight.dim()), 1, &xq, dw ? &xt : nullptr);
    quantise(weight.contiguous(), kGroup, &wq, dx ? &wt : nullptr);
    ctx->save_for_backward({xt.q, xt.scale, wt.q, wt.scale});
    ctx->saved_data["x_shape"] = x.sizes().vec();
    ctx->saved_data["rank"] = (int64_t)weight.dim();
    return mm(xq, wq, x.scalar_type()).view(linear_shape(x, weight));
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Quantised xt{saved[0], saved[1]}, wt{saved[2], saved[3]};
    const bool want_x = ctx->needs_input_grad(0) && wt.defined(), want_w = ctx->needs_input_grad(1) && xt.defined();
    const at::Tensor dy = grads[0];
    if (!dy.defined() || !(want_x || want_w)) return {at::Tensor(), at::Tensor()};
    const c10::cuda::CUDAGuard guard(dy.device());
    at::Tensor dx, dw;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      // hooks on saved tensors may give the codes back in a layout of their own
      if (want_w) xt = operand("fp8_linear", "codes of x", xt.q, xt.scale, (int)xt.q.dim(), false);
      if (want_x) wt = operand("fp8_linear", "codes of weight", wt.q, wt.scale, (int)wt.q.dim(), true);
      const at::Tensor d = as_matrices(dy, ctx->saved_data["rank"].toInt());
      Quantised g, gt;
      quantise(d, 1, want_x ? &g : nullptr, want_w ? &gt : nullptr);
      if (want_x) dx = mm(g, wt, d.scalar_type()).view(ctx->saved_data["x_shape"].toIntVector());
      if (want_w) dw = mm(gt, xt, d.scalar_type());
    }
    if (at::GradMode::is_enabled()) differentiate_no_further(dy, dx, dw);
    return {dx, dw};
  }
};

// Forward mode: a tangent that nobody takes up would count as zero.
void check_no_tangent(const at::Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "fp8_linear: forward-mode differentiation is not supported");
}

at::Tensor fp8_linear_autograd(const at::Tensor& x, const at::Tensor& weight) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
    check_no_tangent(x);
    check_no_tangent(weight);
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad())) return Fp8Linear::apply(x, weight);
  at::AutoDispatchBelowAutograd below;
  return fp8_linear_cuda(x, weight);
}

// contiguous, on the 16-byte boundary that the kernels' wide loads and copies want
at::Tensor aligned(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

at::Tensor experts_fp8_cuda(const at::Tensor& hidden_states, const at::Tensor& router_indices, const at::Tensor& routing_weights,
                            const at::Tensor& gate_up, const at::Tensor& gate_up_scale, const at::Tensor& gate_up_bias,
                            const at::Tensor& down, const at::Tensor& down_scale, const at::Tensor& down_bias,
                            int64_t expert_capacity, int64_t num_experts, int64_t top_k) {
  const at::Tensor* tensors[] = {&hidden_states, &router_indices, &routing_weights, &gate_up_bias, &down_bias};
  const char* names[] = {"hidden_states", "router_indices", "routing_weights", "gate_up_bias", "down_bias"};
  for (int i = 0; i < 5; ++i) {
    TORCH_CHECK(tensors[i]->is_cuda() && tensors[i]->device() == hidden_states.device(), names[i],
                " must be on the CUDA device of hidden_states");
    TORCH_CHECK(tensors[i]->dim() == 2, names[i], " must be 2D");
    if (i != 1)
      TORCH_CHECK(tensors[i]->scalar_type() == hidden_states.scalar_type(), names[i], " must have the dtype of hidden_states (",
                  hidden_states.scalar_type(), "), got ", tensors[i]->scalar_type());
  }
  const auto dt = hidden_states.scalar_type();
  TORCH_CHECK(dt == at::kFloat || dt == at::kBFloat16, "yamoe_b200 supports float32 and bfloat16, got ", dt);
  const int64_t T = hidden_states.size(0), H = hidden_states.size(1), E = num_experts, K = top_k;
  TORCH_CHECK(router_indices.scalar_type() == at::kLong || router_indices.scalar_type() == at::kInt,
              "router_indices must be int64");
  TORCH_CHECK(router_indices.size(0) == T && router_indices.size(1) == K, "router_indices must be [T, K]");
  TORCH_CHECK(routing_weights.size(0) == T && (routing_weights.size(1) == K || routing_weights.size(1) == E),
              "routing_weights must be [T, K] or [T, E]");
  TORCH_CHECK(gate_up.dim() == 3 && gate_up.size(0) == E && gate_up.size(1) == 2 * H && gate_up.size(2) == H,
              "gate_up must be [E, 2*H, H]");
  TORCH_CHECK(down.dim() == 3 && down.size(0) == E && down.size(1) == H && down.size(2) == H, "down must be [E, H, H]");
  TORCH_CHECK(gate_up_bias.size(0) == E && gate_up_bias.size(1) == 2 * H, "gate_up_bias must be [E, 2*H]");
  TORCH_CHECK(down_bias.size(0) == E && down_bias.size(1) == H, "down_bias must be [E, H]");
  TORCH_CHECK(gate_up.device() == hidden_states.device() && down.device() == hidden_states.device() &&
                  gate_up_scale.device() == hidden_states.device() && down_scale.device() == hidden_states.device(),
              "weights and scales must be on the CUDA device of hidden_states");
  const c10::cuda::CUDAGuard guard(hidden_states.device());
  const Quantised g = operand("experts_fp8", "gate_up", gate_up, gate_up_scale, 3, true),
                  d = operand("experts_fp8", "down", down, down_scale, 3, true);
  const at::Tensor hs = aligned(hidden_states), ri = router_indices.to(at::kLong).contiguous(),
                   rw = routing_weights.contiguous(), bg = aligned(gate_up_bias), bd = aligned(down_bias);
  at::Tensor out = at::empty_like(hs);
  const int code = dtype_of(hs);
  const size_t nbytes = yamoe_b200_experts_fp8_workspace_bytes(T, (int)H, (int)E, (int)K, code);
  TORCH_CHECK(nbytes > 0, "yamoe_b200: unsupported shape (H must be a positive multiple of 8, E <= 1024)");
  const at::Tensor ws = workspace(nbytes, hs);
  const yamoe_fp8_matrix_t mg = matrix_of(g), md = matrix_of(d);
  check(yamoe_b200_experts_fp8_forward(hs.data_ptr(), ri.data_ptr<int64_t>(), rw.data_ptr(), (int)rw.size(1), &mg, bg.data_ptr(),
                                       &md, bd.data_ptr(), out.data_ptr(), T, (int)H, (int)E, (int)K, expert_capacity, code,
                                       ws.data_ptr(), (size_t)ws.numel(), current_stream()),
        "experts_fp8");
  if (T > 0) check_device_status(ws, current_stream(), "experts_fp8");
  return out;
}

std::tuple<at::Tensor, at::Tensor> moe_layer_cuda(const at::Tensor& hidden_states, const at::Tensor& router_weight,
                                                  const std::optional<at::Tensor>& router_bias, const at::Tensor& gate_up,
                                                  const at::Tensor& gate_up_bias, const at::Tensor& down,
                                                  const at::Tensor& down_bias, int64_t expert_capacity, int64_t num_experts,
                                                  int64_t top_k, const std::optional<at::Tensor>& gate_up_scale,
                                                  const std::optional<at::Tensor>& down_scale) {
  const int64_t T = hidden_states.size(0), H = hidden_states.size(-1), E = num_experts, K = top_k;
  TORCH_CHECK(hidden_states.dim() == 2, "moe_layer: hidden_states must be 2D [T, H]");
  TORCH_CHECK(hidden_states.scalar_type() == at::kBFloat16, "moe_layer: bfloat16 expected, got ", hidden_states.scalar_type());
  TORCH_CHECK(T <= 32 && T * K <= 256, "moe_layer: at most 32 tokens and 256 assignments, got ", T, " tokens of ", K,
              " (use router_forward and experts, or experts_fp8, for more)");
  const bool has_bias = router_bias.has_value() && router_bias->defined();
  const at::Tensor rb = has_bias ? *router_bias : at::Tensor();
  const at::Tensor* tensors[] = {&router_weight, &gate_up_bias, &down_bias, &rb};
  const char* names[] = {"router_weight", "gate_up_bias", "down_bias", "router_bias"};
  for (int i = 0; i < (has_bias ? 4 : 3); ++i)
    TORCH_CHECK(tensors[i]->device() == hidden_states.device() && tensors[i]->scalar_type() == at::kBFloat16, "moe_layer: ",
                names[i], " must be bfloat16 on the device of hidden_states");
  TORCH_CHECK(router_weight.dim() == 2 && router_weight.size(0) == E && router_weight.size(1) == H,
              "moe_layer: router_weight must be [E, H]");
  TORCH_CHECK(!has_bias || rb.numel() == E, "moe_layer: router_bias must be [E]");
  TORCH_CHECK(gate_up_bias.dim() == 2 && gate_up_bias.size(0) == E && gate_up_bias.size(1) == 2 * H,
              "moe_layer: gate_up_bias must be [E, 2*H]");
  TORCH_CHECK(down_bias.dim() == 2 && down_bias.size(0) == E && down_bias.size(1) == H, "moe_layer: down_bias must be [E, H]");
  TORCH_CHECK(K >= 1 && K <= E, "moe_layer: top_k must be between 1 and the number of experts");
  const bool fp8 = gate_up.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(gate_up_scale.has_value() == fp8 && down_scale.has_value() == fp8,
              "moe_layer: scales belong to float8_e4m3fn weights, and to both of them");
  TORCH_CHECK(gate_up.device() == hidden_states.device() && down.device() == hidden_states.device() &&
                  (!fp8 || (gate_up_scale->device() == hidden_states.device() && down_scale->device() == hidden_states.device())),
              "moe_layer: weights and scales must be on the device of hidden_states");
  const c10::cuda::CUDAGuard guard(hidden_states.device());
  Quantised g, d;
  at::Tensor gu = gate_up, dn = down;
  yamoe_fp8_matrix_t mg{}, md{};
  if (fp8) {
    TORCH_CHECK(gate_up.dim() == 3 && gate_up.size(0) == E && gate_up.size(1) == 2 * H && gate_up.size(2) == H,
                "moe_layer: float8_e4m3fn gate_up must be [E, 2*H, H]");
    TORCH_CHECK(down.dim() == 3 && down.size(0) == E && down.size(1) == H && down.size(2) == H, "moe_layer: down must be [E, H, H]");
    g = operand("moe_layer", "gate_up", gate_up, *gate_up_scale, 3, true);
    d = operand("moe_layer", "down", down, *down_scale, 3, true);
    mg = matrix_of(g);
    md = matrix_of(d);
  } else {
    TORCH_CHECK(gate_up.scalar_type() == at::kBFloat16 && down.scalar_type() == at::kBFloat16,
                "moe_layer: weights must be bfloat16 or float8_e4m3fn");
    TORCH_CHECK(gate_up.dim() == 3 && gate_up.size(0) == E && gate_up.size(1) == H && gate_up.size(2) == 2 * H,
                "moe_layer: gate_up must be [E, H, 2*H]");
    TORCH_CHECK(down.dim() == 3 && down.size(0) == E && down.size(1) == H && down.size(2) == H, "moe_layer: down must be [E, H, H]");
    gu = aligned(gate_up);
    dn = aligned(down);
  }
  const at::Tensor hs = aligned(hidden_states), rw = aligned(router_weight), bg = aligned(gate_up_bias), bd = aligned(down_bias),
                   br = has_bias ? rb.contiguous() : rb;
  at::Tensor out = at::empty({T, H}, hs.options()), scores = at::empty({T, E}, hs.options());
  const size_t nbytes = yamoe_b200_moe_layer_workspace_bytes(T, (int)H, (int)E, (int)K);
  TORCH_CHECK(nbytes > 0, "yamoe_b200: unsupported shape (H must be a positive multiple of 8, E <= 1024, top_k <= 32)");
  const at::Tensor ws = workspace(nbytes, hs);
  check(yamoe_b200_moe_layer(hs.data_ptr(), rw.data_ptr(), has_bias ? br.data_ptr() : nullptr, fp8 ? nullptr : gu.data_ptr(),
                             fp8 ? &mg : nullptr, bg.data_ptr(), fp8 ? nullptr : dn.data_ptr(), fp8 ? &md : nullptr, bd.data_ptr(),
                             out.data_ptr(), scores.data_ptr(), T, (int)H, (int)E, (int)K, expert_capacity, YAMOE_BF16, ws.data_ptr(),
                             (size_t)ws.numel(), current_stream()),
        "moe_layer");
  if (T > 0) check_device_status(ws, current_stream(), "moe_layer");
  return {out, scores};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(yamoe_b200, m) {
  m.def(
      "experts(Tensor hidden_states, Tensor router_indices, Tensor routing_weights, Tensor gate_up_proj, "
      "Tensor gate_up_proj_bias, Tensor down_proj, Tensor down_proj_bias, int expert_capacity, "
      "int num_experts, int top_k) -> Tensor");
  m.def(
      "experts_backward(Tensor grad_out, Tensor hidden_states, Tensor router_indices, Tensor routing_weights, "
      "Tensor gate_up_proj, Tensor gate_up_proj_bias, Tensor down_proj, Tensor down_proj_bias, "
      "int expert_capacity, int num_experts, int top_k) -> Tensor[]");
  m.def("quantize_fp8(Tensor x, int block_rows=1, bool transpose=False) -> (Tensor, Tensor)");
  m.def("fp8_mm(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, ScalarType out_dtype=bfloat16) -> Tensor");
  m.def("fp8_linear(Tensor x, Tensor weight) -> Tensor");
  m.def(
      "experts_fp8(Tensor hidden_states, Tensor router_indices, Tensor routing_weights, Tensor gate_up, Tensor gate_up_scale, "
      "Tensor gate_up_bias, Tensor down, Tensor down_scale, Tensor down_bias, int expert_capacity, int num_experts, int top_k) "
      "-> Tensor");
  m.def(
      "moe_layer(Tensor hidden_states, Tensor router_weight, Tensor? router_bias, Tensor gate_up, Tensor gate_up_bias, Tensor down, "
      "Tensor down_bias, int expert_capacity, int num_experts, int top_k, Tensor? gate_up_scale=None, Tensor? down_scale=None) -> "
      "(Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(yamoe_b200, AutogradCUDA, m) {
  m.impl("fp8_linear", &fp8_linear_autograd);
}

TORCH_LIBRARY_IMPL(yamoe_b200, CUDA, m) {
  m.impl("experts", &experts_cuda);
  m.impl("experts_backward", &experts_backward_cuda);
  m.impl("quantize_fp8", &quantize_fp8_cuda);
  m.impl("fp8_mm", &fp8_mm_cuda);
  m.impl("fp8_linear", &fp8_linear_cuda);
  m.impl("experts_fp8", &experts_fp8_cuda);
  m.impl("moe_layer", &moe_layer_cuda);
}
