// What the sources of the torch binding share: status checks, workspaces, refusals of derivatives that the operators do not have.
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cstdlib>
#include <initializer_list>
#include <string>

#include "../../include/yamoe_b200.h"

namespace {

inline void check(int status, const char* what) {
  TORCH_CHECK(status == YAMOE_OK, "yamoe_b200: ", what, " failed: ", yamoe_b200_status_string(status), " (status ",
              status, ")");
}

// YAMOE_B200_CHECK_STATUS=1: read the device status word after the call (one stream synchronisation)
inline void check_device_status(const at::Tensor& ws, cudaStream_t st, const char* what) {
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

inline at::Tensor workspace(size_t nbytes, const at::Tensor& like) {
  return at::empty({(int64_t)(nbytes > 256 ? nbytes : 256)}, like.options().dtype(at::kByte));
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? YAMOE_BF16 : YAMOE_F32; }
inline cudaStream_t current_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// contiguous, on the 16-byte boundary that the kernels' wide loads and copies want
inline at::Tensor aligned(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// A backward pass computes below the autograd layer: what it returns has no derivative.  Where a graph of it is asked for
// (create_graph), it leads through a node that raises when it is differentiated, on to all that it depends on.
inline void differentiate_no_further(const char* op, std::initializer_list<at::Tensor> from, std::initializer_list<at::Tensor*> grads) {
  torch::autograd::edge_list on = torch::autograd::get_current_node()->next_edges();
  for (const at::Tensor& t : from)
    for (const torch::autograd::Edge& e : torch::autograd::collect_next_edges(t)) on.push_back(e);
  const auto node = std::make_shared<torch::autograd::Error>(std::string(op) + " can be differentiated once only", std::move(on));
  for (at::Tensor* t : grads)
    if (t->defined()) torch::autograd::create_gradient_edge(*t, node);
}

// The result of an operator without a gradient, where one of `from` wants one: a node that raises when it is differentiated, on the way to them.  (Torch's
// default would be a warning then, and no gradient.)
inline void no_gradient(const char* op, std::initializer_list<at::Tensor> from, at::Tensor& result) {
  torch::autograd::edge_list on;
  for (const at::Tensor& t : from)
    for (const torch::autograd::Edge& e : torch::autograd::collect_next_edges(t)) on.push_back(e);
  torch::autograd::create_gradient_edge(result, std::make_shared<torch::autograd::Error>(std::string(op) + " has no gradient", std::move(on)));
}

// Forward mode: a tangent that nobody takes up would count as zero.
inline void check_no_tangent(const char* op, const at::Tensor& t) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  TORCH_CHECK(!t._fw_grad(0).defined(), op, ": forward-mode differentiation is not supported");
}

}  // namespace
