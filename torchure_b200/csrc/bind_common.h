// What the binding files share: the launchers of bindings.cpp that other files call on tensors, and what operators with autograd nodes have in
// common.
#pragma once

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <torch/extension.h>

#include "api.h"
#include "pdl.h"

torch::Tensor attn_err_word();   // device int32[4], set by bounded waits that expired; refused on another GPU than the process's first
int bind_num_sms();              // SMs a persistent kernel may use
void bind_gemm(const torch::Tensor& a, const torch::Tensor& b, torch::Tensor& out, bool a_mn, bool b_mn, int64_t out_mode,
               int64_t splits = 0, int64_t tile_n = 0, bool b_is_old = false);
bool bind_gemm_swiglu(const torch::Tensor& x, const torch::Tensor& w, c10::optional<torch::Tensor> gu, torch::Tensor& act);
bool bind_gemm_swiglu_bwd(const torch::Tensor& dy, const torch::Tensor& w, const torch::Tensor& gu, torch::Tensor& dgu);
void bind_count_launches(int64_t n);      // kernels that an operator with an autograd node in C++ has launched

// torch::empty for GPU tensors without the dispatcher (0.6 us instead of 1.8)
inline torch::Tensor empty(c10::IntArrayRef size, const at::TensorOptions& options) { return at::detail::empty_cuda(size, options); }

// Backward passes run in threads of autograd's, which do not hold the interpreter's lock.
struct Outputs {
  bool poisoned;
  torch::Tensor operator()(const char* name, c10::IntArrayRef size, const at::TensorOptions& options) const {
    torch::Tensor t = empty(size, options);
    if (poisoned) {
      pybind11::gil_scoped_acquire lock;
      pybind11::module_::import("torchure_b200.ops.debug").attr("track")(name, t);
    }
    return t;
  }
};

// Launches overlap (pdl.h): a kernel comes up while the one before ends, and waits before it reads.  The feed-forward forward, us, without and
// with: 8 experts of 1024 x 1536, 512 rows 48, 39; 4096 rows 83, 70; 32768 rows 284, 278.  (A graph keeps plain edges.)
struct Overlap : tb::PdlScope {
  Overlap() : tb::PdlScope(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) {}
};

inline void only_once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient itself has no gradient (create_graph is not supported)");
}
// A dual tensor asks for no gradient, so that calls without gradients would pass its tangent by
template <class... Ts>
void no_tangents(const char* what, const Ts&... tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(... || (tensors.defined() && tensors._fw_grad(0).defined())), what,
                              ": forward-mode derivatives are not supported");
}
